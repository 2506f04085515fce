// Selective state space scan and the short causal convolution in front of it, for prompts and for
// single tokens.
#include "common.cuh"

#include <numeric>

namespace tesm {

// x * sigmoid(x); 0 for x -> -inf (the reciprocal of inf is 0, and x * 0 stays finite for finite x)
__device__ __forceinline__ float silu(float x) { return x * rcp_approx(1.f + ex2_approx(-x * kLog2e)); }

__device__ __forceinline__ float2 silu2(float2 x) {
  const float2 t = __fmul2_rn(x, make_float2(-kLog2e, -kLog2e));
  const float2 d = __fadd2_rn(make_float2(ex2_approx(t.x), ex2_approx(t.y)), make_float2(1.f, 1.f));
  return __fmul2_rn(x, make_float2(rcp_approx(d.x), rcp_approx(d.y)));
}

// softplus(x) = max(x, 0) + log(1 + u), u = e^-|x| in (0, 1].  log(1 + u) = 2 atanh(s) with
// s = u / (2 + u) <= 1/3: the odd series in s keeps full relative accuracy for small u, where
// forming 1 + u would round u away.  Terms to s^13 leave 1.6e-8 relative at s = 1/3.
__device__ __forceinline__ float2 softplus2(float2 x) {
  const float2 u = make_float2(ex2_approx(-fabsf(x.x) * kLog2e), ex2_approx(-fabsf(x.y) * kLog2e));
  const float2 den = __fadd2_rn(u, make_float2(2.f, 2.f));
  const float2 s = __fmul2_rn(u, make_float2(rcp_approx(den.x), rcp_approx(den.y))), q = __fmul2_rn(s, s);
  float2 p = make_float2(1.f / 13.f, 1.f / 13.f);
  p = __ffma2_rn(p, q, make_float2(1.f / 11.f, 1.f / 11.f));
  p = __ffma2_rn(p, q, make_float2(1.f / 9.f, 1.f / 9.f));
  p = __ffma2_rn(p, q, make_float2(1.f / 7.f, 1.f / 7.f));
  p = __ffma2_rn(p, q, make_float2(1.f / 5.f, 1.f / 5.f));
  p = __ffma2_rn(p, q, make_float2(1.f / 3.f, 1.f / 3.f));
  p = __ffma2_rn(p, q, make_float2(1.f, 1.f));
  return __ffma2_rn(__fadd2_rn(s, s), p, make_float2(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)));
}
__device__ __forceinline__ float softplus(float x) {
  const float u = ex2_approx(-fabsf(x) * kLog2e);
  const float s = u * rcp_approx(2.f + u), q = s * s;
  float p = 1.f / 13.f;
  p = fmaf(p, q, 1.f / 11.f);
  p = fmaf(p, q, 1.f / 9.f);
  p = fmaf(p, q, 1.f / 7.f);
  p = fmaf(p, q, 1.f / 5.f);
  p = fmaf(p, q, 1.f / 3.f);
  p = fmaf(p, q, 1.f);
  return fmaf(s + s, p, fmaxf(x, 0.f));
}

template <class T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f(float x) { return x; }
template <>
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f(float x) { return __float2bfloat16_rn(x); }

// N consecutive elements as they are in memory: one 16-byte access per 16 bytes where `vec`
// promises alignment and all N exist, else the first `have` of them one by one (the rest zero).
template <class T, int N>
struct alignas(N * sizeof(T) >= 16 ? 16 : N * sizeof(T)) Pack {
  T v[N];
  __device__ __forceinline__ void load(const T *p, bool vec, int have) {
    if constexpr (N * sizeof(T) % 16 == 0) {
      if (vec && have >= N) {
#pragma unroll
        for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i)
          reinterpret_cast<uint4 *>(v)[i] = reinterpret_cast<const uint4 *>(p)[i];
        return;
      }
    }
    load_single(p, have);
  }
  // for memory that the kernel does not write
  __device__ __forceinline__ void load_read_only(const T *p, bool vec, int have) {
    if constexpr (N * sizeof(T) % 16 == 0) {
      if (vec && have >= N) {
#pragma unroll
        for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i)
          reinterpret_cast<uint4 *>(v)[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
        return;
      }
    }
    load_single(p, have);
  }
  __device__ __forceinline__ void load_single(const T *p, int have) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = i < have ? p[i] : from_f<T>(0.f);
  }
  __device__ __forceinline__ void load_all(const T *p) {  // 8 or 16 bytes, aligned
    if constexpr (N * sizeof(T) == 8)
      *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(p);
    else
      *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
  }
  __device__ __forceinline__ void store(T *p, bool vec, int have) const {
    if constexpr (N * sizeof(T) % 16 == 0) {
      if (vec && have >= N) {
#pragma unroll
        for (int i = 0; i < (int)(N * sizeof(T) / 16); ++i)
          reinterpret_cast<uint4 *>(p)[i] = reinterpret_cast<const uint4 *>(v)[i];
        return;
      }
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (i < have) p[i] = v[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = from_f<T>(0.f);
  }
  __device__ __forceinline__ void pairs(float2 (&f)[(N + 1) / 2]) const {
#pragma unroll
    for (int i = 0; i < (N + 1) / 2; ++i) f[i] = make_float2(to_f(v[2 * i]), 2 * i + 1 < N ? to_f(v[(2 * i + 1) % N]) : 0.f);
  }
};

// A (batch, token, channel) tensor with unit channel stride.
template <class T>
struct Rows {
  T *p;
  int64_t ldb, ldl;
  __device__ __forceinline__ T *at(int64_t b, int64_t t, int64_t c) const { return p + b * ldb + t * ldl + c; }
};

__device__ __forceinline__ int seq_len(const int *lengths, int64_t b, int L) {
  return lengths ? min(max(lengths[b], 0), L) : L;
}

// ------------------------------------------------------------ host-side checks of what is written
struct Span {
  uintptr_t lo, hi;
  uintptr_t row, pitch;  // bytes of a row; rows lie at lo plus multiples of pitch (0: one row)
  // Columns of one buffer, as slices of a projection, lie between one another without a shared byte: so
  // it is where the rows, modulo the distance that all of them keep, do not meet.
  bool meets(const Span &o) const {
    if (lo >= o.hi || o.lo >= hi) return false;
    if (o.lo < lo) return o.meets(*this);
    const uintptr_t g = std::gcd(pitch, o.pitch);
    if (g == 0) return true;
    const uintptr_t off = (o.lo - lo) % g;
    return off < row || off + o.row > g;
  }
};
// a (B, L, n) tensor of `es`-byte elements with element strides ldb, ldl
static Span span3(const void *p, int64_t B, int64_t L, int64_t n, int64_t ldb, int64_t ldl, int64_t es) {
  if (!p) return Span{};
  const uintptr_t lo = (uintptr_t)p;
  return Span{lo, lo + (uintptr_t)(((B - 1) * ldb + (L - 1) * ldl + n) * es), (uintptr_t)(n * es),
              (uintptr_t)(std::gcd(B > 1 ? ldb : 0, L > 1 ? ldl : 0) * es)};
}
static Span span1(const void *p, int64_t bytes) {
  return p ? Span{(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, (uintptr_t)bytes, 0} : Span{};
}
// whether a (B, L, n) tensor holds an element twice
static bool self_overlap(int64_t B, int64_t L, int64_t n, int64_t ldb, int64_t ldl) {
  if (B > 1 && L > 1)
    return ldb < ldl ? ldb < n || ldl < (B - 1) * ldb + n : ldl < n || ldb < (L - 1) * ldl + n;
  return (B > 1 && ldb < n) || (L > 1 && ldl < n);
}

// ------------------------------------------------------------ causal convolution
// y_t = act(bias + sum_j w_j x_{t-K+1+j}).  Bytes bound it: x is read once (and K - 1 rows again per
// tile of tokens), y written once.  A thread owns N channels (16 bytes of them) and walks a tile
// with the last K - 1 inputs in registers, two channels per packed FMA.  16 rows ahead are on
// their way into the thread's own slots of shared memory: registers for as many would halve the
// occupancy (4 rows ahead in registers: 116 us against 91 us, 5.9 TB/s, at 4 x 4096 tokens of 8192
// bf16 channels, K = 4, replayed from a graph; a plain copy of the same bytes takes 87 us).  Rows are addressed by running
// pointers, since 64-bit products per row cost as much as the arithmetic.  Single tokens take kConvBatch
// sequences per thread, so that the weights are read less often (256 sequences: 11 us, against 18 with one).
constexpr int kConvThreads = 128, kConvBatch = 4;

template <class T, int N, int K, int U>
__global__ void __launch_bounds__(kConvThreads)
    k_causal_conv(Rows<const T> x, int B, int L, int D, int TT, int nb, int vec, const float *__restrict__ weight,
                  const float *__restrict__ bias, T *__restrict__ state, const int *__restrict__ lengths, int act,
                  Rows<T> y, int chunks, int tiles) {
  pdl_trigger();
  pdl_wait();
  const int chunk = blockIdx.x % chunks;
  const int tile = blockIdx.x / chunks % tiles;
  const int b0 = blockIdx.x / chunks / tiles * nb, b1 = min(b0 + nb, B);
  const int c = (chunk * kConvThreads + threadIdx.x) * N;
  if (c >= D) return;
  const int have = min(N, D - c);
  constexpr bool kAsync = N * sizeof(T) == 16 && U == 2;  // with D a multiple of N: whole accesses only
  constexpr int kGroups = 8;  // groups of U rows in shared memory
  __shared__ __align__(16) char smem[kAsync ? kGroups * U * kConvThreads * 16 : 16];
  const uint32_t slot = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16;
  constexpr int H2 = (N + 1) / 2;
  float2 w[H2][K], bs[H2];  // pairs of channels, for packed arithmetic
  {
    float wf[2 * H2 * K];  // as in memory: channel by channel
    if (N > 1 && have == N && ((uintptr_t)weight & 15) == 0) {
#pragma unroll
      for (int i = 0; i < N * K / 4; ++i)
        reinterpret_cast<float4 *>(wf)[i] = __ldg(reinterpret_cast<const float4 *>(weight + (int64_t)c * K) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 2 * H2 * K; ++i) wf[i] = i / K < have ? weight[(int64_t)c * K + i] : 0.f;
    }
#pragma unroll
    for (int h = 0; h < H2; ++h) {
      bs[h] = make_float2(bias && 2 * h < have ? bias[c + 2 * h] : 0.f, bias && 2 * h + 1 < have ? bias[c + 2 * h + 1] : 0.f);
#pragma unroll
      for (int j = 0; j < K; ++j) w[h][j] = make_float2(wf[2 * h * K + j], wf[(2 * h + 1) * K + j]);
    }
  }
  const int t0 = tile * TT, t1 = min(t0 + TT, L);
  Pack<T, N> zero;
  zero.zero();
  for (int b = b0; b < b1; ++b) {
    const int T_b = seq_len(lengths, b, L), te = min(t1, T_b);
    T *st = state ? state + (int64_t)b * (K - 1) * D + c : nullptr;
    // the input of position p >= 1 - K; before the start the state's rows, which this kernel replaces
    auto load = [&](Pack<T, N> &q, int p) {
      if (p >= 0)
        q.load_read_only(x.at(b, p, c), vec, have);
      else if (st)
        q.load(st + (int64_t)(p + K - 1) * D, vec, have);
      else
        q.zero();
    };
    if (t0 < te) {
      constexpr int H = (N + 1) / 2;
      Pack<T, N> first[K - 1], next[U];
      // rows [t, t + U) on their way: into this thread's own slots of shared memory (whole 16-byte
      // accesses), or into registers
      const T *xp = x.at(b, t0, c);  // the next row to request
      T *yp = y.at(b, t0, c);        // the next row to store
      auto request = [&](int t) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if constexpr (kAsync) {
            const uint32_t at = (uint32_t)(t + u - t0) % (kGroups * U) * (kConvThreads * 16);
            if (t + u < te) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + at), "l"(xp) : "memory");
          } else {
            next[u].load_read_only(xp, vec, t + u < te ? have : 0);
          }
          xp += x.ldl;
        }
        if constexpr (kAsync) asm volatile("cp.async.commit_group;" ::: "memory");
      };
#pragma unroll
      for (int g = 0; g < (kAsync ? kGroups - 1 : 1); ++g) request(t0 + g * U);
#pragma unroll
      for (int j = 0; j < K - 1; ++j) load(first[j], t0 - (K - 1) + j);
      float2 win[K - 1 + U][H];  // the last K - 1 inputs, then U new ones
#pragma unroll
      for (int j = 0; j < K - 1; ++j) first[j].pairs(win[j]);
      for (int t = t0; t < te; t += U) {
        if constexpr (kAsync) {
          request(t + (kGroups - 1) * U);
          asm volatile("cp.async.wait_group %0;" ::"n"(kGroups - 1) : "memory");
#pragma unroll
          for (int u = 0; u < U; ++u) {  // slots behind the end hold old rows: computed, not stored
            Pack<T, N> q = *reinterpret_cast<const Pack<T, N> *>(smem + (uint32_t)(t + u - t0) % (kGroups * U) * (kConvThreads * 16) + threadIdx.x * 16);
            q.pairs(win[K - 1 + u]);
          }
        } else {
#pragma unroll
          for (int u = 0; u < U; ++u) next[u].pairs(win[K - 1 + u]);
          request(t + U);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          Pack<T, N> out;
#pragma unroll
          for (int h = 0; h < H; ++h) {
            float2 acc = bs[h];
#pragma unroll
            for (int j = 0; j < K; ++j) acc = __ffma2_rn(w[h][j], win[u + j][h], acc);
            if (act) acc = silu2(acc);
            out.v[2 * h] = from_f<T>(acc.x);
            if (2 * h + 1 < N) out.v[2 * h + 1] = from_f<T>(acc.y);
          }
          if (t + u < te) out.store(yp, vec, have);
          yp += y.ldl;
        }
#pragma unroll
        for (int j = 0; j < K - 1; ++j)
#pragma unroll
          for (int h = 0; h < H; ++h) win[j][h] = win[U + j][h];
      }
    }
    for (int t = max(t0, te); t < t1; ++t) zero.store(y.at(b, t, c), vec, have);
    // only the first tile reads the state, so the thread that has read it may replace it
    if (tile == 0 && st && T_b > 0) {
      Pack<T, N> q[K - 1];
#pragma unroll
      for (int j = 0; j < K - 1; ++j) load(q[j], T_b - (K - 1) + j);
#pragma unroll
      for (int j = 0; j < K - 1; ++j) q[j].store(st + (int64_t)j * D, vec, have);
    }
  }
}

// ------------------------------------------------------------ selective scan, prompts
// h_t = exp(dt_t A) h_{t-1} + (dt_t x_t) B_t,  y_t = C_t . h_t + D x_t,  out = y silu(z).
// A channel's N states are spread over LPC lanes with NPT states each (zero-padded to NPT * LPC),
// which walk the sequence in double groups of 2 LPC tokens.  Lane q loads tokens q and LPC + q of
// a group straight from the rows of x, dt and z (any alignment; kScanAhead tokens before their
// use), forms softplus and dt * x for both in packed arithmetic and hands them to the others by
// shuffles; the sums over the states end in the token's lane again (transposed reduction: LPC
// partial sums exchange halves in log2(LPC) rounds), which gates and stores it.  So the
// per-channel work is done once, and only B and C, shared by all channels, go through shared
// memory, in fp32 tiles of 64 tokens.
// One bf16 sequence of 4096 tokens, 8192 channels, 16 states: 334 us.  Neither its bytes bound it
// (41 us) nor its 20 exponentials and reciprocals per token and channel (149 us at 16 a clock and
// SM), but the 9 instructions per state, at 0.4 of the issue rate with the 7 warps that an SM
// gets from one sequence; four sequences of 2048 tokens, twice the work, take 506 us.  Inputs staged
// through shared memory with softplus formed by the loading thread took 354 us; 16 instead of 32
// tokens ahead 368 us; two states per lane (twice the warps, narrower row accesses) 541 us; lanes
// that share the tokens instead, joined by shuffles, 394 us.
// Few channels leave schedulers without a warp: their sequences are cut into segments (a.segs > 1).
// A first launch (ENDS) runs all but the last segment from zero, without outputs, and leaves their
// end states and sums of dt; the second starts each segment from the state that these lead to, since
// the decay over a segment is exp(A sum dt).
template <class T>
struct ScanArgs {
  Rows<const T> x, dt, bm, cm, z;
  Rows<T> out;
  const float *A, *skip, *dt_bias;
  float *state;
  const int *lengths;
  int L, D, N, softplus, vec_bc, chunks;
  // sequences cut into segments of seg tokens (k_ssm_scan): the state at the start of the first, and
  // for each but the last its end state from zero (of the first: from that start) and its sum of dt
  int segs, seg;
  int64_t rows;  // batch * channels
  float *start, *ends, *sums;
};

// The hardware exponential is 2e-8 too small on average where decays matter (arguments of -0.001 to
// -0.5), which a state adds up over as many tokens as it remembers.  2^2.9e-8 puts that back in the
// FMA that forms the argument: mean error 2e-9 instead of -2e-8, states of 73 to 4000 tokens off by
// 2e-7 to 6e-7 instead of 5e-7 to 15e-7 (relative norm; 6e-7 with expf).  A step of 0 still decays by
// exactly 1, to which 2^2.9e-8 rounds.  The bias is this chip's, found by measurement: on another it has to be
// measured again.
constexpr float kEx2Shift = 2.9e-8f;

constexpr int kScanThreads = 128, kScanAhead = 32;

template <int NPT, int LPC>
struct ScanShape {
  static constexpr int NP = NPT * LPC;              // padded states per channel
  static constexpr int CT = kScanThreads / LPC;     // channels per block
  static constexpr int TT = 64;                     // tokens per tile of B and C
  static constexpr int G = 2 * LPC;                 // tokens per double group
  static constexpr int PF = G >= kScanAhead ? 1 : kScanAhead / G;  // double groups ahead
  static constexpr int BV = NP >= 8 ? 8 : NP;       // states per access of B and C
  static constexpr int BITEMS = TT * (NP / BV);
  static constexpr int BIPT = (BITEMS + kScanThreads - 1) / kScanThreads;
  static constexpr int SMEM = 2 * TT * NP * 4;
  // Blocks per SM that the registers allow: 16 states, 4 sequences: 506 us, with 2 blocks 631.  Up to 8 states the
  // rows ahead (PF) do not fit under that cap: 130 to 390 bytes a thread are spilled
  static constexpr int BLOCKS = NP > 16 ? 2 : 4;
};

// A in powers of two; an infinite one times a step of 0, as behind the end, is 0 and not NaN.
__device__ __forceinline__ float rate2(float A) {
  A *= kLog2e;
  return isinf(A) ? copysignf(3.4e38f, A) : A;
}

// h 2^e for the e of a whole segment.  Token by token a state that is 0 or infinite stays so, and one
// that underflows or overflows halfway to its value does not exist: hence four steps, each of which
// stays in range where the result does.
__device__ __forceinline__ float decayed(float h, float e) {
  if (h == 0.f || isinf(h)) return h;
  const float f = ex2_approx(0.25f * e);
  return h * f * f * f * f;
}

template <class T, int NPT, int LPC, bool ENDS>
__global__ void __launch_bounds__(kScanThreads, ScanShape<NPT, LPC>::BLOCKS) k_ssm_scan(const __grid_constant__ ScanArgs<T> a) {
  using S = ScanShape<NPT, LPC>;
  constexpr int NP = S::NP, CT = S::CT, TT = S::TT, BV = S::BV, BIPT = S::BIPT, PF = S::PF, G = S::G;
  constexpr int H = NPT / 2;  // pairs of states, for packed arithmetic
  static_assert(TT % (PF * G) == 0, "whole rounds of groups per tile");
  extern __shared__ __align__(16) float smem[];
  float *sb = smem, *sc = smem + TT * NP;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x;
  const int B = (int)(a.rows / a.D);
  const int s = blockIdx.x / a.chunks / B;
  const int64_t b = blockIdx.x / a.chunks % B;
  const int c = (int)(blockIdx.x % a.chunks) * CT + tid / LPC;
  const int q = tid % LPC, n0 = q * NPT;
  const int t_lo = s * a.seg, len = seq_len(a.lengths, b, a.L), T_b = min(len, t_lo + a.seg);
  const bool live = c < a.D;
  const int64_t at0 = (b * a.D + c) * (int64_t)a.N + n0, all = a.rows * a.N;

  float A2[NPT], h[NPT];
#pragma unroll
  for (int i = 0; i < NPT; ++i) {
    const bool on = live && n0 + i < a.N;
    A2[i] = rate2(on ? a.A[(int64_t)c * a.N + n0 + i] : 0.f);
    h[i] = 0.f;
    if (!on) continue;
    if constexpr (ENDS) {
      if (s == 0 && a.state) a.start[at0 + i] = h[i] = a.state[at0 + i];
    } else if (s == 0) {
      if (a.state) h[i] = a.segs > 1 ? a.start[at0 + i] : a.state[at0 + i];
    } else {
      h[i] = a.ends[at0 + i];
      for (int e = 1; e < s; ++e)
        h[i] = decayed(h[i], a.sums[e * a.rows + b * a.D + c] * A2[i]) + a.ends[e * all + at0 + i];
    }
  }
  float dsum = 0.f;
  const float bias = live && a.dt_bias ? a.dt_bias[c] : 0.f, skip = live && a.skip ? a.skip[c] : 0.f;

  // this lane's rows: tokens q, q + LPC, ...
  const T *px = a.x.at(b, t_lo + q, c), *pd = a.dt.at(b, t_lo + q, c), *pz = a.z.p ? a.z.at(b, t_lo + q, c) : px;
  T *po = a.out.at(b, t_lo + q, c);
  const int64_t sx = LPC * a.x.ldl, sd = LPC * a.dt.ldl, sz = LPC * (a.z.p ? a.z.ldl : a.x.ldl), so = LPC * a.out.ldl;
  const int mine = live ? T_b - q : 0;  // a group that starts at t holds a token of this lane if t < mine
  T nx[PF][2], nd[PF][2], nz[PF][2];
  auto fetch = [&](int k, int t) {
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const bool on = t + w * LPC < mine;
      nx[k][w] = on ? *px : from_f<T>(0.f);
      nd[k][w] = on ? *pd : from_f<T>(0.f);
      if constexpr (!ENDS) nz[k][w] = on ? *pz : from_f<T>(0.f), pz += sz;
      px += sx, pd += sd;
    }
  };
  Pack<T, BV> nb[BIPT], nc[BIPT];
  auto fetch_bc = [&](int t0) {
#pragma unroll
    for (int i = 0; i < BIPT; ++i) {
      const int it = tid + i * kScanThreads, t = t0 + it / (NP / BV), n = it % (NP / BV) * BV;
      const int have = it < S::BITEMS && t < T_b ? a.N - n : 0;
      nb[i].load_read_only(a.bm.at(b, t, n), a.vec_bc, have);
      if constexpr (!ENDS) nc[i].load_read_only(a.cm.at(b, t, n), a.vec_bc, have);
    }
  };
#pragma unroll
  for (int k = 0; k < PF; ++k) fetch(k, t_lo + k * G);
  fetch_bc(t_lo);
  for (int t0 = t_lo; t0 < T_b; t0 += TT) {
    if (t0 > t_lo) __syncthreads();  // the tile before has been read
#pragma unroll
    for (int i = 0; i < BIPT; ++i) {
      const int it = tid + i * kScanThreads, at = it / (NP / BV) * NP + it % (NP / BV) * BV;
      if (it < S::BITEMS) {
#pragma unroll
        for (int e = 0; e < BV; ++e) {
          sb[at + e] = to_f(nb[i].v[e]);
          if constexpr (!ENDS) sc[at + e] = to_f(nc[i].v[e]);
        }
      }
    }
    __syncthreads();
    fetch_bc(t0 + TT);
#pragma unroll 1
    for (int g = 0; g < TT && t0 + g < T_b; g += PF * G) {
#pragma unroll
      for (int k = 0; k < PF; ++k) {
        const int t = t0 + g + k * G;
        const float2 x = make_float2(to_f(nx[k][0]), to_f(nx[k][1]));
        const float2 z = ENDS ? x : make_float2(to_f(nz[k][0]), to_f(nz[k][1]));
        float2 d = __fadd2_rn(make_float2(to_f(nd[k][0]), to_f(nd[k][1])), make_float2(bias, bias));
        fetch(k, t + PF * G);
        if (a.softplus) d = softplus2(d);
        const bool on0 = t < mine, on1 = t + LPC < mine;
        d = make_float2(on0 ? d.x : 0.f, on1 ? d.y : 0.f);  // behind the end: a = 1, no input
        if constexpr (ENDS) dsum += d.x + d.y;
        const float2 u = __fmul2_rn(d, x);
        float ys[2];
#pragma unroll
        for (int w = 0; w < 2; ++w) {
          float p[LPC];
#pragma unroll
          for (int j = 0; j < LPC; ++j) {
            const float dj = __shfl_sync(0xffffffffu, w ? d.y : d.x, j, LPC);
            const float uj = __shfl_sync(0xffffffffu, w ? u.y : u.x, j, LPC);
            const float *bp = sb + (g + k * G + w * LPC + j) * NP + n0, *cp = sc + (g + k * G + w * LPC + j) * NP + n0;
            if constexpr (NPT == 1) {
              h[0] = fmaf(ex2_approx(fmaf(dj, A2[0], kEx2Shift)), h[0], uj * bp[0]);
              if constexpr (!ENDS) p[j] = cp[0] * h[0];
            } else {
              const float2 d2 = make_float2(dj, dj), u2 = make_float2(uj, uj);
              Pack<float, NPT> Bv, Cv;
              Bv.load_all(bp);
              if constexpr (!ENDS) Cv.load_all(cp);
              float2 acc = make_float2(0.f, 0.f);
#pragma unroll
              for (int i = 0; i < H; ++i) {
                const float2 e = __ffma2_rn(d2, make_float2(A2[2 * i], A2[2 * i + 1]), make_float2(kEx2Shift, kEx2Shift));
                float2 hv = make_float2(h[2 * i], h[2 * i + 1]);
                hv = __ffma2_rn(make_float2(ex2_approx(e.x), ex2_approx(e.y)), hv,
                                __fmul2_rn(u2, make_float2(Bv.v[2 * i], Bv.v[2 * i + 1])));
                h[2 * i] = hv.x, h[2 * i + 1] = hv.y;
                if constexpr (!ENDS) {
                  const float2 C2 = make_float2(Cv.v[2 * i], Cv.v[2 * i + 1]);
                  acc = i ? __ffma2_rn(C2, hv, acc) : __fmul2_rn(C2, hv);
                }
              }
              if constexpr (!ENDS) p[j] = acc.x + acc.y;
            }
          }
          if constexpr (!ENDS) {
#pragma unroll
            for (int o = LPC / 2; o; o >>= 1) {
              const bool up = q & o;
#pragma unroll
              for (int j = 0; j < o; ++j) {
                const float keep = up ? p[j + o] : p[j], give = up ? p[j] : p[j + o];
                p[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
              }
            }
            ys[w] = p[0];
          }
        }
        if constexpr (ENDS) continue;
        float2 y = __ffma2_rn(make_float2(skip, skip), x, make_float2(ys[0], ys[1]));
        if (a.z.p) y = __fmul2_rn(y, silu2(z));
        if (on0) *po = from_f<T>(y.x);
        po += so;
        if (on1) *po = from_f<T>(y.y);
        po += so;
      }
    }
  }
  if constexpr (ENDS) {
#pragma unroll
    for (int o = 1; o < LPC; o <<= 1) dsum += __shfl_xor_sync(0xffffffffu, dsum, o);
    if (live && q == 0) a.sums[s * a.rows + b * a.D + c] = dsum;
#pragma unroll
    for (int i = 0; i < NPT; ++i)
      if (live && n0 + i < a.N) a.ends[s * all + at0 + i] = h[i];
    return;
  }
  if (live) {  // outputs behind the end are zeros
    const int t_hi = min(a.L, t_lo + a.seg);
    for (int t = max(len, t_lo) + q; t < t_hi; t += LPC) *a.out.at(b, t, c) = from_f<T>(0.f);
  }
  if (a.state && live && len > 0 && s == a.segs - 1) {
#pragma unroll
    for (int i = 0; i < NPT; ++i)
      if (n0 + i < a.N) a.state[at0 + i] = h[i];
  }
}

// ------------------------------------------------------------ selective scan, single tokens
// One token per sequence: the state is read and written once, which bounds it.  LPC lanes of 4
// states per channel; a thread keeps its row of A for kStepBatch sequences and takes R of them at
// a time: lane q of a channel forms softplus, dt * x and the gate of sequence q % R, the others
// get them by shuffles, and the sums over the states end in that lane again (transposed
// reduction).  With VEC (N a multiple of 4, aligned rows) the states of the next kStepAhead - 1
// groups are on their way into the thread's own slots of shared memory, and the next group's
// inputs into registers, while one group is computed.  256 sequences of 8192 bf16 channels, 16
// states: 64 us, 4.4 TB/s; every lane forming softplus and gate for itself, one sequence at a time,
// took 104 us, and 3 or 4 blocks of 256 threads per SM, which spill, 88 and 127 us.  At the 5 blocks
// that suit this case fp32 inputs spill about 100 bytes a thread (78 us; floor 46), unaligned bf16 ones 80.
constexpr int kStepThreads = 128, kStepAhead = 2, kStepBatch = 16;

template <class T, bool VEC, int LPC>
__global__ void __launch_bounds__(kStepThreads, 5) k_ssm_step(const __grid_constant__ ScanArgs<T> a, int B) {
  constexpr int R = LPC < 4 ? LPC : 4;
  __shared__ __align__(16) char smem[VEC ? kStepAhead * R * kStepThreads * 16 : 16];
  pdl_trigger();
  pdl_wait();
  const int q = threadIdx.x % LPC, n0 = q * 4, my = q % R;
  const int c = (int)(blockIdx.x % a.chunks) * (kStepThreads / LPC) + threadIdx.x / LPC;
  const int b0 = (int)(blockIdx.x / a.chunks) * kStepBatch, b1 = min(b0 + kStepBatch, B);
  const bool live = c < a.D;
  const int have = live ? min(4, a.N - n0) : 0;
  // four states, or inputs of them: with VEC all or none of them exist
  auto load4 = [&](auto &p, const auto *src, bool on) {
    if constexpr (VEC) {
      p.zero();
      if (on && have > 0) p.load_all(src);
    } else {
      p.load(src, false, on ? have : 0);
    }
  };
  Pack<float, 4> A;
  load4(A, a.A + (int64_t)c * a.N + n0, true);
#pragma unroll
  for (int i = 0; i < 4; ++i) A.v[i] = rate2(A.v[i]);
  const float bias = live && a.dt_bias ? a.dt_bias[c] : 0.f, skip = live && a.skip ? a.skip[c] : 0.f;
  const int64_t row = (int64_t)a.D * a.N;
  float *st = a.state ? a.state + b0 * row + (int64_t)c * a.N + n0 : nullptr;
  const float *ahead = st;  // the next state to request
  const uint32_t slot = (uint32_t)__cvta_generic_to_shared(smem) + threadIdx.x * 16;
  int ring = 0;  // the group of slots requested next
  auto request = [&](int b) {
    if constexpr (VEC) {
      if (st && have > 0) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (b + r < b1)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(slot + (ring * R + r) * (kStepThreads * 16)),
                         "l"(ahead) : "memory");
          ahead += row;
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      ring = ring + 1 == kStepAhead ? 0 : ring + 1;
    }
  };
  const T *px = a.x.at(b0 + my, 0, c), *pd = a.dt.at(b0 + my, 0, c), *pz = a.z.p ? a.z.at(b0 + my, 0, c) : nullptr;
  const T *pb = a.bm.at(b0, 0, n0), *pc = a.cm.at(b0, 0, n0);
  T *po = a.out.at(b0 + my, 0, c);
  struct In {
    Pack<T, 4> bm[R], cm[R];
    T x, d, z;
    bool on;  // this lane's sequence has a token
  } next;
  auto fetch = [&](In &in, int b) {  // sequences b .. b + R - 1; b rises by R from call to call
#pragma unroll
    for (int r = 0; r < R; ++r) {
      load4(in.bm[r], pb, b + r < b1);
      load4(in.cm[r], pc, b + r < b1);
      pb += a.bm.ldb, pc += a.cm.ldb;
    }
    in.on = live && b + my < b1 && (!a.lengths || a.lengths[b + my] > 0);
    in.x = in.on ? *px : from_f<T>(0.f);
    in.d = in.on ? *pd : from_f<T>(0.f);
    in.z = in.on && pz ? *pz : from_f<T>(0.f);
    px += R * a.x.ldb, pd += R * a.dt.ldb;
    if (pz) pz += R * a.z.ldb;
  };
#pragma unroll
  for (int k = 0; k < kStepAhead - 1; ++k) request(b0 + k * R);
  fetch(next, b0);
  int used = 0;  // the group of slots read next
  for (int b = b0; b < b1; b += R) {
    request(b + (kStepAhead - 1) * R);
    const In in = next;
    fetch(next, b + R);
    float d = to_f(in.d) + bias;
    if (a.softplus) d = softplus(d);
    if (!in.on) d = 0.f;
    const float u = d * to_f(in.x);
    if constexpr (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(kStepAhead - 1) : "memory");
    float y[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      Pack<float, 4> h;
      if constexpr (VEC) {
        h.zero();
        if (st && have > 0 && b + r < b1)
          h.load_all(reinterpret_cast<const float *>(smem + (used * R + r) * (kStepThreads * 16) + threadIdx.x * 16));
      } else {
        h.load(st, false, st && b + r < b1 ? have : 0);
      }
      const float dr = __shfl_sync(0xffffffffu, d, r, R), ur = __shfl_sync(0xffffffffu, u, r, R);
      const bool on = __shfl_sync(0xffffffffu, in.on, r, R);
      y[r] = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // a sequence without a token may hold anything in its row of B and C
        h.v[i] = fmaf(ex2_approx(fmaf(dr, A.v[i], kEx2Shift)), h.v[i], ur * to_f(in.bm[r].v[i]));
        y[r] = fmaf(to_f(in.cm[r].v[i]), h.v[i], y[r]);
      }
      if (st) {
        if (on) {
          if constexpr (VEC) {
            if (have > 0) *reinterpret_cast<float4 *>(st) = *reinterpret_cast<const float4 *>(h.v);
          } else {
            h.store(st, false, have);
          }
        }
        st += row;
      }
    }
    used = used + 1 == kStepAhead ? 0 : used + 1;
#pragma unroll
    for (int o = R / 2; o; o >>= 1) {
#pragma unroll
      for (int j = 0; j < o; ++j) {
        const bool up = q & o;
        const float keep = up ? y[j + o] : y[j], give = up ? y[j] : y[j + o];
        y[j] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    }
#pragma unroll
    for (int o = R; o < LPC; o <<= 1) y[0] += __shfl_xor_sync(0xffffffffu, y[0], o);
    if (q < R && live && b + my < b1) {
      float o = fmaf(skip, to_f(in.x), y[0]);
      if (a.z.p) o *= silu(to_f(in.z));
      *po = from_f<T>(in.on ? o : 0.f);
    }
    po += R * a.out.ldb;
  }
}

template <class K, class A>
static int launch_scan_k(K kern, const A &a, int64_t blocks, int threads, int smem, cudaStream_t st) {
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return fail(TESM_ELAUNCH, std::string("ssm_scan: ") + cudaGetErrorString(e));
  }
  return launch_k("ssm_scan", kern, dim3((unsigned)blocks), dim3(threads), smem, st, a);
}

template <class T, int NPT, int LPC>
static int launch_scan(ScanArgs<T> a, int64_t B, cudaStream_t st) {
  using S = ScanShape<NPT, LPC>;
  a.chunks = (int)ceil_div(a.D, S::CT);  // blocks as in scan_blocks
  if (a.segs > 1) {
    const int rc = launch_scan_k(k_ssm_scan<T, NPT, LPC, true>, a, B * a.chunks * (a.segs - 1), kScanThreads, S::SMEM, st);
    if (rc) return rc;
  }
  return launch_scan_k(k_ssm_scan<T, NPT, LPC, false>, a, B * a.chunks * a.segs, kScanThreads, S::SMEM, st);
}

template <class T, int LPC>
static int launch_step(ScanArgs<T> a, int64_t B, cudaStream_t st) {
  a.chunks = (int)ceil_div(a.D, kStepThreads / LPC);
  const dim3 grid((unsigned)(a.chunks * ceil_div(B, kStepBatch))), block(kStepThreads);
  const bool vec = a.N % 4 == 0 && a.vec_bc && (((uintptr_t)a.A | (uintptr_t)a.state) & 15) == 0;
  return vec ? launch_k("ssm_scan", k_ssm_step<T, true, LPC>, grid, block, 0, st, a, (int)B)
             : launch_k("ssm_scan", k_ssm_step<T, false, LPC>, grid, block, 0, st, a, (int)B);
}

static int pad_states(int64_t N) {
  int np = 1;
  while (np < N) np <<= 1;
  return np;
}

// Blocks of the prompt kernel, and how many of them an SM holds at once (as in ScanShape).
static int64_t scan_blocks(int64_t B, int64_t D, int np) { return B * ceil_div(D, kScanThreads / (np > 4 ? np / 4 : 1)); }
static int scan_resident(int np) { return np > 16 ? 2 : 4; }

// Tokens per segment.  A warp's step takes about 65 ns however few warps there are, and 36 ns of its
// scheduler where there are many; a second pass adds 22.  So with under one block (a warp per
// scheduler) per SM cutting the sequences wins (8192 tokens, 2048 channels, 16 states: 544 us whole, 281
// in 4, 248 in 8, 220 in 16 segments; 512 tokens: 22 in 4, 29 whole).  The most blocks per SM at which
// it does, times 8, by sweeps of 1, 2, 4, ... 128 states over 0.12 to 3.5 blocks per SM and 512 to 8192
// tokens, both types (time whole / time cut):
//   1 state      18, from 4096 tokens on 20 (2.25: 1.04 to 1.11, 3: 0.86 to 0.94)
//   2 states     14 (1.75: 1.2 to 1.3)
//   4 to 16       7 (0.87: 16 states, 4096 tokens on 1.2 to 1.3; shorter ones 0.85 to 0.94 while their inputs
//                 are in L2, 1.04 to 1.17 from memory; more blocks: 8192 channels 334 us whole, 402 in 2)
//   above 16      4 below 4096 tokens (0.5: 1.1 to 1.5, 0.6: 0.9 to 1.16, 0.87: 0.6 to 0.8), 5 and from 8192 on
//                 6 else (0.75 at 8192: 0.9 to 1.2)
// Segments: as many as fit the SMs at once, up to 32, and 16 at least where they need not all fit: a
// few whole rounds of short segments lose little.  At 2 blocks an SM and under 4096 tokens they do
// (64 states, 0.25 blocks per SM, 2048 tokens: 40 us in 8, 49 in 16, 90 whole).  Segments have 128
// tokens at least, and under four of them do not pay for the second launch.
static int64_t scan_segment(int64_t B, int64_t L, int64_t D, int64_t N) {
  const int np = pad_states(N);
  const int64_t sm = sm_count(), blocks = scan_blocks(B, D, np);  // B, D > 0
  const int limit = np == 1   ? (L < 4096 ? 18 : 20)
                    : np == 2 ? 14
                    : np <= 16 ? 7
                               : (L < 4096 ? 4 : L < 8192 ? 5 : 6);
  if (8 * blocks > limit * sm) return L;
  const bool fit = np > 16 && L < 4096;
  const int64_t room = scan_resident(np) * sm / blocks, most = room > 32 ? 32 : !fit && room < 16 ? 16 : room;
  const int64_t s = L / 128 < most ? L / 128 : most;
  return s < 4 ? L : round_up(ceil_div(L, s), kScanAhead);
}
static int64_t scan_ws_floats(int64_t B, int64_t L, int64_t D, int64_t N) {
  if (B == 0 || D == 0 || L <= 1) return 0;
  const int64_t S = ceil_div(L, scan_segment(B, L, D, N));
  return S > 1 ? S * B * D * N + (S - 1) * B * D : 0;
}

template <class T>
static int ssm_scan_t(ScanArgs<T> a, int64_t B, float *ws, cudaStream_t st) {
  const int np = pad_states(a.N);
  if (a.L == 1) {
    switch (np <= 4 ? 1 : np / 4) {
      case 1: return launch_step<T, 1>(a, B, st);
      case 2: return launch_step<T, 2>(a, B, st);
      case 4: return launch_step<T, 4>(a, B, st);
      case 8: return launch_step<T, 8>(a, B, st);
      case 16: return launch_step<T, 16>(a, B, st);
      default: return launch_step<T, 32>(a, B, st);
    }
  }
  a.rows = B * a.D;
  a.seg = (int)scan_segment(B, a.L, a.D, a.N);
  a.segs = (int)ceil_div(a.L, a.seg);
  a.start = ws;
  a.ends = ws + a.rows * a.N;
  a.sums = ws + a.segs * a.rows * a.N;
  switch (np) {
    case 1: return launch_scan<T, 1, 1>(a, B, st);
    case 2: return launch_scan<T, 2, 1>(a, B, st);
    case 4: return launch_scan<T, 4, 1>(a, B, st);
    case 8: return launch_scan<T, 4, 2>(a, B, st);
    case 16: return launch_scan<T, 4, 4>(a, B, st);
    case 32: return launch_scan<T, 4, 8>(a, B, st);
    case 64: return launch_scan<T, 4, 16>(a, B, st);
    default: return launch_scan<T, 4, 32>(a, B, st);
  }
}

template <class T, int N, int U>
static int launch_conv(Rows<const T> x, int64_t B, int L, int D, int K, int vec, const float *w, const float *bias,
                       T *state, const int *lengths, int act, Rows<T> y, cudaStream_t st) {
  const int chunks = (int)ceil_div(D, kConvThreads * N);
  int TT = 64;  // tokens per tile: shorter while the blocks do not fill the SMs
  while (TT > 8 && B * chunks * ceil_div(L, TT) < 8 * (int64_t)sm_count()) TT >>= 1;
  const int tiles = (int)ceil_div(L, TT);
  // sequences per thread: several where a tile is short, so that the weights are loaded less often
  const int nb = L < 4 && B * chunks >= kConvBatch * 2 * (int64_t)sm_count() ? kConvBatch : 1;
  const dim3 grid((unsigned)(ceil_div(B, nb) * chunks * tiles)), block(kConvThreads);
#define TESM_CONV(KK)                                                                                            \
  case KK:                                                                                                       \
    return launch_k("causal_conv", k_causal_conv<T, N, KK, U>, grid, block, 0, st, x, (int)B, L, D, TT, nb, vec, w, bias, \
                    state, lengths, act, y, chunks, tiles)
  switch (K) {
    TESM_CONV(2);
    TESM_CONV(3);
    TESM_CONV(4);
    TESM_CONV(5);
    TESM_CONV(6);
    TESM_CONV(7);
    TESM_CONV(8);
  }
#undef TESM_CONV
  return fail(TESM_EUNSUPPORTED, "causal_conv: kernel width");
}

template <class T>
static int causal_conv_t(const void *x, int64_t ldb, int64_t ldl, int64_t B, int64_t L, int64_t D, int64_t K,
                         const float *w, const float *bias, void *state, const int *lengths, int act, void *y,
                         int64_t ldyb, int64_t ldyl, cudaStream_t st) {
  const Rows<const T> rx{(const T *)x, ldb, ldl};
  const Rows<T> ry{(T *)y, ldyb, ldyl};
  const uint64_t bits = (uintptr_t)x | (uintptr_t)y | (uintptr_t)state |
                        (uint64_t)((ldb | ldl | ldyb | ldyl | (state ? D : 0)) * (int64_t)sizeof(T));
  constexpr int N = 16 / sizeof(T);
  if (bits % 16 == 0 && L >= 4 && D % N == 0)
    return launch_conv<T, N, 2>(rx, B, (int)L, (int)D, (int)K, 1, w, bias, (T *)state, lengths, act, ry, st);
  if (bits % 16 == 0 && L >= 4)
    return launch_conv<T, N, 4>(rx, B, (int)L, (int)D, (int)K, 1, w, bias, (T *)state, lengths, act, ry, st);
  if (bits % 16 == 0)
    return launch_conv<T, N, 1>(rx, B, (int)L, (int)D, (int)K, 1, w, bias, (T *)state, lengths, act, ry, st);
  return launch_conv<T, 1, 4>(rx, B, (int)L, (int)D, (int)K, 0, w, bias, (T *)state, lengths, act, ry, st);
}

}  // namespace tesm

extern "C" int tesm_b200_causal_conv(const void *x, int dtype, int64_t ldxb, int64_t ldxl, int64_t B, int64_t L,
                                     int64_t D, int64_t K, const float *weight, const float *bias, void *state,
                                     const int32_t *lengths, int silu, void *out, int64_t ldob, int64_t ldol,
                                     tesm_stream_t stream) {
  using namespace tesm;
  if (dtype != TESM_F32 && dtype != TESM_BF16) return fail(TESM_EDTYPE, "causal_conv: dtype");
  TESM_REQUIRE(B >= 0 && L >= 0 && D >= 0 && B < (1ll << 31) && L < (1ll << 30) && D < (1ll << 30),
               "causal_conv: bad shape");
  if (K < 2 || K > 8) return fail(TESM_EUNSUPPORTED, "causal_conv: kernel width 2 to 8");
  if (B == 0 || L == 0 || D == 0) return TESM_OK;
  TESM_REQUIRE(x && weight && out, "causal_conv: null pointer");
  const int64_t chunks = ceil_div(D, kConvThreads);  // products below 2^54 and, behind the first check, 2^58
  TESM_REQUIRE(B * chunks < (1ll << 31) && B * chunks * ceil_div(L, 8) < (1ll << 31), "causal_conv: too many blocks");
  const int64_t es = dtype == TESM_BF16 ? 2 : 4;
  TESM_REQUIRE(ldxb >= 0 && ldxl >= 0 && ldob >= 0 && ldol >= 0, "causal_conv: negative stride");
  TESM_REQUIRE(!self_overlap(B, L, D, ldob, ldol), "causal_conv: out overlaps itself");
  const Span so = span3(out, B, L, D, ldob, ldol, es), ss = span1(state, B * (K - 1) * D * es);
  for (const Span &r : {span3(x, B, L, D, ldxb, ldxl, es), span1(weight, D * K * 4), span1(bias, D * 4),
                        span1(lengths, B * 4)})
    TESM_REQUIRE(!so.meets(r) && !ss.meets(r), "causal_conv: out or state shares memory with an input");
  TESM_REQUIRE(!so.meets(ss), "causal_conv: out shares memory with state");
  cudaStream_t st = (cudaStream_t)stream;
  return dtype == TESM_BF16 ? causal_conv_t<__nv_bfloat16>(x, ldxb, ldxl, B, L, D, K, weight, bias, state, lengths, silu,
                                                           out, ldob, ldol, st)
                            : causal_conv_t<float>(x, ldxb, ldxl, B, L, D, K, weight, bias, state, lengths, silu, out,
                                                   ldob, ldol, st);
}

namespace tesm {
template <class T>
static int ssm_scan_c(const void *x, const void *dt, const void *bm, const void *cm, const void *z, void *out,
                      const int64_t *ld, int64_t B, ScanArgs<T> a, float *ws, cudaStream_t st) {
  a.x = {(const T *)x, ld[0], ld[1]};
  a.dt = {(const T *)dt, ld[2], ld[3]};
  a.bm = {(const T *)bm, ld[4], ld[5]};
  a.cm = {(const T *)cm, ld[6], ld[7]};
  a.z = {(const T *)z, ld[8], ld[9]};
  a.out = {(T *)out, ld[10], ld[11]};
  const int64_t es = sizeof(T);
  uint64_t bc = (uintptr_t)bm | (uintptr_t)cm;
  for (int i : {4, 5, 6, 7}) bc |= (uint64_t)(ld[i] * es);
  a.vec_bc = bc % 16 == 0;
  return ssm_scan_t<T>(a, B, ws, st);
}
// Sizes of which no product leaves 64 bits and no grid 31.
static bool scan_shape_ok(int64_t B, int64_t L, int64_t D) {
  return B >= 0 && L >= 0 && D >= 0 && B < (1ll << 31) && L < (1ll << 30) && D < (1ll << 30) &&
         B * ceil_div(D, 4) < (1ll << 31);
}
}  // namespace tesm

extern "C" int tesm_b200_ssm_scan_workspace(int64_t B, int64_t L, int64_t D, int64_t N, int64_t *bytes_out) {
  using namespace tesm;
  TESM_REQUIRE(bytes_out && scan_shape_ok(B, L, D) && N >= 1 && N <= 128, "ssm_scan_workspace: bad shape");
  *bytes_out = 4 * scan_ws_floats(B, L, D, N);
  return TESM_OK;
}

extern "C" int tesm_b200_ssm_scan(const void *x, const void *dt, const void *bm, const void *cm, const void *z,
                                  void *out, const int64_t *strides, int dtype, int64_t B, int64_t L, int64_t D,
                                  int64_t N, const float *A, const float *skip, const float *dt_bias, int softplus,
                                  float *state, const int32_t *lengths, void *ws, int64_t ws_bytes, tesm_stream_t stream) {
  using namespace tesm;
  if (dtype != TESM_F32 && dtype != TESM_BF16) return fail(TESM_EDTYPE, "ssm_scan: dtype");
  TESM_REQUIRE(scan_shape_ok(B, L, D), "ssm_scan: bad shape");
  if (N < 1 || N > 128) return fail(TESM_EUNSUPPORTED, "ssm_scan: 1 to 128 states per channel");
  if (B == 0 || L == 0 || D == 0) return TESM_OK;
  TESM_REQUIRE(x && dt && bm && cm && out && A && strides, "ssm_scan: null pointer");
  const int64_t es = dtype == TESM_BF16 ? 2 : 4, *ld = strides;
  for (int i = 0; i < 12; ++i) TESM_REQUIRE(ld[i] >= 0, "ssm_scan: negative stride");
  TESM_REQUIRE(!self_overlap(B, L, D, ld[10], ld[11]), "ssm_scan: out overlaps itself");
  const int64_t need = 4 * scan_ws_floats(B, L, D, N);
  TESM_REQUIRE(need == 0 || (ws && ws_bytes >= need && ((uintptr_t)ws & 15) == 0), "ssm_scan: workspace");
  const Span so = span3(out, B, L, D, ld[10], ld[11], es), ss = span1(state, B * D * N * 4);
  const Span sw = need ? span1(ws, need) : Span{};
  for (const Span &r : {span3(x, B, L, D, ld[0], ld[1], es), span3(dt, B, L, D, ld[2], ld[3], es),
                        span3(bm, B, L, N, ld[4], ld[5], es), span3(cm, B, L, N, ld[6], ld[7], es),
                        span3(z, B, L, D, ld[8], ld[9], es), span1(A, D * N * 4), span1(skip, D * 4),
                        span1(dt_bias, D * 4), span1(lengths, B * 4)})
    TESM_REQUIRE(!so.meets(r) && !ss.meets(r) && !sw.meets(r), "ssm_scan: out, state or workspace shares memory with an input");
  TESM_REQUIRE(!so.meets(ss) && !so.meets(sw) && !ss.meets(sw), "ssm_scan: out, state and workspace share memory");
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TESM_BF16) {
    ScanArgs<__nv_bfloat16> a = {};
    a.A = A, a.skip = skip, a.dt_bias = dt_bias, a.state = state, a.lengths = lengths;
    a.L = (int)L, a.D = (int)D, a.N = (int)N, a.softplus = softplus;
    return ssm_scan_c<__nv_bfloat16>(x, dt, bm, cm, z, out, strides, B, a, (float *)ws, st);
  }
  ScanArgs<float> a = {};
  a.A = A, a.skip = skip, a.dt_bias = dt_bias, a.state = state, a.lengths = lengths;
  a.L = (int)L, a.D = (int)D, a.N = (int)N, a.softplus = softplus;
  return ssm_scan_c<float>(x, dt, bm, cm, z, out, strides, B, a, (float *)ws, st);
}
