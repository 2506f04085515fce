// Beam search: one selection step over beams and vocabulary, and the recurrent caches following
// the chosen beams.
#include "common.cuh"

#include <cfloat>

namespace tesm {

constexpr int kMaxBeams = 32;  // one lane per kept candidate

// ------------------------------------------------------------ candidate lists
// A warp holds its best candidates sorted, one per lane: larger values first, equal values by
// lower index.  Value type V is float (raw logits of one row) or double (keys across rows).
constexpr int kNoIndex = 0x7fffffff;

template <class V>
__device__ __forceinline__ bool better(V a, int ia, V b, int ib) {
  return a > b || (a == b && ia < ib);
}

// Insert (x, ix), the same on all lanes, into the warp's list of the K best.
template <class V>
__device__ __forceinline__ void list_insert(V &v, int &i, V x, int ix, int lane) {
  const unsigned ahead = __ballot_sync(0xffffffffu, better(v, i, x, ix));
  const int pos = __popc(ahead);  // the list is sorted: the better entries are its first lanes
  const V pv = __shfl_up_sync(0xffffffffu, v, 1);
  const int pi = __shfl_up_sync(0xffffffffu, i, 1);
  if (lane == pos) v = x, i = ix;
  if (lane > pos) v = pv, i = pi;
}

// The 32 best of two sorted lists: the larger of a[l] and b[31 - l] is a bitonic sequence, sorted
// by five compare-exchange steps.
template <class V>
__device__ __forceinline__ void list_merge(V &v, int &i, V bv, int bi, int lane) {
  bv = __shfl_sync(0xffffffffu, bv, 31 - lane);
  bi = __shfl_sync(0xffffffffu, bi, 31 - lane);
  if (better(bv, bi, v, i)) v = bv, i = bi;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const V ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, i, o);
    const bool other = better(ov, oi, v, i);
    if (other != ((lane & o) != 0)) v = ov, i = oi;
  }
}

// Order-preserving map of a float to an unsigned (larger floats, larger words; never 0 here since
// no NaN reaches it).
__device__ __forceinline__ unsigned order_word(float x) {
  const unsigned b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// ------------------------------------------------------------ rows: softmax statistics and best logits
// Each block takes one part of one row in a single pass: every lane keeps a running maximum and
// the sum of exponentials below it (fp32; joined in fp64), and every warp the list of its best
// logits.  Within a row the order of the log-probabilities is the order of the logits, so no
// candidate needs the row's sum before the second kernel.
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32;
constexpr int kPerThread = 16;                       // logits per thread and step
constexpr int kRowStep = kRowThreads * kPerThread;   // logits per block and step

struct RowStat {
  double sum;  // sum over the part of exp(l - max)
  float max;
  int pad;
};

template <class T>
struct Vec16;  // elements of a 16-byte load
template <>
struct Vec16<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void split(uint4 q, float *v) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
};
template <>
struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void split(uint4 q, float *v) {
    v[0] = __uint_as_float(q.x), v[1] = __uint_as_float(q.y), v[2] = __uint_as_float(q.z), v[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ float one(float x) { return x; }
};

template <class T>
__global__ void __launch_bounds__(kRowThreads)
    k_beam_rows(const T *__restrict__ logits, int64_t ldg, int64_t ldw, int W, int V, int K, int S, int vec,
                const uint8_t *__restrict__ finished, RowStat *__restrict__ stat, float *__restrict__ cval,
                int *__restrict__ cidx) {
  constexpr int VN = Vec16<T>::N, NV = kPerThread / VN;
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int r = blockIdx.x / S, s = blockIdx.x % S;
  pdl_trigger();
  pdl_wait();
  if (finished && finished[r]) return;  // an ended beam keeps its score: its logits are not read
  const T *row = logits + (int64_t)(r / W) * ldg + (int64_t)(r % W) * ldw;
  const int steps = (V + kRowStep - 1) / kRowStep;
  const int first = (int)((int64_t)steps * s / S), last = (int)((int64_t)steps * (s + 1) / S);
  float m = -FLT_MAX, sum = 0.f;
  float lv = -INFINITY;
  int li = kNoIndex;
  for (int step = first; step < last; ++step) {
    const int base = step * kRowStep + tid * VN;
    float v[kPerThread];
#pragma unroll
    for (int u = 0; u < NV; ++u) {
      const int i0 = base + u * kRowThreads * VN;
      if (vec && i0 + VN <= V) {
        Vec16<T>::split(*reinterpret_cast<const uint4 *>(row + i0), v + u * VN);
      } else {
#pragma unroll
        for (int e = 0; e < VN; ++e) v[u * VN + e] = i0 + e < V ? Vec16<T>::one(row[i0 + e]) : -INFINITY;
      }
    }
    float mx = v[0];
#pragma unroll
    for (int e = 1; e < kPerThread; ++e) mx = fmaxf(mx, v[e]);
    float mn = fmaxf(m, mx), part = 0.f;
#pragma unroll
    for (int e = 0; e < kPerThread; ++e) part += ex2_approx((v[e] - mn) * kLog2e);
    if (part != part) {  // a NaN (counts as -inf) or +inf (as the largest finite value) is among them
      mx = -INFINITY;
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) {
        v[e] = v[e] != v[e] ? -INFINITY : fminf(v[e], FLT_MAX);
        mx = fmaxf(mx, v[e]);
      }
      mn = fmaxf(m, mx), part = 0.f;
#pragma unroll
      for (int e = 0; e < kPerThread; ++e) part += ex2_approx((v[e] - mn) * kLog2e);
    }
    sum = sum * ex2_approx((m - mn) * kLog2e) + part;
    m = mn;

    // candidates: the K-th best so far bounds what can still enter; in the first step the K-th
    // largest of the 32 lane maxima does
    float cut = __shfl_sync(0xffffffffu, lv, K - 1);
    int cut_i = __shfl_sync(0xffffffffu, li, K - 1);
    if (step == first) {
      unsigned u = order_word(mx);
      unsigned kth = 0;
      for (int k = 0; k < K; ++k) {
        kth = __reduce_max_sync(0xffffffffu, u);
        const unsigned who = __ballot_sync(0xffffffffu, u == kth);
        if (lane == __ffs(who) - 1) u = 0;
      }
      // the K-th maximum itself has to enter: the cut lies just behind it
      cut = __uint_as_float(kth & 0x80000000u ? kth ^ 0x80000000u : ~kth);
      cut_i = kNoIndex;
    }
    // later steps hold higher indices only, so an equal logit enters in the first step alone
    if (!__any_sync(0xffffffffu, mx > cut || (step == first && mx == cut))) continue;
#pragma unroll
    for (int u = 0; u < NV; ++u)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const float x = v[u * VN + e];
        const int ix = base + u * kRowThreads * VN + e;
        unsigned todo = __ballot_sync(0xffffffffu, better(x, ix, cut, cut_i) && x > -INFINITY);
        while (todo) {
          const int src = __ffs(todo) - 1;
          list_insert(lv, li, __shfl_sync(0xffffffffu, x, src), __shfl_sync(0xffffffffu, ix, src), lane);
          const float kv = __shfl_sync(0xffffffffu, lv, K - 1);
          const int ki = __shfl_sync(0xffffffffu, li, K - 1);
          if (better(kv, ki, cut, cut_i)) cut = kv, cut_i = ki;
          todo &= todo - 1;
          todo &= __ballot_sync(0xffffffffu, better(x, ix, cut, cut_i));
        }
      }
  }

  // join the lanes' statistics, then the warps' statistics and lists
  __shared__ float s_max[kRowWarps];
  __shared__ double s_sum[kRowWarps];
  __shared__ float s_val[kRowWarps][32];
  __shared__ int s_idx[kRowWarps][32];
  const float wm = warp_max(m);
  const double ws = warp_sum_d((double)(sum * ex2_approx((m - wm) * kLog2e)));
  if (lane == 0) s_max[wid] = wm, s_sum[wid] = ws;
#pragma unroll
  for (int half = kRowWarps / 2; half; half >>= 1) {
    if (wid >= half && wid < 2 * half) s_val[wid][lane] = lv, s_idx[wid][lane] = li;
    __syncthreads();
    if (wid < half) list_merge(lv, li, s_val[wid + half][lane], s_idx[wid + half][lane], lane);
  }
  if (wid == 0) {
    const float bm = lane < kRowWarps ? s_max[lane] : -FLT_MAX;
    const float all = warp_max(bm);
    const double total = warp_sum_d(lane < kRowWarps ? s_sum[lane] * (double)ex2_approx((bm - all) * kLog2e) : 0.0);
    const int64_t part = blockIdx.x;
    if (lane == 0) stat[part] = RowStat{total, all, 0};
    if (lane < K) cval[part * K + lane] = lv, cidx[part * K + lane] = li;
  }
}

// ------------------------------------------------------------ pick: the best keys over a prompt's beams
// One block per prompt, one warp per beam: the parts' statistics give the row's log-normaliser,
// the parts' lists its K best logits; keys are formed in fp64, so that two candidates of a row
// whose log-probabilities round to the same fp32 keep the order of their logits.
__global__ void __launch_bounds__(1024)
    k_beam_pick(const RowStat *__restrict__ stat, const float *__restrict__ cval, const int *__restrict__ cidx, int W,
                int V, int K, int S, const float *__restrict__ scores, const uint8_t *__restrict__ finished,
                const int *__restrict__ lengths, int64_t eos, int64_t pad, double alpha,
                int64_t *__restrict__ tokens,
                int *__restrict__ parents, float *__restrict__ out_scores, uint8_t *__restrict__ out_finished,
                int *__restrict__ out_lengths) {
  const int g = blockIdx.x, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = g * W + w;
  __shared__ double s_key[kMaxBeams][32], s_score[kMaxBeams][32];
  __shared__ int s_at[kMaxBeams][32], s_tok[kMaxBeams][32];
  pdl_trigger();
  pdl_wait();
  double key = -INFINITY;
  int at = kNoIndex;  // 32 * beam + rank within the beam: the order of (beam, token) among equal keys
  const bool ended = w < W && finished && finished[r];
  if (w < W) {
    const double base = (double)scores[r];
    const int len = lengths ? lengths[r] : 0;
    double score = -INFINITY;
    int tok = 0;
    if (ended) {
      if (lane == 0) score = base, tok = (int)pad;
    } else {
      const RowStat *st = stat + (int64_t)r * S;
      float pm = -FLT_MAX;
      double ps = 0.0;
      if (lane < S) pm = st[lane].max, ps = st[lane].sum;
      const float m = warp_max(pm);
      const double total = warp_sum_d(ps * exp((double)pm - (double)m));
      float lv = -INFINITY;
      int li = kNoIndex;
      for (int s = 0; s < S; ++s) {
        const int64_t at0 = ((int64_t)r * S + s) * K;
        const float bv = lane < K ? cval[at0 + lane] : -INFINITY;
        const int bi = lane < K ? cidx[at0 + lane] : kNoIndex;
        if (s == 0)
          lv = bv, li = bi;
        else
          list_merge(lv, li, bv, bi, lane);
      }
      if (lv > -INFINITY) score = base + (((double)lv - (double)m) - log(total));
      tok = li;
    }
    if (lane < K && score > -INFINITY) {  // false for NaN scores too
      const int n = len + (ended ? 0 : 1);
      key = alpha != 0.0 ? score / pow((double)(n > 1 ? n : 1), alpha) : score;
      if (key > -INFINITY) at = w * 32 + lane;
      else key = -INFINITY;  // -inf or NaN
    }
    s_score[w][lane] = score;
    s_tok[w][lane] = tok;
  }
  // tree over the beams
  int n = 1;
  while (n < W) n <<= 1;
  for (int half = n >> 1; half; half >>= 1) {
    if (w >= half && w < 2 * half) s_key[w][lane] = key, s_at[w][lane] = at;
    __syncthreads();
    if (w < half) list_merge(key, at, w + half < W ? s_key[w + half][lane] : -INFINITY,
                             w + half < W ? s_at[w + half][lane] : kNoIndex, lane);
  }
  __syncthreads();
  if (w == 0 && lane < K) {
    const int64_t o = (int64_t)g * K + lane;
    const bool empty = at == kNoIndex;
    const int parent = empty ? (lane < W ? lane : W - 1) : at >> 5;
    const int pr = g * W + parent;
    const bool was = finished && finished[pr];
    const int64_t tok = empty ? pad : (int64_t)s_tok[parent][at & 31];
    parents[o] = parent;
    tokens[o] = tok;
    out_scores[o] = empty ? -INFINITY : (float)s_score[parent][at & 31];
    out_finished[o] = was || empty || tok == eos;
    out_lengths[o] = (lengths ? lengths[pr] : 0) + (was || empty ? 0 : 1);
  }
}

// Parts per row: enough blocks to occupy every SM a few times, none with less than one step.
static int beam_splits(int64_t R, int64_t V) {
  const int64_t steps = ceil_div(V, kRowStep);
  int64_t s = ceil_div(4 * (int64_t)sm_count(), R);
  if (s > steps) s = steps;
  if (s > 32) s = 32;  // the second kernel takes one part's statistics per lane
  return s < 1 ? 1 : (int)s;
}

static int64_t beam_ws_bytes(int64_t R, int64_t K, int64_t S) { return R * S * (int64_t)(sizeof(RowStat) + K * 8); }

// ------------------------------------------------------------ states follow their beams
// A thread owns one 16-byte (or narrower) column of the W rows of one prompt: it loads the rows'
// new values into registers and then stores them, so the permutation runs in place with every
// moved row read once and written once, and rows that stay are not touched.  All tensors of one
// call (the caches of every layer) go through the same launch.
constexpr int kMaxStates = 128;
struct StateDesc {
  const char *src;
  char *dst;
  int64_t src_stride, dst_stride;  // bytes
  uint32_t cols;                   // vectors per row
  uint32_t first_block;
  uint32_t vec;                    // bytes per vector
};
struct StateTable {
  StateDesc d[kMaxStates];
  int n;
};
constexpr int kReorderThreads = 256;

template <class VT, int MAXW>
__device__ __forceinline__ void reorder_column(const StateDesc &d, int64_t g, uint32_t col, int Win, int Wout,
                                               const int *__restrict__ parents) {
  const char *src = d.src + g * Win * d.src_stride + (int64_t)col * sizeof(VT);
  char *dst = d.dst + g * Wout * d.dst_stride + (int64_t)col * sizeof(VT);
  const bool in_place = d.src == d.dst;
  VT v[MAXW];
  unsigned moved = 0;
#pragma unroll
  for (int k = 0; k < MAXW; ++k)
    if (k < Wout) {
      const int p = parents[g * Wout + k];
      if ((unsigned)p >= (unsigned)Win) {
        atomicExch(&g_device_status, TESM_EINVAL);  // the row is left as it is
      } else if (!in_place || p != k) {
        v[k] = *reinterpret_cast<const VT *>(src + p * d.src_stride);
        moved |= 1u << k;
      }
    }
#pragma unroll
  for (int k = 0; k < MAXW; ++k)
    if (moved >> k & 1) *reinterpret_cast<VT *>(dst + k * d.dst_stride) = v[k];
}

template <int MAXW>
__global__ void __launch_bounds__(kReorderThreads)
    k_reorder_states(const __grid_constant__ StateTable t, uint32_t G, int Win, int Wout,
                     const int *__restrict__ parents) {
  pdl_trigger();
  pdl_wait();
  int lo = 0, hi = t.n - 1;  // the last state whose first block is not behind this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.d[mid].first_block <= blockIdx.x) lo = mid;
    else hi = mid - 1;
  }
  const StateDesc &d = t.d[lo];
  const uint64_t at = (uint64_t)(blockIdx.x - d.first_block) * kReorderThreads + threadIdx.x;
  if (at >= (uint64_t)G * d.cols) return;
  const uint32_t g = (uint32_t)at / d.cols, col = (uint32_t)at % d.cols;  // G * cols < 2^32
  switch (d.vec) {
    case 16: reorder_column<uint4, MAXW>(d, g, col, Win, Wout, parents); break;
    case 8: reorder_column<uint2, MAXW>(d, g, col, Win, Wout, parents); break;
    case 4: reorder_column<uint32_t, MAXW>(d, g, col, Win, Wout, parents); break;
    case 2: reorder_column<uint16_t, MAXW>(d, g, col, Win, Wout, parents); break;
    default: reorder_column<uint8_t, MAXW>(d, g, col, Win, Wout, parents); break;
  }
}

}  // namespace tesm

extern "C" int tesm_b200_beam_select_workspace(int64_t G, int64_t W, int64_t V, int64_t K, int64_t *bytes_out) {
  using namespace tesm;
  TESM_REQUIRE(bytes_out, "beam_select_workspace: null pointer");
  TESM_REQUIRE(G >= 0 && V >= 1 && W >= 1 && W <= kMaxBeams && K >= 1 && K <= kMaxBeams,
               "beam_select_workspace: bad shape");
  *bytes_out = G ? beam_ws_bytes(G * W, K, beam_splits(G * W, V)) : 0;
  return TESM_OK;
}

extern "C" int tesm_b200_beam_select(const void *logits, int dtype, int64_t ldg, int64_t ldw, int64_t G, int64_t W,
                                     int64_t V, int64_t K, const float *scores, const uint8_t *finished,
                                     const int32_t *lengths, int64_t eos, int64_t pad, double length_penalty,
                                     int64_t *tokens, int32_t *parents, float *out_scores, uint8_t *out_finished,
                                     int32_t *out_lengths, void *ws, int64_t ws_bytes, tesm_stream_t stream) {
  using namespace tesm;
  if (dtype != TESM_F32 && dtype != TESM_BF16) return fail(TESM_EDTYPE, "beam_select: dtype");
  TESM_REQUIRE(G >= 0 && W >= 1 && W <= kMaxBeams && K >= 1 && K <= kMaxBeams,
               "beam_select: 1 to 32 beams in and out");
  TESM_REQUIRE(V >= 1 && V <= (1ll << 30) && G * W < (1ll << 24), "beam_select: bad shape");
  TESM_REQUIRE(pad >= 0 && pad < (1ll << 31), "beam_select: bad pad token");
  TESM_REQUIRE(length_penalty == length_penalty && (length_penalty == 0.0 || lengths),
               "beam_select: a length penalty needs lengths");
  if (G == 0) return TESM_OK;
  TESM_REQUIRE(logits && scores && tokens && parents && out_scores && out_finished && out_lengths && ws,
               "beam_select: null pointer");
  const int64_t R = G * W;
  const int S = beam_splits(R, V);
  TESM_REQUIRE(ws_bytes >= beam_ws_bytes(R, K, S) && ((uintptr_t)ws & 15) == 0, "beam_select: workspace");
  RowStat *stat = reinterpret_cast<RowStat *>(ws);
  float *cval = reinterpret_cast<float *>(stat + R * S);
  int *cidx = reinterpret_cast<int *>(cval + R * S * K);
  const int64_t es = dtype == TESM_BF16 ? 2 : 4;
  const int vec = ((uintptr_t)logits | (uint64_t)(ldg * es) | (uint64_t)(ldw * es)) % 16 == 0;
  cudaStream_t st = (cudaStream_t)stream;
  int rc = dtype == TESM_BF16
               ? launch_k("beam_select", k_beam_rows<__nv_bfloat16>, dim3(R * S), dim3(kRowThreads), 0, st,
                          (const __nv_bfloat16 *)logits, ldg, ldw, (int)W, (int)V, (int)K, S, vec, finished, stat, cval,
                          cidx)
               : launch_k("beam_select", k_beam_rows<float>, dim3(R * S), dim3(kRowThreads), 0, st,
                          (const float *)logits, ldg, ldw, (int)W, (int)V, (int)K, S, vec, finished, stat, cval, cidx);
  if (rc) return rc;
  return launch_k("beam_select", k_beam_pick, dim3(G), dim3(32 * W), 0, st, (const RowStat *)stat,
                  (const float *)cval, (const int *)cidx, (int)W, (int)V, (int)K, S, scores, finished, lengths, eos, pad,
                  length_penalty, tokens, parents, out_scores, out_finished, out_lengths);
}

extern "C" int tesm_b200_reorder_states(const tesm_b200_state_rows *states, int64_t n, int64_t G, int64_t Win,
                                        int64_t Wout, const int32_t *parents, tesm_stream_t stream) {
  using namespace tesm;
  TESM_REQUIRE(n >= 0 && G >= 0 && Win >= 1 && Wout >= 1 && Wout <= kMaxBeams && Win < (1ll << 31),
               "reorder_states: 1 to 32 beams out");
  if (n == 0 || G == 0) return TESM_OK;
  TESM_REQUIRE(states && parents, "reorder_states: null pointer");
  for (int64_t i = 0; i < n; ++i) {
    const tesm_b200_state_rows &s = states[i];
    TESM_REQUIRE(s.row_bytes >= 0, "reorder_states: negative row size");
    if (s.row_bytes == 0) continue;
    TESM_REQUIRE(s.src && s.dst, "reorder_states: null pointer");
    TESM_REQUIRE(s.src_stride >= s.row_bytes && s.dst_stride >= s.row_bytes, "reorder_states: rows overlap");
    TESM_REQUIRE(s.src != s.dst || (Win == Wout && s.src_stride == s.dst_stride),
                 "reorder_states: in place needs as many beams out as in");
  }
  StateTable t;
  t.n = 0;
  uint64_t blocks = 0;
  for (int64_t i = 0; i <= n; ++i) {
    if (t.n && (i == n || t.n == kMaxStates || blocks >= (1ull << 30))) {
      const dim3 grid((unsigned)blocks), block(kReorderThreads);
      cudaStream_t st = (cudaStream_t)stream;
      const uint32_t g = (uint32_t)G;
      const int a = (int)Win, b = (int)Wout;
      const int rc = b <= 4    ? launch_k("reorder_states", k_reorder_states<4>, grid, block, 0, st, t, g, a, b, parents)
                     : b <= 8  ? launch_k("reorder_states", k_reorder_states<8>, grid, block, 0, st, t, g, a, b, parents)
                     : b <= 16 ? launch_k("reorder_states", k_reorder_states<16>, grid, block, 0, st, t, g, a, b, parents)
                               : launch_k("reorder_states", k_reorder_states<32>, grid, block, 0, st, t, g, a, b, parents);
      if (rc) return rc;
      t.n = 0, blocks = 0;
    }
    if (i == n || states[i].row_bytes == 0) continue;
    const tesm_b200_state_rows &s = states[i];
    const uint64_t bits = (uintptr_t)s.src | (uintptr_t)s.dst | (uint64_t)s.src_stride | (uint64_t)s.dst_stride |
                          (uint64_t)s.row_bytes;
    const uint32_t vec = bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
    const uint64_t cols = (uint64_t)s.row_bytes / vec;
    if (cols >= (1ull << 32) || (uint64_t)G * cols >= (1ull << 32))
      return fail(TESM_EUNSUPPORTED, "reorder_states: a state of 2^32 columns or more");
    t.d[t.n] = StateDesc{(const char *)s.src, (char *)s.dst, s.src_stride, s.dst_stride, (uint32_t)cols,
                         (uint32_t)blocks, vec};
    blocks += (uint64_t)ceil_div(G * (int64_t)cols, kReorderThreads);
    ++t.n;
  }
  return TESM_OK;
}
