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

// The larger of the two partners at distance o (the lower lane keeps it).
template <class V>
__device__ __forceinline__ void list_exchange(V &v, int &i, int o, bool low) {
  const V ov = __shfl_xor_sync(0xffffffffu, v, o);
  const int oi = __shfl_xor_sync(0xffffffffu, i, o);
  if (better(ov, oi, v, i) == low) v = ov, i = oi;
}

// The 32 best of two sorted lists: the larger of a[l] and b[31 - l] is a bitonic sequence, sorted
// by five compare-exchange rounds.
template <class V>
__device__ __forceinline__ void list_merge(V &v, int &i, V bv, int bi, int lane) {
  bv = __shfl_sync(0xffffffffu, bv, 31 - lane);
  bi = __shfl_sync(0xffffffffu, bi, 31 - lane);
  if (better(bv, bi, v, i)) v = bv, i = bi;
#pragma unroll
  for (int o = 16; o; o >>= 1) list_exchange(v, i, o, !(lane & o));
}

// Sort one candidate per lane (bitonic).
template <class V>
__device__ __forceinline__ void list_sort(V &v, int &i, int lane) {
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1) list_exchange(v, i, o, !(lane & o) == !(lane & size));
}

// Order-preserving map of a float to an unsigned (larger floats, larger words) and back.
__device__ __forceinline__ unsigned order_word(float x) {
  const unsigned b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float order_float(unsigned w) {
  return __uint_as_float(w & 0x80000000u ? w ^ 0x80000000u : ~w);
}
__device__ __forceinline__ void word_exchange(unsigned &w, int o, bool low) {
  const unsigned x = __shfl_xor_sync(0xffffffffu, w, o);
  w = low ? max(w, x) : min(w, x);
}

// ------------------------------------------------------------ rows: softmax statistics and best logits
// Each block takes one part of one row.  The pass over the part keeps, per thread, a running maximum
// and the sum of exponentials below it, nothing else.  The exponentials are the hardware's (2^-22 relative)
// and a thread's sum is fp32, joined in fp64: a score is off by up to about 1e-6, which can turn
// round beams that near, never tokens of one beam; fp64 exponentials would cost many times the pass.  Within a row
// the order of the log-probabilities is the order of the logits, and the K-th largest of the 256
// threads' maxima bounds the part's K-th best logit from below.  So only the threads whose
// maximum reaches it (K of them, more with ties) hold candidates, and of their logits only the
// steps whose own maximum reaches it are read again.  240 fp32 rows of 151936 logits, 32 best: 41 us
// with the second kernel (3.6 TB/s; the pass alone 30 us, 25 us for plain loads of the same bytes, the
// second look 5 us, the pick 5 us).  A candidate list kept during the pass took 99 us.
constexpr int kRowThreads = 256, kRowWarps = kRowThreads / 32, kRowBlocks = 4 /* per SM */;

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
  static __device__ __forceinline__ void split(uint4 q, float2 *v) {
    const unsigned w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
  }
  static __device__ __forceinline__ float one(__nv_bfloat16 x) { return __bfloat162float(x); }
};
template <>
struct Vec16<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void split(uint4 q, float2 *v) {
    v[0] = make_float2(__uint_as_float(q.x), __uint_as_float(q.y));
    v[1] = make_float2(__uint_as_float(q.z), __uint_as_float(q.w));
  }
  static __device__ __forceinline__ float one(float x) { return x; }
};

constexpr int kRowVecs = 4;  // 16-byte loads per thread and step
constexpr int kSubs = 4;     // classes of steps whose maxima a thread keeps apart
template <class T>
constexpr int row_step() { return kRowThreads * kRowVecs * Vec16<T>::N; }  // logits per block and step

__device__ __forceinline__ float clean_logit(float x) { return x != x ? -INFINITY : fminf(x, FLT_MAX); }

template <class T>
__global__ void __launch_bounds__(kRowThreads, kRowBlocks)
    k_beam_rows(const T *__restrict__ logits, int64_t ldg, int64_t ldw, int W, int V, int K, int S, int vec,
                const uint8_t *__restrict__ finished, RowStat *__restrict__ stat, float *__restrict__ cval,
                int *__restrict__ cidx) {
  constexpr int VN = Vec16<T>::N, NV = kRowVecs, STEP = row_step<T>();
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int r = blockIdx.x / S, s = blockIdx.x % S;
  pdl_wait();
  pdl_trigger();  // after the wait: the second kernel reads inputs before its own
  if (finished && finished[r]) return;  // an ended beam keeps its score: its logits are not read
  const T *row = logits + (int64_t)(r / W) * ldg + (int64_t)(r % W) * ldw;
  const int steps = (V + STEP - 1) / STEP;
  const int first = (int)((int64_t)steps * s / S), last = (int)((int64_t)steps * (s + 1) / S);
  float m = -FLT_MAX, sum = 0.f;
  float sub[kSubs];  // maxima of this thread's steps first + k, first + k + kSubs, ...
#pragma unroll
  for (int k = 0; k < kSubs; ++k) sub[k] = -INFINITY;
  auto consume = [&](float2 (&v)[NV][VN / 2], float &sub_max) {
    auto top = [&]() {
      float mx = fmaxf(v[0][0].x, v[0][0].y);
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < VN / 2; ++e) mx = fmaxf(mx, fmaxf(v[u][e].x, v[u][e].y));
      return mx;
    };
    float mx = top(), mn = fmaxf(m, mx);
    auto total = [&]() {
      float2 part = make_float2(0.f, 0.f);
      const float2 off = make_float2(-mn, -mn), scale = make_float2(kLog2e, kLog2e);
#pragma unroll
      for (int u = 0; u < NV; ++u) {
        float2 p = make_float2(0.f, 0.f);  // vector by vector: fewer roundings than one chain
#pragma unroll
        for (int e = 0; e < VN / 2; ++e) {
          const float2 t = __fmul2_rn(__fadd2_rn(v[u][e], off), scale);
          p = __fadd2_rn(p, make_float2(ex2_approx(t.x), ex2_approx(t.y)));
        }
        part = __fadd2_rn(part, p);
      }
      return part.x + part.y;
    };
    float part = total();
    if (part != part) {  // a NaN (counts as -inf) or +inf (as the largest finite value) is among them
#pragma unroll
      for (int u = 0; u < NV; ++u)
#pragma unroll
        for (int e = 0; e < VN / 2; ++e) v[u][e] = make_float2(clean_logit(v[u][e].x), clean_logit(v[u][e].y));
      mx = top(), mn = fmaxf(m, mx);
      part = total();
    }
    sum = sum * ex2_approx((m - mn) * kLog2e) + part;
    m = mn;
    sub_max = fmaxf(sub_max, mx);
  };
  // whole steps of whole 16-byte vectors, one step ahead; then the others logit by logit, as are all rows
  // where one may start off a 16-byte boundary (256 rows of 49999 logits: 21.8 us in bf16, 19.6 in fp32; of
  // 50000: 17.1 and 17.2)
  const int whole = vec ? min(last, V / STEP) : first;
  const T *p = row + (int64_t)first * STEP + tid * VN;
  uint4 q[NV];
  if (first < whole) {
#pragma unroll
    for (int u = 0; u < NV; ++u) q[u] = *reinterpret_cast<const uint4 *>(p + u * kRowThreads * VN);
  }
  for (int step = first; step < last; step += kSubs) {
#pragma unroll
    for (int k = 0; k < kSubs; ++k) {
      if (step + k >= last) break;
      float2 v[NV][VN / 2];
      if (step + k < whole) {
#pragma unroll
        for (int u = 0; u < NV; ++u) Vec16<T>::split(q[u], v[u]);
        p += STEP;
        if (step + k + 1 < whole) {
#pragma unroll
          for (int u = 0; u < NV; ++u) q[u] = *reinterpret_cast<const uint4 *>(p + u * kRowThreads * VN);
        }
      } else {
#pragma unroll
        for (int u = 0; u < NV; ++u) {
          const int i0 = (step + k) * STEP + (u * kRowThreads + tid) * VN;
          if (vec && i0 + VN <= V) {
            Vec16<T>::split(*reinterpret_cast<const uint4 *>(row + i0), v[u]);
          } else {
#pragma unroll
            for (int e = 0; e < VN; ++e) {
              const float x = i0 + e < V ? Vec16<T>::one(row[i0 + e]) : -INFINITY;
              if (e % 2) v[u][e / 2].y = x;
              else v[u][e / 2].x = x;
            }
          }
        }
      }
      consume(v, sub[k]);
    }
  }

  // the K-th largest of the threads' maxima (sorted within warps, then merged), and the statistics
  __shared__ float s_max[kRowWarps];
  __shared__ double s_sum[kRowWarps];
  __shared__ unsigned s_word[kRowWarps][32], s_count;
  __shared__ unsigned short s_hot[kRowThreads * kSubs];
  __shared__ float s_val[kRowWarps][32];
  __shared__ int s_idx[kRowWarps][32];
  const float wm = warp_max(m);
  const double ws = warp_sum_d((double)(sum * ex2_approx((m - wm) * kLog2e)));
  unsigned word = order_word(m);
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int o = size >> 1; o; o >>= 1) word_exchange(word, o, !(lane & o) == !(lane & size));
  s_word[wid][lane] = word;
  if (lane == 0) s_max[wid] = wm, s_sum[wid] = ws;
  if (tid == 0) s_count = 0;
  __syncthreads();
#pragma unroll
  for (int half = kRowWarps / 2; half; half >>= 1) {
    if (wid < half) {
      word = max(word, s_word[wid + half][31 - lane]);
#pragma unroll
      for (int o = 16; o; o >>= 1) word_exchange(word, o, !(lane & o));
      s_word[wid][lane] = word;
    }
    __syncthreads();
  }
  const float bound = order_float(s_word[0][K - 1]);
  // the hot (thread, class of steps) pairs, in any order: what they hold is sorted afterwards
#pragma unroll
  for (int k = 0; k < kSubs; ++k)
    if (sub[k] >= bound && sub[k] > -INFINITY) s_hot[atomicAdd(&s_count, 1u)] = (unsigned short)(tid * kSubs + k);
  __syncthreads();
  // the hot threads' logits again: the block's hot (thread, class of steps) pairs go round the warps,
  // their logits to the lanes
  float lv = -INFINITY;
  int li = kNoIndex;
  float cut = bound;
  int cut_i = kNoIndex;  // the bound itself enters
  constexpr int PER = 32 / VN, AHEAD = 4;  // vectors per load of a warp, loads in flight
  const int hots = (int)s_count;
  for (int h = wid; h < hots; h += kRowWarps) {
    const int t = s_hot[h] / kSubs, k_sub = s_hot[h] % kSubs;
    const int vecs = (last - first - k_sub + kSubs - 1) / kSubs * NV;
    for (int k0 = 0; k0 < vecs; k0 += AHEAD * PER) {
      float xs[AHEAD];
      int ixs[AHEAD];
#pragma unroll
      for (int g = 0; g < AHEAD; ++g) {
        const int k = k0 + g * PER + lane / VN;  // this lane: logit lane % VN of vector k
        ixs[g] = (first + k_sub + k / NV * kSubs) * STEP + (k % NV * kRowThreads + t) * VN + lane % VN;
        xs[g] = k < vecs && ixs[g] < V ? Vec16<T>::one(row[ixs[g]]) : -INFINITY;
      }
#pragma unroll
      for (int g = 0; g < AHEAD; ++g) {
        const float x = clean_logit(xs[g]);
        const int ix = ixs[g];
        unsigned in = __ballot_sync(0xffffffffu, x > -INFINITY && better(x, ix, cut, cut_i));
        if (!in) continue;
        if (__popc(in) > 6) {  // many at once: sort them and merge the lists
          float xv = in >> lane & 1 ? x : -INFINITY;
          int xi = in >> lane & 1 ? ix : kNoIndex;
          list_sort(xv, xi, lane);
          list_merge(lv, li, xv, xi, lane);
        } else {
          for (; in; in &= in - 1) {
            const int src = __ffs(in) - 1;
            list_insert(lv, li, __shfl_sync(0xffffffffu, x, src), __shfl_sync(0xffffffffu, ix, src), lane);
          }
        }
        const float kth = __shfl_sync(0xffffffffu, lv, K - 1);
        const int kth_i = __shfl_sync(0xffffffffu, li, K - 1);
        if (better(kth, kth_i, cut, cut_i)) cut = kth, cut_i = kth_i;
      }
    }
  }
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
// the parts' lists its K best logits.  Keys are formed in fp64 from those statistics, so that two candidates of a row
// whose log-probabilities round to the same fp32 keep the order of their logits; the logarithms and
// powers of all beams are taken by one warp, lane per beam, since fp64 functions cost as much for
// one lane as for 32.  Launched while the first kernel runs; it waits for it where it reads its output,
// which is not __restrict__: as constant for this kernel's life it could be loaded before the wait.
__global__ void __launch_bounds__(1024)
    k_beam_pick(const RowStat *stat, const float *cval, const int *cidx, int W, int V, int K, int S,
                const float *__restrict__ scores, const uint8_t *__restrict__ finished,
                const int *__restrict__ lengths, int64_t eos, int64_t pad, double alpha,
                int64_t *__restrict__ tokens, int *__restrict__ parents, float *__restrict__ out_scores,
                uint8_t *__restrict__ out_finished, int *__restrict__ out_lengths) {
  const int g = blockIdx.x, w = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = g * W + w;
  __shared__ double s_key[kMaxBeams][32], s_score[kMaxBeams][32];
  __shared__ double s_total[kMaxBeams], s_base[kMaxBeams], s_scale[kMaxBeams];
  __shared__ int s_at[kMaxBeams][32], s_tok[kMaxBeams][32], s_len[kMaxBeams], s_ended[kMaxBeams];
  pdl_trigger();
  const bool ended = finished && finished[r];
  double base = 0.0, scale = 1.0;  // of beam `lane`, in warp 0
  if (w == 0 && lane < W) {
    const int rl = g * W + lane;
    const int len = lengths ? lengths[rl] : 0;
    const bool end = finished && finished[rl];
    base = (double)scores[rl];
    const int n = len + (end ? 0 : 1);
    if (alpha != 0.0) scale = pow((double)(n > 1 ? n : 1), alpha);
    s_len[lane] = len;
    s_ended[lane] = end;
  }
  pdl_wait();
  float m = 0.f, lv = -INFINITY;
  int li = kNoIndex;
  if (!ended) {
    const RowStat *st = stat + (int64_t)r * S;
    float pm = -FLT_MAX;
    double ps = 0.0;
    if (lane < S) pm = st[lane].max, ps = st[lane].sum;
    // the parts' lists, as many whole ones at a time as fill the lanes
    const int per = 32 / K, n = S * K;
    for (int at0 = 0; at0 < n; at0 += per * K) {
      const int at1 = at0 + lane;
      const bool in = lane < per * K && at1 < n;
      float bv = in ? cval[(int64_t)r * n + at1] : -INFINITY;
      int bi = in ? cidx[(int64_t)r * n + at1] : kNoIndex;
      if (per > 1) list_sort(bv, bi, lane);
      if (at0 == 0)
        lv = bv, li = bi;
      else
        list_merge(lv, li, bv, bi, lane);
    }
    m = warp_max(pm);
    const double total = warp_sum_d(ps * (double)ex2_approx((pm - m) * kLog2e));
    if (lane == 0) s_total[w] = total;
  }
  __syncthreads();
  if (w == 0 && lane < W) {
    s_base[lane] = s_ended[lane] ? base : base - log(s_total[lane]);
    s_scale[lane] = scale;
  }
  __syncthreads();
  double score = -INFINITY, key = -INFINITY;
  int at = kNoIndex;  // 32 * beam + rank within the beam: the order of (beam, token) among equal keys
  if (ended) {
    if (lane == 0) score = s_base[w], li = (int)pad;
  } else if (lv > -INFINITY) {
    score = ((double)lv - (double)m) + s_base[w];
  }
  if (lane < K && score > -INFINITY) {  // false for NaN scores too
    key = alpha != 0.0 ? score / s_scale[w] : score;
    if (key > -INFINITY) at = w * 32 + lane;
    else key = -INFINITY;  // -inf or NaN
  }
  s_score[w][lane] = score;
  s_tok[w][lane] = li;
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
    const bool was = s_ended[parent];
    const int64_t tok = empty ? pad : (int64_t)s_tok[parent][at & 31];
    parents[o] = parent;
    tokens[o] = tok;
    out_scores[o] = empty ? -INFINITY : (float)s_score[parent][at & 31];
    out_finished[o] = was || empty || tok == eos;
    out_lengths[o] = s_len[parent] + (was || empty ? 0 : 1);
  }
}

// launch_k with the programmatic attribute set: the kernel may start while the one before it in the
// stream runs (the pair's own ordering; other kernels go by launch_k).
template <typename... KArgs, typename... Args>
static int launch_after(const char *what, void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                        Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...);
  if (e != cudaSuccess) return fail(TESM_ELAUNCH, std::string(what) + ": " + cudaGetErrorString(e));
  return TESM_OK;
}

// Parts per row: as many as run at once, none with less than one step.  A second, partly filled
// round of blocks costs more than idle SMs in the first (240 fp32 rows of 151936: 41 us with 2
// parts, 48 with 4).  From 592 rows on a row has one part, and the rows beyond a full round cost
// another (32000 bf16 logits: 592 rows 20.6 us, 600 to 640 rows 23.8, 1184 rows 30.4).
static int beam_splits(int64_t R, int64_t V, int dtype) {
  const int64_t steps = ceil_div(V, dtype == TESM_BF16 ? row_step<__nv_bfloat16>() : row_step<float>());
  int64_t s = kRowBlocks * (int64_t)sm_count() / R;
  if (s > steps) s = steps;
  if (s > 32) s = 32;  // the second kernel takes one part's statistics per lane
  return s < 1 ? 1 : (int)s;
}

// Sizes of which no product leaves 64 bits and no grid 31.
static bool beam_shape_ok(int64_t G, int64_t W, int64_t V, int64_t K) {
  return W >= 1 && W <= kMaxBeams && K >= 1 && K <= kMaxBeams && V >= 1 && V <= (1ll << 30) && G >= 0 &&
         G <= ((1ll << 24) - 1) / W;
}

static int64_t beam_ws_bytes(int64_t R, int64_t K, int64_t S) { return R * S * (int64_t)(sizeof(RowStat) + K * 8); }

// ------------------------------------------------------------ states follow their beams
// A thread owns one 16-byte (or narrower) column of the W rows of one prompt: it loads the rows'
// new values into registers and then stores them, so the permutation runs in place with every
// moved row read once and written once, and rows that stay are not touched.  All tensors of one
// call (the caches of every layer) go through the same launch.  Memory bounds it: 96 tensors of
// 256 rows (184 MB), random parents of four beams: 40 us, 6.5 TB/s of rows read and written.
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

// The widest access that all rows of a state are aligned to.
static uint32_t state_vec(const tesm_b200_state_rows &s) {
  const uint64_t bits = (uintptr_t)s.src | (uintptr_t)s.dst | (uint64_t)s.src_stride | (uint64_t)s.dst_stride |
                        (uint64_t)s.row_bytes;
  return bits % 16 == 0 ? 16 : bits % 8 == 0 ? 8 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 1;
}

}  // namespace tesm

extern "C" int tesm_b200_beam_select_workspace(int dtype, int64_t G, int64_t W, int64_t V, int64_t K, int64_t *bytes_out) {
  using namespace tesm;
  if (dtype != TESM_F32 && dtype != TESM_BF16) return fail(TESM_EDTYPE, "beam_select_workspace: dtype");
  TESM_REQUIRE(bytes_out, "beam_select_workspace: null pointer");
  TESM_REQUIRE(beam_shape_ok(G, W, V, K), "beam_select_workspace: bad shape");
  *bytes_out = G ? beam_ws_bytes(G * W, K, beam_splits(G * W, V, dtype)) : 0;
  return TESM_OK;
}

extern "C" int tesm_b200_beam_select(const void *logits, int dtype, int64_t ldg, int64_t ldw, int64_t G, int64_t W,
                                     int64_t V, int64_t K, const float *scores, const uint8_t *finished,
                                     const int32_t *lengths, int64_t eos, int64_t pad, double length_penalty,
                                     int64_t *tokens, int32_t *parents, float *out_scores, uint8_t *out_finished,
                                     int32_t *out_lengths, void *ws, int64_t ws_bytes, tesm_stream_t stream) {
  using namespace tesm;
  if (dtype != TESM_F32 && dtype != TESM_BF16) return fail(TESM_EDTYPE, "beam_select: dtype");
  TESM_REQUIRE(W >= 1 && W <= kMaxBeams && K >= 1 && K <= kMaxBeams, "beam_select: 1 to 32 beams in and out");
  TESM_REQUIRE(beam_shape_ok(G, W, V, K), "beam_select: bad shape");
  TESM_REQUIRE(pad >= 0 && pad < (1ll << 31), "beam_select: bad pad token");
  TESM_REQUIRE(length_penalty == length_penalty && (length_penalty == 0.0 || lengths),
               "beam_select: a length penalty needs lengths");
  if (G == 0) return TESM_OK;
  TESM_REQUIRE(logits && scores && tokens && parents && out_scores && out_finished && out_lengths && ws,
               "beam_select: null pointer");
  const int64_t R = G * W;
  const int S = beam_splits(R, V, dtype);
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
  return launch_after("beam_select", k_beam_pick, dim3(G), dim3(32 * W), 0, st, (const RowStat *)stat,
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
    const uint64_t cols = (uint64_t)s.row_bytes / state_vec(s);
    if (cols >= (1ull << 32) || (uint64_t)G >= (1ull << 32) || (uint64_t)G * cols >= (1ull << 32))
      return fail(TESM_EUNSUPPORTED, "reorder_states: a state of 2^32 columns or more");
    const char *lo = (const char *)s.dst, *hi = lo + (G * Wout - 1) * s.dst_stride + s.row_bytes;
    TESM_REQUIRE((const char *)(parents + G * Wout) <= lo || (const char *)parents >= hi,
                 "reorder_states: parents lie inside a state");
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
    const uint32_t vec = state_vec(s);
    const uint64_t cols = (uint64_t)s.row_bytes / vec;
    t.d[t.n] = StateDesc{(const char *)s.src, (char *)s.dst, s.src_stride, s.dst_stride, (uint32_t)cols,
                         (uint32_t)blocks, vec};
    blocks += (uint64_t)ceil_div(G * (int64_t)cols, kReorderThreads);
    ++t.n;
  }
  return TESM_OK;
}
