// Log probabilities of given tokens, with rank, entropy and the k best alternatives, from logits (gfx950).
//
// Per row x (V values; f32, bf16 or f16, widened to f32 before anything else):
//   m = max x,  S = sum e^(x - m),  U = sum e^(x - m) (x - m)  (terms with e^(x - m) = 0 count nothing)
//   lse = m + ln S,  entropy = ln S - U / S,  log p(i) = (x_i - m) - ln S
//   rank(i) = 1 + #{x_j > x_i} + #{j < i : x_j = x_i}: i's place in the order (value descending, index ascending),
//   the order of the k best as well.
// (x_i - m) - ln S, not x_i - lse: a row whose values are all large (masked to the type's lowest value) keeps ln S.
//
// One pass over the row: every lane keeps a running m, S, U, rescaled once per 16 values, and every wave the k
// best of what it has seen.  Bytes bound it: 16 values of a lane cost about 12 VALU operations each, one of them a
// quarter-rate exponential, where the vector units could do about 22 per f32 value (11 per 16-bit value) at HBM rate.
#include <algorithm>

#include "kernels.h"
#include "mk_common.h"

namespace mk {

namespace {

constexpr int LP_WAVES = 4, LP_TH = 64 * LP_WAVES;
constexpr int LP_E = 16;                 // values of a lane per tile
constexpr int LP_TILE = 64 * LP_E;       // values of a wave per tile
constexpr int LP_CAP = 128;              // list entries of a wave: the k <= 64 kept and one ballot's worth of new ones
constexpr float NEG_MAX = -3.402823466e38f;
constexpr float LOG2E = 1.4426950408889634f;

__device__ inline float neg_inf() { return -__builtin_inff(); }

// Order of the alternatives: the larger value first, the lower index among equals.
__device__ inline bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

__device__ inline void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Running softmax statistics of one lane (or of a merged set).  m starts at the lowest finite value, so that a set
// of only -inf has S = 0 and no infinity is subtracted from another.
struct Stat {
  float m = NEG_MAX, s = 0.f, u = 0.f;
  // moves the reference maximum to mn >= m; the difference is kept finite (e^-1e4 is 0 anyway), 0 * -inf would be NaN
  __device__ void raise(float mn) {
    const float d = fmaxf(m - mn, -1e4f), f = fast_exp2(d * LOG2E);
    u = f * fmaf(d, s, u);
    s *= f;
    m = mn;
  }
  __device__ void merge(float m2, float s2, float u2) {
    Stat o;
    o.m = m2; o.s = s2; o.u = u2;
    const float mn = fmaxf(m, m2);
    raise(mn);
    o.raise(mn);
    s += o.s;
    u += o.u;
  }
};

// The k best (value, index) a wave has been offered, in the wave's LDS slice, and the threshold an entry has to beat:
// no worse than the k-th best so far.
struct TopList {
  float* val;
  int* idx;
  int k, cnt;
  float tv;
  int ti;

  // index bound `end`: entries at end or beyond never enter (padding)
  __device__ void init(float* v, int* i, int k_, int end) {
    val = v; idx = i; k = k_; cnt = 0;
    tv = neg_inf(); ti = end;
  }
  __device__ bool passes(float v, int i) const { return better(v, i, tv, ti); }

  // Keeps the k best of the list, in order, each entry's place the number of entries that beat it.
  __device__ void prune() {
    const int lane = threadIdx.x & 63;
    wave_fence();
    const bool h0 = lane < cnt, h1 = lane + 64 < cnt;
    const float v0 = h0 ? val[lane] : 0.f, v1 = h1 ? val[lane + 64] : 0.f;
    const int i0 = h0 ? idx[lane] : 0, i1 = h1 ? idx[lane + 64] : 0;
    int r0 = 0, r1 = 0;
    for (int j = 0; j < cnt; ++j) {
      const float v = val[j];
      const int i = idx[j];
      r0 += better(v, i, v0, i0);
      r1 += better(v, i, v1, i1);
    }
    wave_fence();
    if (h0 && r0 < k) { val[r0] = v0; idx[r0] = i0; }
    if (h1 && r1 < k) { val[r1] = v1; idx[r1] = i1; }
    wave_fence();
    if (cnt >= k) {
      cnt = k;
      tv = val[k - 1];
      ti = idx[k - 1];
    }
  }
  // one value of every lane; the list has room for a whole ballot after a prune
  __device__ void offer(float v, int i) {
    unsigned long long mask = __ballot(passes(v, i));
    if (!mask) return;
    if (cnt + __popcll(mask) > LP_CAP) {
      prune();
      mask = __ballot(passes(v, i));
      if (!mask) return;
    }
    if (passes(v, i)) {
      const int at = cnt + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
      val[at] = v;
      idx[at] = i;
    }
    cnt += __popcll(mask);
  }
};

// Values in sortable form: unsigned order is float order (NaN aside; -0 just below +0, which only loosens a bound).
__device__ inline uint32_t sort_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return (int)b < 0 ? ~b : b | 0x80000000u;
}
__device__ inline float from_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// A value that at least k of the wave's 64 lanes reach with v (k <= 64): the k-th largest lane value cut to its upper
// 16 key bits, by bisection on ballots.  At least k values of a tile are at least this large when v is the lanes' maxima.
__device__ inline float kth_bound(float v, int k) {
  const uint32_t key = sort_key(v);
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 16; --b) {
    const uint32_t c = t | (1u << b);
    if (__popcll(__ballot(key >= c)) >= k) t = c;
  }
  return t < sort_key(neg_inf()) ? neg_inf() : from_key(t);
}

template <typename T>
struct Load;
template <>
struct Load<float> {
  static constexpr int VEC = 4;
  typedef float V __attribute__((ext_vector_type(4), aligned(4)));
  __device__ static float f(float v) { return v; }
  __device__ static void unpack(const V& v, float* o) {
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = v[e];
  }
};
template <>
struct Load<__bf16> {
  static constexpr int VEC = 8;
  typedef uint16_t V __attribute__((ext_vector_type(8), aligned(2)));
  __device__ static float f(__bf16 v) { return static_cast<float>(v); }
  __device__ static void unpack(const V& v, float* o) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = bf2f(v[e]);
  }
};
template <>
struct Load<_Float16> {
  static constexpr int VEC = 8;
  typedef _Float16 V __attribute__((ext_vector_type(8), aligned(2)));
  __device__ static float f(_Float16 v) { return static_cast<float>(v); }
  __device__ static void unpack(const V& v, float* o) {
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<float>(v[e]);
  }
};

// Workspace entry of one (row, split): m, s, u, unused; n_ids counts; k values; k indices.
__host__ __device__ inline size_t part_floats(int n_ids, int k) { return 4 + (size_t)n_ids + 2 * (size_t)k; }

struct RowShared {
  float val[LP_WAVES][LP_CAP];
  int idx[LP_WAVES][LP_CAP];
  float m[LP_WAVES], s[LP_WAVES], u[LP_WAVES];
  int cnt[LP_WAVES];
  float idv[LP_MAX_IDS];
  int idn[LP_MAX_IDS];
  int rank[LP_WAVES][LP_MAX_IDS];
};

__device__ inline long long id_at(const LogprobArgs& a, size_t i) {
  return a.ids64 ? static_cast<const long long*>(a.ids)[i] : static_cast<const int*>(a.ids)[i];
}

// The row's given tokens: index (-1 outside the vocabulary) and value, into LDS by the whole workgroup.
template <typename T>
__device__ inline void load_ids(const LogprobArgs& a, int row, const T* x, RowShared& sh) {
  for (int j = threadIdx.x; j < a.n_ids; j += LP_TH) {
    const long long id = id_at(a, (size_t)row * a.n_ids + j);
    const bool in = id >= 0 && id < a.V;
    sh.idn[j] = in ? (int)id : -1;
    sh.idv[j] = in ? Load<T>::f(x[id]) : __builtin_inff();
  }
}

// Merged statistics st (all threads), ranks' counts in sh.rank[0], the sorted list of cnt entries in lv / li (LDS)
// -> the row's outputs.
__device__ inline void write_row(const LogprobArgs& a, int row, const Stat& st, const RowShared& sh, const float* lv,
                                 const int* li) {
  const bool nan = !(st.s == st.s), empty = st.s == 0.f;   // an infinite logit makes s NaN as well
  const float q = __builtin_nanf(""), ls = logf(st.s);
  if (threadIdx.x == 0) {
    a.lse[row] = nan ? q : empty ? neg_inf() : st.m + ls;
    a.entropy[row] = nan ? q : empty ? 0.f : ls - st.u / st.s;
  }
  for (int j = threadIdx.x; j < a.n_ids; j += LP_TH) {
    const size_t o = (size_t)row * a.n_ids + j;
    const bool in = sh.idn[j] >= 0;
    a.token_lp[o] = nan ? q : empty || !in ? neg_inf() : (sh.idv[j] - st.m) - ls;
    a.ranks[o] = nan || !in ? -1 : 1 + sh.rank[0][j];
  }
  for (int j = threadIdx.x; j < a.top; j += LP_TH) {
    const size_t o = (size_t)row * a.top + j;
    a.top_lp[o] = nan ? q : empty ? neg_inf() : (lv[j] - st.m) - ls;
    a.top_ids[o] = nan ? -1 : li[j];
  }
}

// Merges the waves' sorted lists (counts in sh.cnt): entry e of wave w goes to its place among all.  The places below k
// are written to ov / oi, which must not be the lists.
__device__ inline void merge_lists(const RowShared& sh, int k, float* ov, int* oi) {
  const int w = threadIdx.x >> 6, e = threadIdx.x & 63;
  if (e >= min(sh.cnt[w], k)) return;
  const float v = sh.val[w][e];
  const int i = sh.idx[w][e];
  int place = e;
#pragma unroll
  for (int o = 0; o < LP_WAVES; ++o) {
    if (o == w) continue;
    int lo = 0, hi = min(sh.cnt[o], k);
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (better(sh.val[o][mid], sh.idx[o][mid], v, i)) lo = mid + 1;
      else hi = mid;
    }
    place += lo;
  }
  if (place < k) {
    ov[place] = v;
    oi[place] = i;
  }
}

// One (row, split): values [split * chunk, min(V, + chunk)) of the row, chunk a multiple of LP_TILE.  The waves take
// its tiles in turn, so that a wave sees its values in index order tile by tile.
template <typename T, bool SPLIT>
__global__ __launch_bounds__(LP_TH, 6) void logprob_rows_kernel(LogprobArgs a, int splits, int chunk, float* part) {
  using L = Load<T>;
  constexpr int VEC = L::VEC, NV = LP_E / VEC;
  __shared__ RowShared sh;
  __shared__ float ov[LP_MAX_TOP];
  __shared__ int oi[LP_MAX_TOP];
  const int row = blockIdx.x / splits, split = blockIdx.x - row * splits;
  const int lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T* x = static_cast<const T*>(a.x) + (size_t)row * a.ldx;
  const int c0 = split * chunk, c1 = min(a.V, c0 + chunk);

  // tile at t0: lane's value e is element t0 + (e / VEC) 64 VEC + lane VEC + e % VEC
  auto at = [&](int t0, int e) { return t0 + (e / VEC) * 64 * VEC + lane * VEC + e % VEC; };
  typename L::V raw[NV];
  auto load = [&](int t0) {
#pragma unroll
    for (int q = 0; q < NV; ++q) raw[q] = *reinterpret_cast<const typename L::V*>(x + at(t0, q * VEC));
  };
  int t0 = c0 + w * LP_TILE;
  if (t0 + LP_TILE <= c1) load(t0);
  load_ids<T>(a, row, x, sh);
  for (int j = lane; j < a.n_ids; j += 64) sh.rank[w][j] = 0;
  __syncthreads();

  Stat st;
  TopList top;
  top.init(sh.val[w], sh.idx[w], a.top, c1);
  for (; t0 < c1; t0 += LP_WAVES * LP_TILE) {
    float v[LP_E];
    if (t0 + LP_TILE <= c1) {
#pragma unroll
      for (int q = 0; q < NV; ++q) L::unpack(raw[q], v + q * VEC);
    } else {
#pragma unroll
      for (int e = 0; e < LP_E; ++e) {
        const int i = at(t0, e);
        v[e] = i < c1 ? L::f(x[i]) : neg_inf();
      }
    }
    const int tn = t0 + LP_WAVES * LP_TILE;
    if (tn + LP_TILE <= c1) load(tn);

    float tm = v[0];
#pragma unroll
    for (int e = 1; e < LP_E; ++e) tm = fmaxf(tm, v[e]);
    st.raise(fmaxf(st.m, tm));
    float s = 0.f, u = 0.f;
#pragma unroll
    for (int e = 0; e < LP_E; ++e) {
      // the difference first: its rounding is relative to itself, where x log2(e) - m log2(e) would round at |x|
      const float d = v[e] - st.m, p = fast_exp2(d * LOG2E);
      s += p;
      u = fmaf(p, fmaxf(d, -200.f), u);   // p is 0 below -200: no 0 * -inf
    }
    st.s += s;
    st.u += u;

    for (int j = 0; j < a.n_ids; ++j) {
      const float iv = sh.idv[j];
      const int id = sh.idn[j];
      int n = 0;
      if (t0 + LP_TILE <= id) {            // every value here has a lower index
#pragma unroll
        for (int e = 0; e < LP_E; ++e) n += __popcll(__ballot(v[e] >= iv));
      } else if (t0 > id) {
#pragma unroll
        for (int e = 0; e < LP_E; ++e) n += __popcll(__ballot(v[e] > iv));
      } else {
#pragma unroll
        for (int e = 0; e < LP_E; ++e) n += __popcll(__ballot(better(v[e], at(t0, e), iv, id)));
      }
      if (lane == 0) sh.rank[w][j] += n;
    }

    if (a.top && __ballot(tm >= top.tv)) {
      if (top.cnt == 0) {                  // nothing known yet: a bound from the lanes' maxima
        const float b = kth_bound(tm, top.k);
        if (b > top.tv) {
          top.tv = b;
          top.ti = c1;
        }
      }
#pragma unroll
      for (int e = 0; e < LP_E; ++e) top.offer(v[e], at(t0, e));
      if (top.cnt > min(top.k + 32, 2 * top.k)) top.prune();
    }
  }

  // the lanes' statistics, then the waves'
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) st.merge(__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.u, o));
  if (a.top) top.prune();
  if (lane == 0) {
    sh.m[w] = st.m;
    sh.s[w] = st.s;
    sh.u[w] = st.u;
    sh.cnt[w] = top.cnt;
  }
  for (int j = threadIdx.x; j < a.top; j += LP_TH) {
    ov[j] = neg_inf();
    oi[j] = 0x7fffffff;
  }
  __syncthreads();
  Stat all;
#pragma unroll
  for (int o = 0; o < LP_WAVES; ++o) all.merge(sh.m[o], sh.s[o], sh.u[o]);
  for (int j = threadIdx.x; j < a.n_ids; j += LP_TH) {
    int n = 0;
#pragma unroll
    for (int o = 0; o < LP_WAVES; ++o) n += sh.rank[o][j];
    sh.rank[0][j] = n;
  }
  if (a.top) merge_lists(sh, a.top, ov, oi);
  __syncthreads();
  if constexpr (!SPLIT) {
    write_row(a, row, all, sh, ov, oi);
  } else {
    float* p = part + (size_t)blockIdx.x * part_floats(a.n_ids, a.top);
    if (threadIdx.x == 0) {
      p[0] = all.m;
      p[1] = all.s;
      p[2] = all.u;
    }
    for (int j = threadIdx.x; j < a.n_ids; j += LP_TH) reinterpret_cast<int*>(p)[4 + j] = sh.rank[0][j];
    float* pv = p + 4 + a.n_ids;
    for (int j = threadIdx.x; j < a.top; j += LP_TH) {
      pv[j] = ov[j];
      reinterpret_cast<int*>(pv)[a.top + j] = oi[j];
    }
  }
}

// One row from its splits' entries, in a fixed order.
template <typename T>
__global__ __launch_bounds__(LP_TH) void logprob_merge_kernel(LogprobArgs a, int splits, const float* part) {
  __shared__ RowShared sh;
  __shared__ float ov[LP_MAX_TOP];
  __shared__ int oi[LP_MAX_TOP];
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t pf = part_floats(a.n_ids, a.top);
  const float* p = part + (size_t)row * splits * pf;
  load_ids<T>(a, row, static_cast<const T*>(a.x) + (size_t)row * a.ldx, sh);

  Stat st;
  for (int i = threadIdx.x; i < splits; i += LP_TH) st.merge(p[i * pf], p[i * pf + 1], p[i * pf + 2]);
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) st.merge(__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.u, o));
  if (lane == 0) {
    sh.m[w] = st.m;
    sh.s[w] = st.s;
    sh.u[w] = st.u;
  }
  for (int j = threadIdx.x; j < a.n_ids; j += LP_TH) {
    int n = 0;
    for (int i = 0; i < splits; ++i) n += reinterpret_cast<const int*>(p + i * pf)[4 + j];
    sh.rank[0][j] = n;
  }
  if (a.top) {
    const int k = a.top, n = splits * k;
    TopList top;
    top.init(sh.val[w], sh.idx[w], k, a.V);
    for (int i = w * 64; i < n; i += LP_TH) {
      const int e = i + lane, s = min(e, n - 1) / k, j = min(e, n - 1) - s * k;
      const float* pv = p + s * pf + 4 + a.n_ids;
      // lanes past the entries hold what the splits' own padding is: -inf under an index that no bound admits
      const float v = e < n ? pv[j] : neg_inf();
      const int id = e < n ? reinterpret_cast<const int*>(pv)[k + j] : 0x7fffffff;
      if (top.cnt == 0) {
        const float b = kth_bound(v, k);
        if (b > top.tv) {
          top.tv = b;
          top.ti = a.V;
        }
      }
      top.offer(v, id);
      if (top.cnt > min(k + 32, 2 * k)) top.prune();
    }
    top.prune();
    if (lane == 0) sh.cnt[w] = top.cnt;
    for (int j = threadIdx.x; j < k; j += LP_TH) {
      ov[j] = neg_inf();
      oi[j] = 0x7fffffff;
    }
  }
  __syncthreads();
  Stat all;
#pragma unroll
  for (int o = 0; o < LP_WAVES; ++o) all.merge(sh.m[o], sh.s[o], sh.u[o]);
  if (a.top) merge_lists(sh, a.top, ov, oi);
  __syncthreads();
  write_row(a, row, all, sh, ov, oi);
}

template <typename T>
int launch_t(const LogprobArgs& a, void* ws, hipStream_t st) {
  const int splits = logprob_splits(a.T, a.V);
  const int tiles = (a.V + LP_TILE - 1) / LP_TILE;
  const int chunk = (tiles + splits - 1) / splits * LP_TILE;
  float* part = static_cast<float*>(ws);
  const dim3 block(LP_TH);
  if (splits == 1) {
    hipLaunchKernelGGL((logprob_rows_kernel<T, false>), dim3(a.T), block, 0, st, a, 1, chunk, nullptr);
  } else {
    hipLaunchKernelGGL((logprob_rows_kernel<T, true>), dim3((unsigned)((size_t)a.T * splits)), block, 0, st, a, splits, chunk, part);
    hipLaunchKernelGGL((logprob_merge_kernel<T>), dim3(a.T), block, 0, st, a, splits, part);
  }
  MK_HIP_CHECK(hipGetLastError());
  return MK_OK;
}

}  // namespace

size_t logprob_scratch_bytes(int T, int V, int n_ids, int top) {
  const int splits = logprob_splits(T, V);
  return splits == 1 ? 0 : (size_t)T * splits * part_floats(n_ids, top) * sizeof(float);
}

int launch_logprobs(const LogprobArgs& a, void* ws, hipStream_t st) {
  if (a.T == 0) return MK_OK;
  switch (a.dtype) {
    case 0: return launch_t<float>(a, ws, st);
    case 1: return launch_t<__bf16>(a, ws, st);
    case 2: return launch_t<_Float16>(a, ws, st);
  }
  set_error("logprobs: unknown logits type");
  return MK_EINVAL;
}

}  // namespace mk
