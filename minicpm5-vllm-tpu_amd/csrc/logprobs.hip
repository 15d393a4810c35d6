// Log probabilities of given tokens, with rank, entropy and the k best alternatives, from logits (gfx950).
//
// Per row x (V values; f32, bf16 or f16, widened to f32 before anything else):
//   m = max x,  S = sum e^(x - m),  U = sum e^(x - m) (x - m)  (terms with e^(x - m) = 0 count nothing)
//   lse = m + ln S,  entropy = ln S - U / S,  log p(i) = (x_i - m) - ln S
//   rank(i) = 1 + #{x_j > x_i} + #{j < i : x_j = x_i}: i's place in the order (value descending, index ascending),
//   the order of the k best as well.
// (x_i - m) - ln S, not x_i - lse: a row whose values are all large (masked to the type's lowest value) keeps ln S.  ln S
// is log1p(S - 1) with S - 1 summed without the row's largest term: where one token is all but certain, an f32 S near 1
// would lose what that token's log probability and the entropy consist of (a token 12 above 32768 others: relative error
// 1e-3 that way, 3e-7 this way).
//
// One pass over the row: every lane keeps a running m, S, U, rescaled once per 16 values, and every wave a list of what
// may be among the k best.  Bytes bound many rows: (2048, 130560) bf16 121 us, 4.4 TB/s, (1000, 130560) f32 107 us,
// 4.9 TB/s; a value costs about 12 VALU operations, one of them a quarter-rate exponential, and the vector units are 65 %
// busy at 16-bit values.  One row is bound by its latencies: loads, bound, listing, merge, 13.5 us at 130560 values.
#include <algorithm>

#include "kernels.h"
#include "mk_common.h"

namespace mk {

namespace {

constexpr int LP_E = 16;                 // values of a lane per tile
constexpr int LP_TILE = 64 * LP_E;       // values of a wave per tile
constexpr int LP_CAP = 128;              // list entries of a wave: the k <= 64 kept and one ballot's worth of new ones
constexpr float NEG_MAX = -3.402823466e38f;
constexpr float LOG2E = 1.4426950408889634f;

__device__ inline float neg_inf() { return -__builtin_inff(); }

__device__ inline void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Reductions over the wave, the result in every lane: within rows of 16 lanes by DPP (lane ^ 1, lane ^ 2, then mirrored
// halves and rows, whose lanes hold equal values by then), across the four rows by two permutes.
template <int CTRL>
__device__ inline float dpp(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
template <class F>
__device__ inline float wave_reduce(float v, F f) {
  v = f(v, dpp<0xb1>(v));    // quad_perm [1, 0, 3, 2]
  v = f(v, dpp<0x4e>(v));    // quad_perm [2, 3, 0, 1]
  v = f(v, dpp<0x141>(v));   // row_half_mirror
  v = f(v, dpp<0x140>(v));   // row_mirror
  v = f(v, __shfl_xor(v, 16));
  return f(v, __shfl_xor(v, 32));
}
__device__ inline float wave_max(float v) { return wave_reduce(v, [](float a, float b) { return fmaxf(a, b); }); }
__device__ inline float wave_sum(float v) { return wave_reduce(v, [](float a, float b) { return a + b; }); }

// Running softmax statistics.  m starts at the lowest finite value, so that a set of only -inf has S = 0 and no
// infinity is subtracted from another.
struct Stat {
  float m = NEG_MAX, s = 0.f, u = 0.f;
  // moves the reference maximum to mn >= m; the difference is kept finite (e^-1e4 is 0 anyway), 0 * -inf would be NaN
  __device__ void raise(float mn) {
    const float d = fmaxf(m - mn, -1e4f), f = fast_exp2(d * LOG2E);
    u = f * fmaf(d, s, u);
    s *= f;
    m = mn;
  }
  // raises every lane to the wave's maximum; the first lane with values that holds it (0 where none has any)
  __device__ int join() {
    const float lm = m;
    const bool some = s > 0.f;
    raise(wave_max(lm));
    const unsigned long long mask = __ballot(some && lm == m);
    return mask ? __builtin_ctzll(mask) : 0;
  }
};

// Values in sortable form: unsigned order is float order, -0 as +0 (NaN aside).
__device__ inline uint32_t sort_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.f);
  return (int)b < 0 ? ~b : b | 0x80000000u;
}
__device__ inline float from_key(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
// An alternative as one number: the larger value first, the lower index among equals, is the larger entry.
typedef unsigned long long u64;
__device__ inline u64 entry(float v, int i) { return (u64)sort_key(v) << 32 | ~(uint32_t)i; }
__device__ inline float entry_value(u64 e) { return from_key((uint32_t)(e >> 32)); }
__device__ inline int entry_index(u64 e) { return (int)~(uint32_t)e; }

// What a wave has kept of the values it was offered (a superset of its part of the k best), in the wave's LDS slice, and
// the bound a new entry has to pass: above tv, or equal to it at an index below ti.
struct TopList {
  u64* e;
  int k, cnt;
  float tv;
  int ti;

  // indices at end or beyond never pass (padding)
  __device__ void init(u64* e_, int k_, int end) {
    e = e_; k = k_; cnt = 0;
    tv = neg_inf(); ti = end;
  }
  __device__ bool passes(float v, int i) const { return v > tv || (v == tv && i < ti); }
  // at least k values of the row are known to be >= b
  __device__ void bound(float b, int end) {
    if (b > tv) {
      tv = b;
      ti = end;
    }
  }
  // Keeps the k best: an entry's place is the number of entries above it.
  __device__ void prune() {
    const int lane = threadIdx.x & 63;
    wave_fence();
    const u64 e0 = lane < cnt ? e[lane] : 0, e1 = lane + 64 < cnt ? e[lane + 64] : 0;
    int r0 = 0, r1 = 0;
#pragma unroll 4
    for (int j = 0; j < cnt; ++j) {
      const u64 o = e[j];
      r0 += o > e0;
      r1 += o > e1;
    }
    wave_fence();
    if (lane < cnt && r0 < k) e[r0] = e0;
    if (lane + 64 < cnt && r1 < k) e[r1] = e1;
    wave_fence();
    if (cnt >= k) {
      cnt = k;
      tv = entry_value(e[k - 1]);
      ti = entry_index(e[k - 1]);
    }
  }
  // Whether a lane with a value of v at index i0 or later may pass: the tie with the bound only below its index.
  __device__ bool may_pass(float v, int i0) const { return i0 < ti ? v >= tv : v > tv; }
  // one value of the lanes that have one; after a prune the list has room for a whole ballot
  __device__ void offer(bool have, float v, int i) {
    if (cnt > LP_CAP - 64) prune();
    const bool in = have && passes(v, i);
    const u64 mask = __ballot(in);
    if (in)
      e[cnt + __builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0))] = entry(v, i);
    cnt += __popcll(mask);
  }
};

// A value that at least k of the wave's 64 lanes reach with v (k <= 64): the k-th largest lane value cut to its upper
// 16 key bits, by bisection on ballots.
__device__ inline float kth_bound(float v, int k) {
  const uint32_t key = sort_key(v);
  uint32_t t = 0;
#pragma unroll 4
  for (uint32_t b = 1u << 31; b >= 1u << 16; b >>= 1)
    if (__popcll(__ballot(key >= (t | b))) >= k) t |= b;
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

// Workspace of one (row, split): m, s, u, s without its largest term; of each given token the count of values above it and, from the split
// that holds it, its value; the list of k entries, 8-byte aligned.
__host__ __device__ inline size_t part_floats(int n_ids, int k) { return 4 + 2 * (size_t)n_ids + 2 * (size_t)k; }

template <int WAVES>
struct RowShared {
  u64 list[WAVES][LP_CAP];   // by wave
  u64 all[WAVES * 64];       // what is left of them at the end, in any order
  float m[WAVES], s[WAVES], u[WAVES];
  float rest;                // the s of the wave that holds the maximum without it
  int n;                     // entries of all
  float gmax[64];            // largest value seen by each of 64 groups of lanes
  int rank[WAVES][LP_MAX_IDS];
};

// The waves' statistics as one, in every thread; `first`: the first wave that holds the maximum, sx: s without that wave's.
template <int WAVES>
__device__ inline Stat merge_stats(const RowShared<WAVES>& sh, int& first, float& sx) {
  Stat st;
#pragma unroll
  for (int o = 0; o < WAVES; ++o) st.m = fmaxf(st.m, sh.m[o]);
  first = -1;
  sx = 0.f;
#pragma unroll
  for (int o = 0; o < WAVES; ++o) {
    Stat x;
    x.m = sh.m[o]; x.s = sh.s[o]; x.u = sh.u[o];
    const bool is = first < 0 && x.s > 0.f && x.m == st.m;
    first = is ? o : first;
    x.raise(st.m);
    st.s += x.s;
    st.u += x.u;
    sx += is ? 0.f : x.s;
  }
  return st;
}

// The wave's list, at most 64 entries of it, into sh.all.
template <int WAVES>
__device__ inline void give_list(RowShared<WAVES>& sh, TopList& top) {
  const int lane = threadIdx.x & 63;
  if (top.cnt > 64) top.prune();
  int base = 0;
  if (lane == 0) base = atomicAdd(&sh.n, top.cnt);
  base = __builtin_amdgcn_readfirstlane(base);
  wave_fence();
  if (lane < top.cnt) sh.all[base + lane] = top.e[lane];
}

// The k best of sh.all: every entry counts the entries above it and, if fewer than k, takes that place, whatever the
// order they lie in.  put(place, entry)
template <int WAVES, class F>
__device__ inline void best_of_all(const RowShared<WAVES>& sh, int k, F put) {
  const int n = sh.n;
  for (int t = threadIdx.x; t < n; t += 64 * WAVES) {
    const u64 e = sh.all[t];
    int r = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) r += sh.all[j] > e;
    if (r < k) put(r, e);
  }
}

// The row's outputs: its statistics, r the sum without its largest term.  ln S = log1p(r): where one token is all but
// certain, 1 + r in f32 would lose r, which its log probability and the entropy are made of.
struct RowOut {
  bool nan, empty;
  float m, u, s, ls;
  __device__ RowOut(const Stat& st, float r) : m(st.m), u(st.u), s(st.s) {
    nan = !(s == s);         // an infinite logit makes s NaN as well
    empty = s == 0.f;
    ls = log1pf(r);
  }
  __device__ float lp(float v) const {
    return nan ? __builtin_nanf("") : empty ? neg_inf() : (v - m) - ls;
  }
  __device__ void stats(const LogprobArgs& a, int row) const {
    a.lse[row] = nan ? __builtin_nanf("") : empty ? neg_inf() : m + ls;
    a.entropy[row] = nan ? __builtin_nanf("") : empty ? 0.f : ls - u / s;
  }
  __device__ void token(const LogprobArgs& a, int row, int j, bool in, float v, int above) const {
    const size_t o = (size_t)row * a.n_ids + j;
    a.token_lp[o] = nan || in ? lp(v) : neg_inf();
    if (a.ranks) a.ranks[o] = nan || !in ? -1 : 1 + above;
  }
  __device__ void top(const LogprobArgs& a, int row, int place, u64 e) const {
    const size_t o = (size_t)row * a.top + place;
    a.top_lp[o] = lp(entry_value(e));
    a.top_ids[o] = nan ? -1 : entry_index(e);
  }
};

__device__ inline long long id_at(const LogprobArgs& a, size_t i) {
  return a.ids64 ? static_cast<const long long*>(a.ids)[i] : static_cast<const int*>(a.ids)[i];
}

// One (row, split): values [split * chunk, min(V, + chunk)) of the row, chunk a multiple of LP_TILE.  The waves take its
// tiles in turn.  Given token j belongs to lane j of every wave.
template <typename T, int WAVES, bool SPLIT>
__global__ __launch_bounds__(64 * WAVES, WAVES == 16 ? 4 : 6) void logprob_rows_kernel(LogprobArgs a, int splits, int chunk,
                                                                                       float* part) {
  using L = Load<T>;
  constexpr int VEC = L::VEC, NV = LP_E / VEC, TH = 64 * WAVES;
  __shared__ RowShared<WAVES> sh;
  const int row = SPLIT ? blockIdx.x / splits : blockIdx.x, split = SPLIT ? blockIdx.x - row * splits : 0;
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
  int id = -1, above = 0;
  float iv = __builtin_inff();
  if (lane < a.n_ids) {
    const long long i = id_at(a, (size_t)row * a.n_ids + lane);
    if (i >= 0 && i < a.V) {
      id = (int)i;
      iv = L::f(x[id]);
    }
  }
  if (threadIdx.x == 0) sh.n = 0;          // read after the loop's barrier
  float lmax = neg_inf();
  auto publish = [&] {
    float g = lmax;
    g = fmaxf(g, dpp<0xb1>(g));
    g = fmaxf(g, dpp<0x4e>(g));
    if constexpr (WAVES >= 8) g = fmaxf(g, dpp<0x141>(g));
    if constexpr (WAVES >= 16) g = fmaxf(g, dpp<0x140>(g));
    constexpr int LANES = WAVES;           // of a group
    static_assert(LANES == 4 || LANES == 8 || LANES == 16, "groups are quads, half rows or rows");
    if (lane % LANES == 0) *const_cast<volatile float*>(&sh.gmax[threadIdx.x / LANES]) = g;
  };

  Stat st;
  TopList top;
  top.init(sh.list[w], a.top, c1);
  for (bool first = true; first || t0 < c1; first = false, t0 += WAVES * LP_TILE) {
    float v[LP_E];
    if (t0 + LP_TILE <= c1) {
#pragma unroll
      for (int q = 0; q < NV; ++q) L::unpack(raw[q], v + q * VEC);
    } else {   // the last tile, or a first one of nothing
#pragma unroll
      for (int e = 0; e < LP_E; ++e) {
        const int i = at(t0, e);
        v[e] = i < c1 ? L::f(x[i]) : neg_inf();
      }
    }
    const int tn = t0 + WAVES * LP_TILE;
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

    for (int j = 0; a.ranks && j < a.n_ids; ++j) {
      const float jv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(iv), j));
      const int ji = __builtin_amdgcn_readlane(id, j);
      int n = 0;
      if (t0 + LP_TILE <= ji) {            // every value here has a lower index
#pragma unroll
        for (int e = 0; e < LP_E; ++e) n += __popcll(__ballot(v[e] >= jv));
      } else if (t0 > ji) {
#pragma unroll
        for (int e = 0; e < LP_E; ++e) n += __popcll(__ballot(v[e] > jv));
      } else {
#pragma unroll
        for (int e = 0; e < LP_E; ++e) n += __popcll(__ballot(v[e] > jv || (v[e] == jv && at(t0, e) < ji)));
      }
      above += lane == j ? n : 0;
    }

    if (a.top) {
      // Lower bounds of the k-th best, so that few values of a row are ever listed.  64 groups of lanes (rows of 16 in
      // 16 waves, halves of them in 8, quads in 4) publish the largest value each has seen; the k-th largest of those is reached by k
      // values: of 16384 random ones about 24 reach the bound for k = 20.  A wave takes a new bound only where a value of
      // its tile passes the last one.  Other waves' entries may be older: lower, still bounds.
      lmax = fmaxf(lmax, tm);
      if (first) {
        // where less than k groups may have a value: the wave's own lanes
        if (c1 - c0 < WAVES * LP_TILE) top.bound(kth_bound(tm, a.top), c1);
        publish();
        __syncthreads();
      }
      if (__ballot(top.may_pass(tm, t0))) {
        if (!first) publish();
        top.bound(kth_bound(*const_cast<volatile float*>(&sh.gmax[lane]), a.top), c1);
        // The lane's values that may pass: mostly one, its largest (the first of equals); any others are read again, as v
        // has no index.
        uint32_t some = 0, best = 1u << LP_E;
#pragma unroll
        for (int e = LP_E - 1; e >= 0; --e) {
          some |= (uint32_t)top.may_pass(v[e], t0) << e;
          best = v[e] == tm ? 1u << e : best;
        }
        float cv = tm;
        uint32_t bit = some & best;
        while (__ballot(some)) {
          const int i = at(t0, __builtin_ctz(bit | 1u << LP_E));
          top.offer(bit && i < c1, cv, i);
          some &= ~bit;
          bit = some & (0u - some);
          const int next = at(t0, __builtin_ctz(bit | 1u << LP_E));
          if (bit && next < c1) cv = L::f(x[next]);
        }
      }
    }
  }

  const int holder = st.join();
  const float own = st.s;                  // the lane's
  st.s = wave_sum(st.s);
  st.u = wave_sum(st.u);
  if (lane == 0) {
    sh.m[w] = st.m;
    sh.s[w] = st.s;
    sh.u[w] = st.u;
  }
  if (a.top) give_list(sh, top);
  if (lane < a.n_ids) sh.rank[w][lane] = above;
  __syncthreads();
  if (w == 0 && lane < a.n_ids) {
    above = 0;
#pragma unroll
    for (int o = 0; o < WAVES; ++o) above += sh.rank[o][lane];
  }
  int fw;
  float r;
  const Stat all = merge_stats(sh, fw, r);
  if (all.s < 1.25f && all.s > 0.f) {
    // One term outweighs the others, and its lane's sum has lost what they are (above 1.25 s - 1 is exact to 4e-7).  Its
    // wave adds them again without it.
    if (w == fw) {
      float p = lane == holder ? 0.f : own;
      const int mine = c0 + w * LP_TILE;
      for (int q = lane; q < (c1 - mine + WAVES * LP_TILE - 1) / (WAVES * LP_TILE) * LP_E; q += 64) {
        const int e = q % LP_E, i = mine + q / LP_E * (WAVES * LP_TILE) + (e / VEC) * 64 * VEC + holder * VEC + e % VEC;
        const float v = i < c1 ? L::f(x[i]) : neg_inf();
        p += v < all.m ? fast_exp2((v - all.m) * LOG2E) : 0.f;
      }
      p = wave_sum(p);
      if (lane == 0) sh.rest = p;
    }
    __syncthreads();
    r += sh.rest;
  } else {
    r = all.s - 1.f;
  }
  if constexpr (!SPLIT) {
    const RowOut out(all, r);
    if (threadIdx.x == 0) out.stats(a, row);
    if (w == 0 && lane < a.n_ids) out.token(a, row, lane, id >= 0, iv, above);
    if (out.nan) {
      for (int j = threadIdx.x; j < a.top; j += TH) out.top(a, row, j, 0);
    } else if (a.top) {
      best_of_all(sh, a.top, [&](int place, u64 e) { out.top(a, row, place, e); });
    }
  } else {
    float* p = part + (size_t)blockIdx.x * part_floats(a.n_ids, a.top);
    if (threadIdx.x == 0) {
      p[0] = all.m;
      p[1] = all.s;
      p[2] = all.u;
      p[3] = r;
    }
    if (w == 0 && lane < a.n_ids) {
      reinterpret_cast<int*>(p)[4 + 2 * lane] = above;
      p[5 + 2 * lane] = iv;
    }
    u64* pe = reinterpret_cast<u64*>(p + 4 + 2 * a.n_ids);
    if (a.top && threadIdx.x < a.top && threadIdx.x >= sh.n) pe[threadIdx.x] = 0;   // below every value's entry
    if (a.top) best_of_all(sh, a.top, [&](int place, u64 e) { pe[place] = e; });
  }
}

// One row from its splits' workspace entries, in a fixed order.  Four waves: the splits are few.
__global__ __launch_bounds__(256) void logprob_merge_kernel(LogprobArgs a, int splits, const float* part) {
  __shared__ RowShared<4> sh;
  __shared__ float rest[4];                // a wave's s without the largest term
  const int row = blockIdx.x, lane = threadIdx.x & 63;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const size_t pf = part_floats(a.n_ids, a.top);
  const float* p = part + (size_t)row * splits * pf;

  // a thread a split (at most one workgroup a CU splits a row); the first split that holds the maximum gives its sum
  // without it
  Stat st;
  float sx = 0.f;
  if (threadIdx.x < splits) {
    const float* e = p + threadIdx.x * pf;
    st.m = e[0]; st.s = e[1]; st.u = e[2];
    sx = e[3];
  }
  int above = 0;
  bool in = false;
  float iv = 0.f;
  if (w == 0 && lane < a.n_ids) {
    const long long i = id_at(a, (size_t)row * a.n_ids + lane);
    in = i >= 0 && i < a.V;
    iv = p[5 + 2 * lane];
    for (int q = 0; q < splits; ++q) above += reinterpret_cast<const int*>(p + q * pf)[4 + 2 * lane];
  }
  if (threadIdx.x == 0) sh.n = 0;
  __syncthreads();
  TopList top;
  top.init(sh.list[w], a.top, a.V);
  if (a.top) {
    const int k = a.top, n = splits * k;
    auto get = [&](int i) {
      const int s = i / k, j = i - s * k;
      return reinterpret_cast<const u64*>(p + s * pf + 4 + 2 * a.n_ids)[j];
    };
    for (int i = w * 64; i < n; i += 256) {
      const u64 e = i + lane < n ? get(i + lane) : 0;
      const float v = e ? entry_value(e) : neg_inf();
      const int at = e ? entry_index(e) : a.V;
      if (i == w * 64) top.bound(kth_bound(v, k), a.V);
      top.offer(e != 0, v, at);
    }
    give_list(sh, top);
  }
  const int holder = st.join();
  sx = wave_sum(lane == holder ? sx : st.s);
  st.s = wave_sum(st.s);
  st.u = wave_sum(st.u);
  if (lane == 0) {
    sh.m[w] = st.m;
    sh.s[w] = st.s;
    sh.u[w] = st.u;
    rest[w] = sx;
  }
  __syncthreads();
  int fw;
  float r;
  const Stat all = merge_stats(sh, fw, r);
  r += fw < 0 ? 0.f : rest[fw];
  const RowOut out(all, r);
  if (threadIdx.x == 0) out.stats(a, row);
  if (w == 0 && lane < a.n_ids) out.token(a, row, lane, in, iv, above);
  if (out.nan) {
    for (int j = threadIdx.x; j < a.top; j += 256) out.top(a, row, j, 0);
  } else if (a.top) {
    best_of_all(sh, a.top, [&](int place, u64 e) { out.top(a, row, place, e); });
  }
}

template <typename T>
int launch_t(const LogprobArgs& a, void* ws, hipStream_t st) {
  const LogprobPlan pl = logprob_plan(a.T, a.V);
  const int tiles = (a.V + LP_TILE - 1) / LP_TILE;
  const int chunk = (tiles + pl.splits - 1) / pl.splits * LP_TILE;
  float* part = static_cast<float*>(ws);
  if (pl.splits > 1) {
    hipLaunchKernelGGL((logprob_rows_kernel<T, 16, true>), dim3((unsigned)(a.T * pl.splits)), dim3(1024), 0, st, a, pl.splits,
                       chunk, part);
    hipLaunchKernelGGL(logprob_merge_kernel, dim3(a.T), dim3(256), 0, st, a, pl.splits, part);
  } else if (pl.waves == 8) {
    hipLaunchKernelGGL((logprob_rows_kernel<T, 8, false>), dim3(a.T), dim3(512), 0, st, a, 1, chunk, nullptr);
  } else if (pl.waves == 16) {
    hipLaunchKernelGGL((logprob_rows_kernel<T, 16, false>), dim3(a.T), dim3(1024), 0, st, a, 1, chunk, nullptr);
  } else {
    hipLaunchKernelGGL((logprob_rows_kernel<T, 4, false>), dim3(a.T), dim3(256), 0, st, a, 1, chunk, nullptr);
  }
  MK_HIP_CHECK(hipGetLastError());
  return MK_OK;
}

// ------------------------------------------------------------------------------------------------ from hidden states
// The rows' log probabilities from the statistics the LM head product leaves (launch_gemm_lse): a workgroup has 32 rows,
// whole cache lines of the statistics.  Its waves first make the given tokens' logits, dot products of f32 sums, a wave
// each; then 32 threads a row merge its `tiles` entries.
constexpr int HF_ROWS = 32, HF_WAVES = 16, HF_PARTS = 64 * HF_WAVES / HF_ROWS;

__global__ __launch_bounds__(64 * HF_WAVES) void head_finish_kernel(HeadLogprobArgs a, int tiles, const float* part) {
  __shared__ float sh[3][HF_WAVES][HF_ROWS];
  __shared__ float dot[HF_ROWS * LP_MAX_IDS];
  __shared__ double lse[HF_ROWS];
  const int r = threadIdx.x % HF_ROWS, q = threadIdx.x / HF_ROWS, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int row0 = blockIdx.x * HF_ROWS, row = row0 + r, given = min(HF_ROWS, a.T - row0) * a.n_ids;
  auto id_of = [&](int i) {
    const size_t o = (size_t)row0 * a.n_ids + i;
    return a.ids64 ? static_cast<const long long*>(a.ids)[o] : static_cast<const int*>(a.ids)[o];
  };
  for (int i = w; i < given; i += HF_WAVES) {
    const long long id = id_of(i);
    const bool in = id >= 0 && id < a.V;
    const uint16_t *h = a.hidden + (size_t)(row0 + i / a.n_ids) * a.H, *wt = a.weight + (size_t)(in ? id : 0) * a.H;
    float d = 0.f;
    for (int k = lane * 8; k < a.H; k += 512) {
      const u32x4 hv = *reinterpret_cast<const u32x4*>(h + k), wv = *reinterpret_cast<const u32x4*>(wt + k);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        d = fmaf(bf_lo(hv[e]), bf_lo(wv[e]), d);
        d = fmaf(bf_hi(hv[e]), bf_hi(wv[e]), d);
      }
    }
    d = wave_sum(d);
    if (lane == 0) dot[i] = d;
  }
  // log2 units: m a reference exponent, as the tiles' are
  float m = NEG_MAX, s = 0.f, u = 0.f;
  auto merge = [&](float m2, float s2, float u2) {
    const float mn = fmaxf(m, m2), d1 = fmaxf(m - mn, -1e4f), d2 = fmaxf(m2 - mn, -1e4f);
    const float f1 = fast_exp2(d1), f2 = fast_exp2(d2);
    u = f1 * fmaf(d1, s, u) + f2 * fmaf(d2, s2, u2);
    s = f1 * s + f2 * s2;
    m = mn;
  };
  const float* p = part + min(row, a.T - 1);
#pragma unroll 8
  for (int t = q; t < tiles; t += HF_PARTS) {
    const float* e = p + (size_t)t * 3 * a.T;
    merge(e[0], e[a.T], e[2 * (size_t)a.T]);
  }
#pragma unroll
  for (int o = HF_ROWS; o <= 32; o <<= 1) merge(__shfl_xor(m, o), __shfl_xor(s, o), __shfl_xor(u, o));
  if (lane < HF_ROWS) {
    sh[0][w][r] = m;
    sh[1][w][r] = s;
    sh[2][w][r] = u;
  }
  __syncthreads();
  if (q == 0) {
#pragma unroll
    for (int o = 1; o < HF_WAVES; ++o) merge(sh[0][o][r], sh[1][o][r], sh[2][o][r]);
    const double ln2 = 0.6931471805599453, l2 = (double)log2f(s);
    lse[r] = ((double)m + l2) * ln2;
    if (row < a.T) {
      a.lse[row] = (float)lse[r];
      a.entropy[row] = (float)((l2 - (double)(u / s)) * ln2);
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < given; i += 64 * HF_WAVES) {
    const long long id = id_of(i);
    const double l = lse[i / a.n_ids];
    // a NaN row is NaN for every id; rounding may put a certain token a step above 0
    a.token_lp[(size_t)row0 * a.n_ids + i] =
        !(l == l) ? __builtin_nanf("") : id >= 0 && id < a.V ? fminf((float)((double)dot[i] - l), 0.f) : neg_inf();
  }
}

// Rows of a pass over the vocabulary that keeps statistics only: 16384, 100 MB of them at V = 130560.
constexpr int HEAD_PASS = 16384;

}  // namespace

size_t logprob_scratch_bytes(int T, int V, int n_ids, int top) {
  const int splits = logprob_plan(T, V).splits;
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

size_t head_logprob_scratch_bytes(int T, int V, int n_ids) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  if (head_logprobs_stored(T)) return up((size_t)T * V * sizeof(float)) + logprob_scratch_bytes(T, V, n_ids, 0);
  return (size_t)((V + LSE_ROWS - 1) / LSE_ROWS) * 3 * std::min(T, HEAD_PASS) * sizeof(float);
}

int launch_head_logprobs(const HeadLogprobArgs& a, void* ws, hipStream_t st) {
  // the products take operands under 4 GiB: the vocabulary in slices of whole tiles
  const int slice = (int)std::min<size_t>(a.V, ((((size_t)1 << 32) - 1) / ((size_t)a.H * 2)) / LSE_ROWS * LSE_ROWS);
  MK_REQUIRE(slice >= 1, "lm_head_logprobs: H too large");
  GemmArgs g{};
  g.in = GemmIn::BF16;
  g.K = g.lda = g.ldb = a.H;
  if (head_logprobs_stored(a.T)) {
    float* logits = static_cast<float*>(ws);
    g.epi = Epi::F32;
    g.A = a.hidden;
    g.M = a.T;
    g.ldo = a.V;
    for (int v0 = 0; v0 < a.V; v0 += slice) {
      g.B = a.weight + (size_t)v0 * a.H;
      g.N = std::min(slice, a.V - v0);
      g.out = logits + v0;
      const int rc = launch_lm_head(g, st);
      if (rc) return rc;
    }
    LogprobArgs l{logits, (size_t)a.V, 0, a.ids, a.ids64, a.n_ids, a.T, a.V, 0, a.token_lp, nullptr, nullptr, nullptr,
                  a.entropy, a.lse};
    return launch_logprobs(l, static_cast<char*>(ws) + ((size_t)a.T * a.V * sizeof(float) + 255) / 256 * 256, st);
  }
  const int tiles = (a.V + LSE_ROWS - 1) / LSE_ROWS;
  for (int t0 = 0; t0 < a.T; t0 += HEAD_PASS) {
    HeadLogprobArgs h = a;
    h.T = std::min(HEAD_PASS, a.T - t0);
    h.hidden = a.hidden + (size_t)t0 * a.H;
    const size_t at = (size_t)t0 * a.n_ids;
    h.ids = static_cast<const char*>(a.ids) + at * (a.ids64 ? 8 : 4);
    h.token_lp = a.token_lp + at;
    h.entropy = a.entropy + t0;
    h.lse = a.lse + t0;
    g.B = h.hidden;
    g.N = g.ldo = h.T;
    for (int v0 = 0; v0 < a.V; v0 += slice) {
      g.A = a.weight + (size_t)v0 * a.H;
      g.M = std::min(slice, a.V - v0);
      g.out = static_cast<float*>(ws) + (size_t)(v0 / LSE_ROWS) * 3 * h.T;
      const int rc = launch_gemm_lse(g, st);
      if (rc) return rc;
    }
    hipLaunchKernelGGL(head_finish_kernel, dim3((h.T + HF_ROWS - 1) / HF_ROWS), dim3(64 * HF_WAVES), 0, st, h, tiles,
                       static_cast<const float*>(ws));
    MK_HIP_CHECK(hipGetLastError());
  }
  return MK_OK;
}

}  // namespace mk
