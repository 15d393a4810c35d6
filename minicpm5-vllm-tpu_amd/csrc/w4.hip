// 4-bit weights with group scales (gfx950): quantisation, its inverse, and products with few rows of activations.
//
// Format.  W (N, K): along K every row is cut into groups of `group` (32, 64 or 128) values, the last one filled up with
// zeros; group g of row n has the scale s = bf16(amax / 7) and codes c = round_half_even(w / s) in [-7, 7], W ~ c s.
// A group whose amax / 7 is below the smallest normal number has s = 0 and codes 0; a group with an infinity or a NaN
// has s = NaN.  Stored are s (bf16) and 4 bits u a value, 8 + c at even k and 8 - c at odd k (the product's reason).
//
// Layout.  Blocks of 16 rows x 128 values of K, 1 KB, [row block][K block]: lane l of a wave has the 16 bytes at 16 l,
// word t of them row l % 16, values 32 t + 8 (l / 16) .. + 7 -- operand A of the 16x16x32 MFMA t of the block, so the
// product reads weights as whole-wave 1 KB loads and moves nothing between lanes.  Value 2 p of a word is nibble p, value
// 2 p + 1 nibble 4 + p of the word rotated right by 3: rotated right by 4 p the word has both where the mantissas of two
// bf16 take them, so a rotation (none for p = 0) and one and-or make a pair.  Rows and values past N and K hold code 0
// (scale 0).  Scales: [row block][K block][row / 4][group of the block][row % 4], so a lane's four accumulator rows have
// theirs next to each other.
#include <algorithm>

#include "kernels.h"
#include "mk_common.h"

namespace mk {

namespace {

constexpr int W4_ROWS = 16, W4_K = 128;

// ------------------------------------------------------------------------------------------------ quantisation
// Bytes bound both directions (2 read and 1/2 written a value, and back): the 130560 x 1536 head 98 us each, 5.1 TB/s.  A wave makes blocks of 16 rows x 128 values: lane l reads the four
// 16-byte pieces of row l % 16 that its 16 bytes of codes come from.
typedef uint16_t h8 __attribute__((ext_vector_type(8), aligned(2)));

__device__ inline float shfl_max(float v, int mask) { return fmaxf(v, __shfl_xor(v, mask)); }

template <int GROUP>
__global__ __launch_bounds__(256) void w4_quantize_kernel(const uint16_t* __restrict__ w, size_t ldw, int N, int K, int nkb,
                                                          long blocks, uint8_t* __restrict__ codes,
                                                          uint16_t* __restrict__ scales) {
  constexpr int GPB = W4_K / GROUP;   // groups of a block
  const int lane = threadIdx.x & 63, r = lane & 15, kq = lane >> 4;
  const long b = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= blocks) return;
  const long rb = b / nkb;
  const int kb = (int)(b - rb * nkb);
  const long n = rb * W4_ROWS + r;
  const uint16_t* row = w + (n < N ? n : 0) * ldw;
  h8 raw[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int k = kb * W4_K + 32 * t + 8 * kq;
    if (n < N && k + 8 <= K) {
      raw[t] = *reinterpret_cast<const h8*>(row + k);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) raw[t][i] = n < N && k + i < K ? row[k + i] : 0;
    }
  }
  // |w| as bits: order of the non-negative floats, and everything from 0x7f80 on is not finite
  uint32_t am[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    am[t] = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) am[t] = max(am[t], (uint32_t)raw[t][i] & 0x7fffu);
    am[t] = max(am[t], (uint32_t)__shfl_xor((int)am[t], 16));
    am[t] = max(am[t], (uint32_t)__shfl_xor((int)am[t], 32));
  }
  uint16_t sc[GPB];
  u32x4 out;
#pragma unroll
  for (int g = 0; g < GPB; ++g) {
    constexpr int TG = 4 / GPB;
    uint32_t a = am[g * TG];
#pragma unroll
    for (int t = 1; t < TG; ++t) a = max(a, am[g * TG + t]);
    const float q = bf2f((uint16_t)a) / 7.f;
    sc[g] = a >= 0x7f80u ? 0x7fc0 : q < 1.17549435e-38f ? 0 : f2bf(q);
    const float s = bf2f(sc[g]);
    // w / s, correctly rounded where it matters: the residual of the first estimate is exact, so that a quotient halfway
    // between two codes comes out exactly.  Tiny groups are scaled up for it: their residuals would be subnormal.
    const float f = s < 0x1p-60f ? 0x1p64f : 1.f, sf = s * f, inv = s > 0.f ? 1.f / sf : 0.f;
#pragma unroll
    for (int t = g * TG; t < (g + 1) * TG; ++t) {
      uint32_t word = 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float v = bf2f(raw[t][i]) * f;
        float c = v * inv;
        c = fmaf(fmaf(-c, sf, v), inv, c);
        const int q = (int)fminf(fmaxf(rintf(c), -7.f), 7.f), u = i % 2 ? 8 - q : 8 + q;
        word |= (uint32_t)u << (4 * (i / 2) + 16 * (i % 2));
      }
      out[t] = __builtin_rotateleft32(word, 3);
    }
  }
  reinterpret_cast<u32x4*>(codes)[(size_t)b * 64 + lane] = out;
  if (kq == 0) {
    uint16_t* sp = scales + (size_t)b * W4_ROWS * GPB + (r >> 2) * 4 * GPB + (r & 3);
#pragma unroll
    for (int g = 0; g < GPB; ++g) sp[4 * g] = sc[g];
  }
}

template <int GROUP, bool F32>
__global__ __launch_bounds__(256) void w4_dequantize_kernel(const uint8_t* __restrict__ codes,
                                                            const uint16_t* __restrict__ scales, int N, int K, int nkb,
                                                            long blocks, void* __restrict__ out, size_t ldo) {
  constexpr int GPB = W4_K / GROUP;
  const int lane = threadIdx.x & 63, r = lane & 15, kq = lane >> 4;
  const long b = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (b >= blocks) return;
  const long rb = b / nkb;
  const int kb = (int)(b - rb * nkb);
  const long n = rb * W4_ROWS + r;
  if (n >= N) return;
  const u32x4 c = reinterpret_cast<const u32x4*>(codes)[(size_t)b * 64 + lane];
  const uint16_t* sp = scales + (size_t)b * W4_ROWS * GPB + (r >> 2) * 4 * GPB + (r & 3);
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const uint32_t word = __builtin_rotateright32(c[t], 3);
    const float s = bf2f(sp[4 * (t * GPB / 4)]);
    const int k = kb * W4_K + 32 * t + 8 * kq;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int u = word >> (4 * (i / 2) + 16 * (i % 2)) & 15;
      v[i] = (float)(i % 2 ? 8 - u : u - 8) * s;
    }
    if constexpr (F32) {
      float* o = static_cast<float*>(out) + n * ldo + k;
      typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
      if (k + 8 <= K) {
        reinterpret_cast<f4*>(o)[0] = f4{v[0], v[1], v[2], v[3]};
        reinterpret_cast<f4*>(o)[1] = f4{v[4], v[5], v[6], v[7]};
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < K) o[i] = v[i];
      }
    } else {
      uint16_t* o = static_cast<uint16_t*>(out) + n * ldo + k;
      h8 p;
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = f2bf(v[i]);
      if (k + 8 <= K) {
        *reinterpret_cast<h8*>(o) = p;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (k + i < K) o[i] = p[i];
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------ product
// y (M, N) = x (M, K) (c s)^T, f32 accumulation.  For few rows the weight stream is the bound: the 130560 x 1536 head takes
// 22.3 us for one row (4.65 TB/s, what a large copy reaches), 27 for 16.  Beyond, a block of 16 x 128 weights costs a wave
// 28 VALU operations of unpacking, and per group and 16 rows of x four to start, four to scale the accumulators and two or
// more MFMAs, which no longer hide behind the stream: 48 rows 38.7 us, 64 rows 51.2 (K = 2048: 40 rows 48, 64 rows 56).
// Small weights are bound by latency, one pass of loads after another (1536 x 4608, one row 5.3 us).
//
// u becomes a bf16 number by standing in mantissa bits 3 - 6 of 16.0 at even k and of -16.0 at odd k: 16 + u = 24 + c and
// -(16 + u) = c - 24, exact.  What is too much is 24 d, d the even x less the odd ones of a group, and taken off before
// it is added: the group's accumulators start at -24 d (f32) and end at sum c x, which is scaled by s (f32) into the row's
// total.  The roundings between are relative to 24 |d|, which x of one sign do not raise (with + 24 at every k, x uniform
// in 0 .. 1 and groups of 128 gave 2.2e-6 of the result's norm).
//
// x is staged in LDS, as many blocks of 128 values of K at a time as fit (zeros past K), each block its rows of 256 bytes,
// 16-byte piece p of row m at p ^ (m % 16) so that the 16 rows of an operand read are on distinct banks; its group sums are
// made on the way.  MFMA columns past the rows hold whatever lies there, columns do not mix and theirs are not stored.  A
// workgroup's waves are sets of kw: a set has R row blocks, whose K blocks are dealt to its waves, their totals added in
// wave order at the end.  A wave loads the next of its blocks while it multiplies one.
constexpr int w4_waves(int mg) { return mg == 1 ? 8 : 16; }
constexpr int w4_xb(int mg) { return w4_waves(mg) * 8192; }   // LDS bytes of x, and of its sums (groups of 32)
constexpr int w4_sb(int mg) { return w4_xb(mg) / 16; }

// mask: 0x00780078, the mantissa bits of the codes; one: 0xc1804180, bf16 16.0 and -16.0
__device__ inline uint32_t pair_bf16(uint32_t w, int p, uint32_t mask, uint32_t one) {
  return (__builtin_rotateright32(w, 4 * p) & mask) | one;
}

template <int MG, int R, int GROUP>
__global__ __launch_bounds__(64 * w4_waves(MG), 4) void w4_gemm_kernel(W4GemmArgs a, int nkb, int kw, int bpc) {
  constexpr int W4_WAVES = w4_waves(MG), W4_TH = 64 * W4_WAVES, W4_XB = w4_xb(MG), W4_SB = w4_sb(MG);
  constexpr int GPB = W4_K / GROUP, ROWS = 16 * MG;
  static_assert(R > 1 || W4_WAVES * MG * 64 * 16 <= W4_XB, "the totals of a dealt K fit where x was");
  __shared__ __attribute__((aligned(16))) char smem[W4_XB + W4_SB];
  const int lane = threadIdx.x & 63, c16 = lane & 15, kq = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int kwi = w % kw;
  const int mrow0 = blockIdx.y * ROWS, M = std::min(ROWS, a.M - mrow0);
  const uint16_t* x = a.x + (size_t)mrow0 * a.ldx;
  const long nrb = (a.N + W4_ROWS - 1) / W4_ROWS;
  const long rb0 = ((long)blockIdx.x * (W4_WAVES / kw) + w / kw) * R;
  float* sums = reinterpret_cast<float*>(smem + W4_XB);
  const int ppr = bpc * 16;                   // 16-byte pieces of a staged row
  const int RA = MG == 1 ? M : ROWS;          // rows of a staged block

  f32x4 tot[R][MG];
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int m = 0; m < MG; ++m) tot[r][m] = f32x4{0.f, 0.f, 0.f, 0.f};

  // kept in registers the compiler cannot see through: as literals they would make an and and an or of the and-or
  uint32_t mask = 0x00780078u, one = 0xc1804180u;
  asm volatile("" : "+s"(mask), "+v"(one));

  typedef uint16_t SC __attribute__((ext_vector_type(4 * GPB)));
  u32x4 cw[R];
  SC sc[R];
  auto load = [&](int kb) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const size_t b = (size_t)std::min(rb0 + r, nrb - 1) * nkb + kb;
      cw[r] = reinterpret_cast<const u32x4*>(a.codes)[b * 64 + lane];
      sc[r] = *reinterpret_cast<const SC*>(a.scales + b * W4_ROWS * GPB + kq * 4 * GPB);
    }
  };
  // this lane's operand row (of every 16) and its piece of k-step t in a staged block
  const int xrow = MG == 1 ? std::min(c16, M - 1) : c16;
  int xoff[4];
#pragma unroll
  for (int t = 0; t < 4; ++t) xoff[t] = xrow * 256 + (((4 * t + kq) ^ xrow) & 15) * 16;
  if (kwi < nkb) load(kwi);

  for (int c0 = 0; c0 < nkb; c0 += bpc) {
    if (c0) __syncthreads();   // the last chunk's operand reads are done
    // stage x: thread -> (row, 16-byte piece), the pieces of a row on consecutive lanes, four of a thread's loads on the way
    // together
    for (int i0 = threadIdx.x; i0 < M * ppr; i0 += 4 * W4_TH) {
      h8 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + q * W4_TH, m = i / ppr, k = c0 * W4_K + 8 * (i - m * ppr);
        v[q] = h8{0, 0, 0, 0, 0, 0, 0, 0};
        if (m >= M) continue;
        const uint16_t* xr = x + (size_t)m * a.ldx;
        if (k + 8 <= a.K) {
          v[q] = *reinterpret_cast<const h8*>(xr + k);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (k + e < a.K) v[q][e] = xr[k + e];
        }
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = i0 + q * W4_TH, m = i / ppr, p = i - m * ppr;
        if (m >= M) break;
        *reinterpret_cast<u32x4*>(smem + ((p >> 4) * RA + m) * 256 + ((p ^ m) & 15) * 16) = __builtin_bit_cast(u32x4, v[q]);
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < 8; e += 2) s += bf2f(v[q][e]) - bf2f(v[q][e + 1]);
#pragma unroll
        for (int o = 1; o < GROUP / 8; o <<= 1) s += __shfl_xor(s, o);   // ppr is a multiple of 16: whole groups
        if (p % (GROUP / 8) == 0) sums[(p / (GROUP / 8)) * RA + m] = -24.f * s;
      }
    }
    __syncthreads();
    const int ce = std::min(c0 + bpc, nkb);
    for (int kb = c0 + kwi; kb < ce; kb += kw) {
      const int lb = kb - c0;   // block of the chunk
      u32x4 cb[R];
      SC sb[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        cb[r] = cw[r];
        sb[r] = sc[r];
      }
      if (kb + kw < nkb) load(kb + kw);
#pragma unroll
      for (int g = 0; g < GPB; ++g) {
        f32x4 acc[R][MG];
#pragma unroll
        for (int m = 0; m < MG; ++m) {
          const float z = sums[(lb * GPB + g) * RA + 16 * m + xrow];
#pragma unroll
          for (int r = 0; r < R; ++r) acc[r][m] = f32x4{z, z, z, z};
        }
#pragma unroll
        for (int t = g * 4 / GPB; t < (g + 1) * 4 / GPB; ++t) {
          u32x4 av[R];
#pragma unroll
          for (int r = 0; r < R; ++r)
#pragma unroll
            for (int p = 0; p < 4; ++p) av[r][p] = pair_bf16(cb[r][t], p, mask, one);
#pragma unroll
          for (int m = 0; m < MG; ++m) {
            const u32x4 bv = *reinterpret_cast<const u32x4*>(smem + lb * RA * 256 + xoff[t] + m * 4096);
#pragma unroll
            for (int r = 0; r < R; ++r) acc[r][m] = mfma_bf16_16x16x32(av[r], bv, acc[r][m]);
          }
          if constexpr (MG * R >= 4) __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float s = bf2f(sb[r][4 * g + j]);
#pragma unroll
            for (int m = 0; m < MG; ++m) tot[r][m][j] = fmaf(acc[r][m][j], s, tot[r][m][j]);
          }
      }
    }
  }
  if (kw > 1) {
    __syncthreads();
    f32x4* red = reinterpret_cast<f32x4*>(smem);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int m = 0; m < MG; ++m) red[((w * R + r) * MG + m) * 64 + lane] = tot[r][m];
    __syncthreads();
    if (kwi) return;
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int m = 0; m < MG; ++m)
        for (int o = 1; o < kw; ++o) {
          const f32x4 v = red[(((w + o) * R + r) * MG + m) * 64 + lane];
#pragma unroll
          for (int j = 0; j < 4; ++j) tot[r][m][j] += v[j];
        }
  }
  // accumulator lane: activation row 16 m + l % 16, weight rows 4 (l / 16) .. + 3 of the block
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const long n = (rb0 + r) * W4_ROWS + 4 * kq;
    if (n >= a.N) continue;
#pragma unroll
    for (int m = 0; m < MG; ++m) {
      if (16 * m + c16 >= M) continue;
      const int row = mrow0 + 16 * m + c16;
      const f32x4 v = tot[r][m];
      if (a.out_f32) {
        float* o = static_cast<float*>(a.out) + (size_t)row * a.ldo + n;
        typedef float f4 __attribute__((ext_vector_type(4), aligned(4)));
        if (n + 4 <= a.N) *reinterpret_cast<f4*>(o) = f4{v[0], v[1], v[2], v[3]};
        else
          for (int j = 0; j < 4 && n + j < a.N; ++j) o[j] = v[j];
      } else {
        uint16_t* o = static_cast<uint16_t*>(a.out) + (size_t)row * a.ldo + n;
        typedef uint16_t h4 __attribute__((ext_vector_type(4), aligned(2)));
        if (n + 4 <= a.N) *reinterpret_cast<h4*>(o) = h4{f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])};
        else
          for (int j = 0; j < 4 && n + j < a.N; ++j) o[j] = f2bf(v[j]);
      }
    }
  }
}

template <int MG, int R>
void launch_tile(const W4GemmArgs& a, int nkb, int kw, int bpc, hipStream_t st) {
  const long nrb = (a.N + W4_ROWS - 1) / W4_ROWS, per = (long)w4_waves(MG) / kw * R;
  const dim3 grid((unsigned)((nrb + per - 1) / per), (a.M + 16 * MG - 1) / (16 * MG)), block(64 * w4_waves(MG));
  switch (a.group) {
    case 32: hipLaunchKernelGGL((w4_gemm_kernel<MG, R, 32>), grid, block, 0, st, a, nkb, kw, bpc); break;
    case 64: hipLaunchKernelGGL((w4_gemm_kernel<MG, R, 64>), grid, block, 0, st, a, nkb, kw, bpc); break;
    default: hipLaunchKernelGGL((w4_gemm_kernel<MG, R, 128>), grid, block, 0, st, a, nkb, kw, bpc); break;
  }
}

}  // namespace

int launch_w4_gemm(const W4GemmArgs& a, hipStream_t st) {
  const int nkb = (a.K + W4_K - 1) / W4_K;
  const W4Plan pl = w4_plan(a.M, (a.N + W4_ROWS - 1) / W4_ROWS, nkb);
  if (pl.r == 1) {
    switch (pl.mg) {
      case 1: launch_tile<1, 1>(a, nkb, pl.kw, pl.bpc, st); break;
      case 2: launch_tile<2, 1>(a, nkb, pl.kw, pl.bpc, st); break;
      case 3: launch_tile<3, 1>(a, nkb, pl.kw, pl.bpc, st); break;
      default: launch_tile<4, 1>(a, nkb, pl.kw, pl.bpc, st); break;
    }
  } else {
    switch (pl.mg) {
      case 1: launch_tile<1, 2>(a, nkb, pl.kw, pl.bpc, st); break;
      case 2: launch_tile<2, 2>(a, nkb, pl.kw, pl.bpc, st); break;
      case 3: launch_tile<3, 2>(a, nkb, pl.kw, pl.bpc, st); break;
      default: launch_tile<4, 2>(a, nkb, pl.kw, pl.bpc, st); break;
    }
  }
  MK_HIP_CHECK(hipGetLastError());
  return MK_OK;
}

int launch_w4_quantize(const uint16_t* w, size_t ldw, int N, int K, int group, uint8_t* codes, uint16_t* scales,
                       hipStream_t st) {
  const int nkb = (K + W4_K - 1) / W4_K;
  const long blocks = (long)((N + W4_ROWS - 1) / W4_ROWS) * nkb;
  const dim3 grid((unsigned)((blocks + 3) / 4)), block(256);
  switch (group) {
    case 32: hipLaunchKernelGGL((w4_quantize_kernel<32>), grid, block, 0, st, w, ldw, N, K, nkb, blocks, codes, scales); break;
    case 64: hipLaunchKernelGGL((w4_quantize_kernel<64>), grid, block, 0, st, w, ldw, N, K, nkb, blocks, codes, scales); break;
    default: hipLaunchKernelGGL((w4_quantize_kernel<128>), grid, block, 0, st, w, ldw, N, K, nkb, blocks, codes, scales); break;
  }
  MK_HIP_CHECK(hipGetLastError());
  return MK_OK;
}

int launch_w4_dequantize(const uint8_t* codes, const uint16_t* scales, int N, int K, int group, void* out, bool f32,
                         size_t ldo, hipStream_t st) {
  const int nkb = (K + W4_K - 1) / W4_K;
  const long blocks = (long)((N + W4_ROWS - 1) / W4_ROWS) * nkb;
  const dim3 grid((unsigned)((blocks + 3) / 4)), block(256);
#define MK_DEQ(G)                                                                                                     \
  if (f32) hipLaunchKernelGGL((w4_dequantize_kernel<G, true>), grid, block, 0, st, codes, scales, N, K, nkb, blocks,  \
                              out, ldo);                                                                              \
  else hipLaunchKernelGGL((w4_dequantize_kernel<G, false>), grid, block, 0, st, codes, scales, N, K, nkb, blocks,     \
                          out, ldo);
  switch (group) {
    case 32: MK_DEQ(32) break;
    case 64: MK_DEQ(64) break;
    default: MK_DEQ(128) break;
  }
#undef MK_DEQ
  MK_HIP_CHECK(hipGetLastError());
  return MK_OK;
}

}  // namespace mk
