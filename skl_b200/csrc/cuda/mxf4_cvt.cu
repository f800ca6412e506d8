// mxf4_cvt.cu -- quantisation of matrices to OCP MX-FP4 and the way back.
//
// MX-FP4 (OCP Microscaling Formats v1.0): 32 consecutive elements of a row share one E8M0 scale byte s, an element is an
// E2M1 code c (two per byte, low nibble first) and stands for value(c) * 2^(s - 127); s = 255 is NaN.  For a block with
// largest magnitude A the scale exponent is floor(log2 A) - 2 (2 = the exponent of E2M1's largest value), not below -127:
// with fp32 bits of A that is s = max(exponent field - 2, 0), no logarithm.  x * 2^(127 - s) is exact, so the only rounding
// is the conversion to E2M1 (nearest even, magnitudes above 6 become 6), which is one hardware instruction for two values.
// A block that holds an infinity or a NaN (exponent field 255 of A, taken as an integer maximum of the magnitude bits) gets
// s = 255 and zero codes.  Elements behind the end of a row count as zeros.
//
// All kernels are bound by HBM: 17/32 byte per element on the packed side plus the element itself on the other.
#include "loads.cuh"
#include "numerics.cuh"

namespace sklb {
namespace {

constexpr int THREADS = 256;

template <int DT>
__device__ __forceinline__ float widen(uint32_t bits) {
  return DT == SKL_DT_F32 ? u2f(bits) : DT == SKL_DT_BF16 ? dec_bf16(bits) : dec_f16(bits);
}
template <int DT>
__device__ __forceinline__ float load_one(const void *p, int64_t i) {
  return DT == SKL_DT_F32 ? u2f(ld_u32((const float *)p + i)) : widen<DT>(ld_u16((const uint16_t *)p + i));
}
__device__ __forceinline__ uint32_t mag_bits(float x) { return f2u(x) & 0x7FFFFFFFu; }

// scale byte of a block whose largest magnitude has the fp32 bits `top`, and the factor its elements are multiplied by
__device__ __forceinline__ uint32_t scale_byte(uint32_t top, float &factor) {
  const uint32_t ef = top >> 23;
  const uint32_t s = ef == 255u ? 255u : (ef > 2u ? ef - 2u : 0u);
  factor = ef == 255u ? 0.0f : u2f((254u - s) << 23);  // 2^(127 - s); s <= 252 for a finite block
  return s;
}
// code byte of two elements (lo in the low nibble); a NaN block passes factor 0, whose products need not be zero
__device__ __forceinline__ uint32_t codes2(float lo, float hi, float factor) {
  uint16_t r;
  asm("{.reg .b8 t; cvt.rn.satfinite.e2m1x2.f32 t, %1, %2; cvt.u16.u8 %0, t;}" : "=h"(r) : "f"(hi * factor), "f"(lo * factor));
  return r;
}

// 8 consecutive elements of a row as raw words (4 for a 16-bit type, 8 for fp32)
template <int DT>
struct Eight {
  static constexpr int W = DT == SKL_DT_F32 ? 8 : 4;
  uint32_t w[W];
  __device__ __forceinline__ float get(int e) const {
    if (DT == SKL_DT_F32) return u2f(w[e % W]);
    return widen<DT>((e & 1) ? w[e / 2] >> 16 : w[e / 2] & 0xFFFFu);
  }
};
template <int DT>
__device__ __forceinline__ void load_eight(Eight<DT> &v, const void *base, int64_t first) {
  const uint4 *p = reinterpret_cast<const uint4 *>((const uint8_t *)base + first * (DT == SKL_DT_F32 ? 4 : 2));
  const uint4 a = ld_v4(p);
  v.w[0] = a.x, v.w[1] = a.y, v.w[2] = a.z, v.w[3] = a.w;
  if (DT == SKL_DT_F32) {
    const uint4 b = ld_v4(p + 1);
    v.w[4 % Eight<DT>::W] = b.x, v.w[5 % Eight<DT>::W] = b.y, v.w[6 % Eight<DT>::W] = b.z, v.w[7 % Eight<DT>::W] = b.w;
  }
}
template <int DT>
__device__ __forceinline__ void load_eight_tail(Eight<DT> &v, const void *base, int64_t first, int count) {
#pragma unroll
  for (int i = 0; i < Eight<DT>::W; ++i) v.w[i] = 0u;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (e < count) {
      if (DT == SKL_DT_F32) v.w[e % Eight<DT>::W] = ld_u32((const uint32_t *)base + first + e);
      else v.w[(e / 2) % Eight<DT>::W] |= ld_u16((const uint16_t *)base + first + e) << (16 * (e & 1));
    }
  }
}

// Which rows and groups of 8 elements a thread takes: a warp takes 32 * UNROLL consecutive groups of the matrix (rows one
// after the other, 4 groups to a block), its lanes 32 consecutive ones at a time.  Where they lie in one row (`whole`, the same
// for the warp) everything follows from the first with constants; the general case divides for every group, which is half
// of the instructions of these kernels.
template <int UNROLL>
struct Groups {
  uint64_t row0;   // row and group of the warp's first group
  uint32_t rem0;
  bool whole;
  __device__ __forceinline__ Groups(uint32_t m, uint32_t per_row) {
    const uint64_t first = (uint64_t)blockIdx.x * (THREADS * UNROLL) + (threadIdx.x >> 5) * (32u * UNROLL);
    if (first >> 32) {
      row0 = first / per_row;
      rem0 = (uint32_t)(first - row0 * per_row);
    } else {
      row0 = (uint32_t)first / per_row;
      rem0 = (uint32_t)first - (uint32_t)row0 * per_row;
    }
    whole = row0 < m && rem0 + 32u * UNROLL <= per_row;
  }
  // row (m: behind the end) and group of this lane's u-th group
  __device__ __forceinline__ void at(int u, uint32_t m, uint32_t per_row, uint32_t &row, uint32_t &g) const {
    const uint32_t r = rem0 + u * 32 + (threadIdx.x & 31);
    if (whole) {
      row = (uint32_t)row0;
      g = r;
    } else {
      const uint64_t wide = row0 + r / per_row;
      row = wide < m ? (uint32_t)wide : m;
      g = r % per_row;
    }
  }
  // the block whose scale this lane loads or stores, one byte for all groups of the warp: block lane % UNROLL * 8 + lane / 4 of the
  // warp's 8 * UNROLL (UNROLL = 4) or block lane / 4 (UNROLL = 1, the first lane of each quad)
  __device__ __forceinline__ bool own_block(uint32_t m, uint32_t per_row, uint32_t &r, uint32_t &blk) const {
    const uint32_t lane = threadIdx.x & 31, i = rem0 + (UNROLL == 1 ? lane & ~3u : (lane % UNROLL) * 32u + (lane & ~3u));
    if (whole) {
      r = (uint32_t)row0;
      blk = i >> 2;
      return UNROLL > 1 || (lane & 3u) == 0u;
    }
    const uint64_t wide = row0 + i / per_row;
    r = wide < m ? (uint32_t)wide : m;
    blk = i % per_row >> 2;
    return wide < m && (UNROLL > 1 || (lane & 3u) == 0u);
  }
};

// 8 elements of a block (four lanes together hold it): the block's scale byte and the lane's codes
template <int DT>
__device__ __forceinline__ uint32_t encode_eight(const Eight<DT> &v, uint32_t &s) {
  uint32_t top = 0;
  if (DT == SKL_DT_F32) {
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, mag_bits(v.get(e)));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
  } else {
    // magnitudes of 16-bit floats order like their bits, two at a time
    uint32_t pair = 0;
#pragma unroll
    for (int i = 0; i < Eight<DT>::W; ++i) pair = __vmaxu2(pair, v.w[i] & 0x7FFF7FFFu);
    pair = __vmaxu2(pair, __shfl_xor_sync(0xFFFFFFFFu, pair, 1));
    pair = __vmaxu2(pair, __shfl_xor_sync(0xFFFFFFFFu, pair, 2));
    top = f2u(widen<DT>(max(pair & 0xFFFFu, pair >> 16)));
  }
  float factor;
  s = scale_byte(top, factor);
  uint32_t w;
  if (DT == SKL_DT_BF16) {  // the exact product by a power of two, two elements at a time (what underflows becomes a zero code)
    const uint32_t f = (f2u(factor) >> 16) * 0x00010001u;
    uint32_t p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(p[i]) : "r"(v.w[i % Eight<DT>::W]), "r"(f));
    w = codes2(u2f(p[0] << 16), u2f(p[0] & 0xFFFF0000u), 1.0f) | codes2(u2f(p[1] << 16), u2f(p[1] & 0xFFFF0000u), 1.0f) << 8 |
        codes2(u2f(p[2] << 16), u2f(p[2] & 0xFFFF0000u), 1.0f) << 16 | codes2(u2f(p[3] << 16), u2f(p[3] & 0xFFFF0000u), 1.0f) << 24;
  } else {
    w = codes2(v.get(0), v.get(1), factor) | codes2(v.get(2), v.get(3), factor) << 8 | codes2(v.get(4), v.get(5), factor) << 16 |
        codes2(v.get(6), v.get(7), factor) << 24;
  }
  return s == 255u ? 0u : w;
}

// Rows with unit stride, 16-byte aligned.  Four lanes share a block: a lane takes 8 elements (one or two 16-byte loads), the
// block's largest magnitude is two shuffles, the lane's 8 codes are one 4-byte store; loads and stores of a warp are
// contiguous.  UNROLL groups per thread keep that many loads in flight, and the warp's 32 scale bytes leave in one store.
// bf16 16384 x 4096: 28.9 us, 5.9 TB/s, 0.91 of a copy's rate (66 % of the issue slots are busy); fp32 14336 x 4096: 39.6 us.
template <int DT, int UNROLL>
__global__ void __launch_bounds__(THREADS)
    quant_rows_kernel(uint8_t *__restrict__ dst, int64_t rsd, uint8_t *__restrict__ scales, int64_t rss,
                      const void *__restrict__ src, int64_t rs, uint32_t m, uint32_t k, uint32_t kblocks) {
  static_assert(UNROLL == 1 || UNROLL == 4, "a lane stores one scale byte");
  dep_wait();
  const uint32_t per_row = kblocks * 4u;
  const Groups<UNROLL> at(m, per_row);
  Eight<DT> v[UNROLL];
  uint32_t byte = 0, s;
  if (at.whole && (at.rem0 + 32u * UNROLL) * 8u <= k) {
    const uint32_t g = at.rem0 + (threadIdx.x & 31);
    const int64_t from = (int64_t)at.row0 * rs + (int64_t)g * 8;
    uint8_t *to = dst + (int64_t)at.row0 * rsd + (int64_t)g * 4;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) load_eight<DT>(v[u], src, from + 256 * u);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      *reinterpret_cast<uint32_t *>(to + 128 * u) = encode_eight<DT>(v[u], s);
      if (UNROLL == 1 || (int)(threadIdx.x & 3) == u) byte = s;
    }
  } else {
    uint32_t row[UNROLL], g[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      at.at(u, m, per_row, row[u], g[u]);
      const int64_t from = (int64_t)row[u] * rs + (int64_t)g[u] * 8;
      const int left = row[u] < m ? (int)k - (int)(g[u] * 8) : 0;
      if (left >= 8) load_eight<DT>(v[u], src, from);
      else load_eight_tail<DT>(v[u], src, from, left);
    }
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      const uint32_t w = encode_eight<DT>(v[u], s);
      if (row[u] < m) *reinterpret_cast<uint32_t *>(dst + (int64_t)row[u] * rsd + (int64_t)g[u] * 4) = w;
      if (UNROLL == 1 || (int)(threadIdx.x & 3) == u) byte = s;
    }
  }
  uint32_t r, blk;
  if (at.own_block(m, per_row, r, blk)) scales[(int64_t)r * rss + blk] = (uint8_t)byte;
}

// Any two strides, any alignment: one warp per block of 32, one element per lane (consecutive lanes read consecutive
// elements of the row), codes stored byte by byte from the even lanes.
template <int DT>
__global__ void __launch_bounds__(THREADS)
    quant_any_kernel(uint8_t *__restrict__ dst, int64_t rsd, uint8_t *__restrict__ scales, int64_t rss,
                     const void *__restrict__ src, int64_t rs, int64_t cs, uint32_t m, uint32_t k, uint32_t kblocks) {
  dep_wait();
  const uint64_t total = (uint64_t)m * kblocks, stride = (uint64_t)gridDim.x * (THREADS / 32);
  const int lane = threadIdx.x & 31;
  for (uint64_t i = (uint64_t)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5); i < total; i += stride) {
    const uint32_t row = (uint32_t)(i / kblocks), kb = (uint32_t)(i - (uint64_t)row * kblocks);
    const uint32_t kk = kb * 32u + lane;
    const float x = kk < k ? load_one<DT>(src, (int64_t)row * rs + (int64_t)kk * cs) : 0.0f;
    float factor;
    const uint32_t s = scale_byte(__reduce_max_sync(0xFFFFFFFFu, mag_bits(x)), factor);
    const float next = __shfl_down_sync(0xFFFFFFFFu, x, 1);
    const uint32_t c = s == 255u ? 0u : codes2(x, next, factor);
    if ((lane & 1) == 0) dst[(int64_t)row * rsd + (int64_t)kb * 16 + (lane >> 1)] = (uint8_t)c;
    if (lane == 0) scales[(int64_t)row * rss + kb] = (uint8_t)s;
  }
}

// Unit stride along the rows' index (a column of a row-major source becomes a packed row).  A lane owns RPL neighbouring
// packed rows and a whole block of each, so the maximum is its own; the warp reads runs of 32 * RPL elements, the CTA's
// eight warps take eight blocks of k, and the codes go through shared memory so that each packed row is written as a run of
// 128 bytes.  RPL is chosen for 8-byte loads; 1 serves any alignment.  fp32 14336 x 4096: 49.2 us, 5.4 TB/s, 0.84 of a copy's rate;
// bf16 16384 x 4096: 36.8 us, 0.71, where the instructions per element (half the issue slots) weigh more against fewer bytes.
template <int DT, int RPL>
__global__ void __launch_bounds__(THREADS)
    quant_columns_kernel(uint8_t *__restrict__ dst, int64_t rsd, uint8_t *__restrict__ scales, int64_t rss,
                         const void *__restrict__ src, int64_t cs, uint32_t m, uint32_t k, uint32_t kblocks,
                         uint32_t row_tiles, int vec_store) {
  constexpr int ROWS = 32 * RPL, PITCH = 128 + 16;
  __shared__ __align__(16) uint8_t codes[ROWS * PITCH];
  __shared__ uint8_t sc[ROWS][8];
  dep_wait();
  const uint32_t tile_r = blockIdx.x % row_tiles, tile_k = blockIdx.x / row_tiles;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t row = tile_r * ROWS + lane * RPL, kb = tile_k * 8u + warp;
  if (kb < kblocks) {
    constexpr int WORDS = RPL == 1 ? 1 : 2;  // 32-bit words per load
    uint32_t raw[32][WORDS];
#pragma unroll
    for (int e = 0; e < 32; ++e) {
      const uint32_t kk = kb * 32u + e;
      const int64_t at = (int64_t)kk * cs + row;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) raw[e][i] = 0u;
      if (kk < k) {
        if (RPL == 1) {
          if (row < m) raw[e][0] = DT == SKL_DT_F32 ? ld_u32((const uint32_t *)src + at) : ld_u16((const uint16_t *)src + at);
        } else if (row + RPL <= m) {
          const uint2 t = ld_v2((const uint8_t *)src + at * (DT == SKL_DT_F32 ? 4 : 2));
          raw[e][0] = t.x;
          raw[e][WORDS - 1] = t.y;
        } else {
#pragma unroll
          for (int i = 0; i < RPL; ++i) {
            if (row + i < m) {
              if (DT == SKL_DT_F32) raw[e][i % WORDS] = ld_u32((const uint32_t *)src + at + i);
              else raw[e][(i / 2) % WORDS] |= ld_u16((const uint16_t *)src + at + i) << (16 * (i & 1));
            }
          }
        }
      }
    }
    // 16-bit types, RPL = 4: a word holds two rows' elements, whose maxima and products (bf16) are taken two at a time
    constexpr bool PAIRED = DT != SKL_DT_F32 && RPL > 1;
    uint32_t pair_top[WORDS];
    if (PAIRED) {
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        pair_top[j] = 0;
#pragma unroll
        for (int e = 0; e < 32; ++e) pair_top[j] = __vmaxu2(pair_top[j], raw[e][j] & 0x7FFF7FFFu);
      }
    }
    uint32_t s_of[RPL];
    float factor_of[RPL];
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
      uint32_t top = 0;
      if (PAIRED) {
        const uint32_t bits = pair_top[(i / 2) % WORDS];
        top = f2u(widen<DT>((i & 1) ? bits >> 16 : bits & 0xFFFFu));
      } else {
#pragma unroll
        for (int e = 0; e < 32; ++e) top = max(top, mag_bits(DT == SKL_DT_F32 ? u2f(raw[e][i % WORDS]) : widen<DT>(raw[e][0] & 0xFFFFu)));
      }
      s_of[i] = scale_byte(top, factor_of[i]);
    }
    if (PAIRED && DT == SKL_DT_BF16) {  // exact products by powers of two (what underflows becomes a zero code)
#pragma unroll
      for (int j = 0; j < WORDS; ++j) {
        const uint32_t f = f2u(factor_of[(2 * j) % RPL]) >> 16 | (f2u(factor_of[(2 * j + 1) % RPL]) & 0xFFFF0000u);
#pragma unroll
        for (int e = 0; e < 32; ++e) asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(raw[e][j]) : "r"(raw[e][j]), "r"(f));
      }
    }
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
      auto val = [&](int e) {
        if (DT == SKL_DT_F32) return u2f(raw[e][i % WORDS]);
        const uint32_t w = raw[e][(i / 2) % WORDS];
        if (DT == SKL_DT_BF16) return u2f((i & 1) ? w & 0xFFFF0000u : w << 16);
        return widen<DT>((i & 1) ? w >> 16 : w & 0xFFFFu);
      };
      const uint32_t s = s_of[i];
      const float factor = PAIRED && DT == SKL_DT_BF16 ? 1.0f : factor_of[i];
      uint32_t w[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        w[q] = codes2(val(8 * q), val(8 * q + 1), factor) | codes2(val(8 * q + 2), val(8 * q + 3), factor) << 8 |
               codes2(val(8 * q + 4), val(8 * q + 5), factor) << 16 | codes2(val(8 * q + 6), val(8 * q + 7), factor) << 24;
        if (s == 255u) w[q] = 0u;
      }
      const int r = lane * RPL + i;
      *reinterpret_cast<uint4 *>(codes + r * PITCH + warp * 16) = make_uint4(w[0], w[1], w[2], w[3]);
      sc[r][warp] = (uint8_t)s;
    }
  }
  __syncthreads();
  const uint32_t kb0 = tile_k * 8u, kbs = min(8u, kblocks - kb0);
  for (uint32_t j = threadIdx.x; j < ROWS * 8u; j += THREADS) {
    const uint32_t r = j >> 3, b = j & 7u, out = tile_r * ROWS + r;
    if (out < m && b < kbs) {
      uint8_t *p = dst + (int64_t)out * rsd + (int64_t)(kb0 + b) * 16;
      const uint8_t *q = codes + r * PITCH + b * 16;
      if (vec_store) {
        *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(q);
      } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) p[e] = q[e];
      }
      scales[(int64_t)out * rss + kb0 + b] = sc[r][b];
    }
  }
}

// ---------------------------------------------------------------------------------------------------- read back
__device__ __forceinline__ float scale_value(uint32_t s) {
  return u2f(s == 255u ? 0x7FC00000u : (s == 0u ? 0x00400000u : s << 23));  // 2^(s - 127); 2^-127 is subnormal
}
template <int DT>
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  return DT == SKL_DT_BF16 ? pack_bf16x2_no_nan(lo, hi) : pack_f16x2_no_nan(lo, hi);
}
template <int DT>
__device__ __forceinline__ void store_one(void *dst, int64_t at, float v) {
  if (DT == SKL_DT_F32) ((float *)dst)[at] = v;
  else ((uint16_t *)dst)[at] = (uint16_t)(narrow2<DT>(v, 0.0f) & 0xFFFFu);
}

// 8 elements from their codes
template <int DT>
__device__ __forceinline__ void decode_eight(uint32_t w, uint32_t s, float (&x)[8]) {
  const float f = scale_value(s);
  uint32_t h[4];
  asm("{.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    x[2 * q] = __fmul_rn(dec_f16(h[q] & 0xFFFFu), f);
    x[2 * q + 1] = __fmul_rn(dec_f16(h[q] >> 16), f);
  }
}
template <int DT>
__device__ __forceinline__ void store_eight(void *dst, int64_t at, const float (&x)[8]) {
  if (DT == SKL_DT_F32) {
    float4 *o = reinterpret_cast<float4 *>((float *)dst + at);
    o[0] = make_float4(x[0], x[1], x[2], x[3]);
    o[1] = make_float4(x[4], x[5], x[6], x[7]);
  } else {
    *reinterpret_cast<uint4 *>((uint16_t *)dst + at) =
        make_uint4(narrow2<DT>(x[0], x[1]), narrow2<DT>(x[2], x[3]), narrow2<DT>(x[4], x[5]), narrow2<DT>(x[6], x[7]));
  }
}

// A thread widens 8 elements: one 4-byte load, one (16-bit types) or two 16-byte stores; the loads and stores of a warp are
// contiguous, its 32 scale bytes come in one load.  vec: 4-byte aligned packed rows and 16-byte aligned output rows; without
// it, and in the ragged end of a row, single bytes and elements.  16384 x 4096 to bf16: 27.7 us, 6.1 TB/s, 0.95 of a copy's
// rate; 14336 x 4096 to fp32: 47.8 us.
template <int DT, int UNROLL>
__global__ void __launch_bounds__(THREADS)
    widen_rows_kernel(void *__restrict__ dst, int64_t rsd, const uint8_t *__restrict__ src, int64_t rsa,
                      const uint8_t *__restrict__ scales, int64_t rss, uint32_t m, uint32_t k, int vec) {
  static_assert(UNROLL == 1 || UNROLL == 4, "a lane loads one scale byte");
  dep_wait();
  const uint32_t per_row = (k + 31u) / 32u * 4u;
  const Groups<UNROLL> at(m, per_row);
  uint32_t w[UNROLL], r, blk;
  const uint32_t byte = at.own_block(m, per_row, r, blk) ? ld_u8(scales + (int64_t)r * rss + blk) : 0u;
  float x[8];
  if (vec && at.whole && (at.rem0 + 32u * UNROLL) * 8u <= k) {
    const uint32_t g = at.rem0 + (threadIdx.x & 31);
    const uint8_t *from = src + (int64_t)at.row0 * rsa + (int64_t)g * 4;
    const int64_t to = (int64_t)at.row0 * rsd + (int64_t)g * 8;
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) w[u] = ld_u32(from + 128 * u);
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) {
      decode_eight<DT>(w[u], __shfl_sync(0xFFFFFFFFu, byte, (threadIdx.x & 28) + (UNROLL == 1 ? 0 : u)), x);
      store_eight<DT>(dst, to + 256 * u, x);
    }
    return;
  }
  uint32_t row[UNROLL], g[UNROLL], s[UNROLL];
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    at.at(u, m, per_row, row[u], g[u]);
    w[u] = 0u;
    if (row[u] < m) {
      const uint8_t *p = src + (int64_t)row[u] * rsa + (int64_t)g[u] * 4;
      if (vec) w[u] = ld_u32(p);
      else w[u] = ld_u8(p) | ld_u8(p + 1) << 8 | ld_u8(p + 2) << 16 | ld_u8(p + 3) << 24;
    }
  }
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) s[u] = __shfl_sync(0xFFFFFFFFu, byte, (threadIdx.x & 28) + (UNROLL == 1 ? 0 : u));
#pragma unroll
  for (int u = 0; u < UNROLL; ++u) {
    if (row[u] >= m || g[u] * 8u >= k) continue;
    decode_eight<DT>(w[u], s[u], x);
    const int64_t to = (int64_t)row[u] * rsd + (int64_t)g[u] * 8;
    const uint32_t left = k - g[u] * 8u;
    if (vec && left >= 8u) {
      store_eight<DT>(dst, to, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if ((uint32_t)e < left) store_one<DT>(dst, to + e, x[e]);
    }
  }
}

// fp16 as the exact sum of two bf16 values: hi keeps 8 of the 11 significant bits, lo the rest (x - hi is exact in fp32, has
// at most 3 significant bits and an exponent that bf16 holds).  An infinity or NaN stays in hi, lo is then zero.
// dst: rows of 2 * ld elements, hi at 0, lo at ld; the columns behind k are zeros.
__global__ void __launch_bounds__(THREADS)
    split_f16_kernel(uint16_t *__restrict__ dst, uint32_t ld, const uint16_t *__restrict__ src, int64_t rs, uint32_t m, uint32_t k) {
  dep_wait();
  const uint64_t total = (uint64_t)m * ld, stride = (uint64_t)gridDim.x * THREADS;
  for (uint64_t i = (uint64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += stride) {
    const uint32_t row = (uint32_t)(i / ld), col = (uint32_t)(i - (uint64_t)row * ld);
    const float x = col < k ? dec_f16(ld_u16(src + (int64_t)row * rs + col)) : 0.0f;
    const uint32_t hi = enc_bf16(x);
    const bool finite = (f2u(x) & 0x7F800000u) != 0x7F800000u;
    dst[(uint64_t)row * 2 * ld + col] = (uint16_t)hi;
    dst[(uint64_t)row * 2 * ld + ld + col] = (uint16_t)(finite ? enc_bf16(x - dec_bf16(hi)) : 0u);
  }
}

// Rows of 16-bit elements at any pitch and 2-byte alignment to rows of `ld` elements (a multiple of 8) on 16-byte boundaries, zeros
// behind column k: what the TMA of the tensor-core kernel asks of an operand.  A thread writes 8 elements at once; its 2-byte
// loads meet the lines that its neighbours bring to the L1.
__global__ void __launch_bounds__(THREADS)
    align_rows_kernel(uint16_t *__restrict__ dst, uint32_t ld, const uint16_t *__restrict__ src, int64_t rs, uint32_t m, uint32_t k) {
  dep_wait();
  const uint32_t per_row = ld / 8u;
  const uint64_t total = (uint64_t)m * per_row, stride = (uint64_t)gridDim.x * THREADS;
  for (uint64_t i = (uint64_t)blockIdx.x * THREADS + threadIdx.x; i < total; i += stride) {
    const uint32_t row = (uint32_t)(i / per_row), col = (uint32_t)(i - (uint64_t)row * per_row) * 8u;
    const uint16_t *from = src + (int64_t)row * rs + col;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (col + e < k) w[e >> 1] |= ld_u16(from + e) << (16 * (e & 1));
    *reinterpret_cast<uint4 *>(dst + (uint64_t)row * ld + col) = make_uint4(w[0], w[1], w[2], w[3]);
  }
}

// Launches as a programmatic dependent: the kernel's set-up overlaps the end of the one before it on the stream; every
// kernel here waits (griddepcontrol.wait) before it touches memory.
template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), uint64_t grid, cudaStream_t s, A... args) {
  if (grid == 0 || grid > 0x7FFFFFFFull) return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(THREADS);
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SKLB_COUNT_LAUNCH();
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

inline bool aligned(const void *p, size_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

constexpr int UNROLL = 4;

template <int DT>
cudaError_t launch_quant(uint8_t *dst, int64_t rsd, uint8_t *scales, int64_t rss, const void *src, int64_t rs, int64_t cs,
                         uint32_t m, uint32_t k, cudaStream_t s) {
  const int es = DT == SKL_DT_F32 ? 4 : 2;
  const uint32_t kblocks = (k + 31) / 32;
  if (cs == 1 && aligned(src, 16) && (m == 1 || rs * es % 16 == 0) && aligned(dst, 4) && (m == 1 || rsd % 4 == 0)) {
    const uint64_t groups = (uint64_t)m * kblocks * 4;
    // Small problems: one group per thread, so that more SMs take part.  Rows of 4096 quantised and read back, one / four groups to
    // a thread: bf16 2^15 groups 2.6 / 2.9 us, 2^17 3.3 / 3.1, 2^18 4.3 / 3.8, 2^20 12.8 / 9.6; fp32 2^15 2.9 / 3.9, 2^17 4.2 / 4.1,
    // 2^18 5.5 / 5.7, 2^20 16.9 / 17.8.
    if (groups < (1u << 18)) return launch(quant_rows_kernel<DT, 1>, ceil_div(groups, THREADS), s, dst, rsd, scales, rss, src, rs, m, k, kblocks);
    return launch(quant_rows_kernel<DT, UNROLL>, ceil_div(groups, THREADS * UNROLL), s, dst, rsd, scales, rss, src, rs, m, k, kblocks);
  }
  if (rs == 1 && m > 1) {
    constexpr int RPL = DT == SKL_DT_F32 ? 2 : 4;
    const int vec_store = aligned(dst, 16) && rsd % 16 == 0;
    const uint64_t kt = ceil_div(kblocks, 8);
    if (aligned(src, 8) && (k == 1 || cs * es % 8 == 0)) {
      const uint32_t rt = (uint32_t)ceil_div(m, 32 * RPL);
      return launch(quant_columns_kernel<DT, RPL>, rt * kt, s, dst, rsd, scales, rss, src, cs, m, k, kblocks, rt, vec_store);
    }
    const uint32_t rt = (uint32_t)ceil_div(m, 32);
    return launch(quant_columns_kernel<DT, 1>, rt * kt, s, dst, rsd, scales, rss, src, cs, m, k, kblocks, rt, vec_store);
  }
  uint64_t grid = ceil_div((uint64_t)m * kblocks, THREADS / 32);
  if (grid > 148 * 64) grid = 148 * 64;
  return launch(quant_any_kernel<DT>, grid, s, dst, rsd, scales, rss, src, rs, cs, m, k, kblocks);
}

template <int DT>
cudaError_t launch_widen(void *dst, int64_t rsd, const uint8_t *src, int64_t rsa, const uint8_t *scales, int64_t rss,
                         uint32_t m, uint32_t k, cudaStream_t s) {
  const int es = DT == SKL_DT_F32 ? 4 : 2;
  const int vec = aligned(src, 4) && aligned(dst, 16) && (m == 1 || (rsa % 4 == 0 && rsd * es % 16 == 0));
  const uint64_t groups = (uint64_t)m * ((k + 31) / 32) * 4;
  if (groups < (1u << 18)) return launch(widen_rows_kernel<DT, 1>, ceil_div(groups, THREADS), s, dst, rsd, src, rsa, scales, rss, m, k, vec);
  return launch(widen_rows_kernel<DT, UNROLL>, ceil_div(groups, THREADS * UNROLL), s, dst, rsd, src, rsa, scales, rss, m, k, vec);
}

}  // namespace
}  // namespace sklb

using namespace sklb;

extern "C" int skl_b200_launch_quant_mxf4(void *dst, int64_t rsd, void *scales, int64_t rss, const void *src, int src_type,
                                          int64_t rs, int64_t cs, uint32_t m, uint32_t k, void *stream) {
  cudaStream_t s = (cudaStream_t)stream;
  uint8_t *d = (uint8_t *)dst, *sc = (uint8_t *)scales;
  switch (src_type) {
    case SKL_DT_F32: return (int)launch_quant<SKL_DT_F32>(d, rsd, sc, rss, src, rs, cs, m, k, s);
    case SKL_DT_BF16: return (int)launch_quant<SKL_DT_BF16>(d, rsd, sc, rss, src, rs, cs, m, k, s);
    case SKL_DT_F16: return (int)launch_quant<SKL_DT_F16>(d, rsd, sc, rss, src, rs, cs, m, k, s);
    default: return (int)cudaErrorInvalidValue;
  }
}

extern "C" int skl_b200_launch_widen_mxf4(void *dst, int dst_type, int64_t rsd, const void *src, int64_t rsa,
                                          const void *scales, int64_t rss, uint32_t m, uint32_t k, void *stream) {
  cudaStream_t s = (cudaStream_t)stream;
  const uint8_t *p = (const uint8_t *)src, *sc = (const uint8_t *)scales;
  switch (dst_type) {
    case SKL_DT_F32: return (int)launch_widen<SKL_DT_F32>(dst, rsd, p, rsa, sc, rss, m, k, s);
    case SKL_DT_BF16: return (int)launch_widen<SKL_DT_BF16>(dst, rsd, p, rsa, sc, rss, m, k, s);
    case SKL_DT_F16: return (int)launch_widen<SKL_DT_F16>(dst, rsd, p, rsa, sc, rss, m, k, s);
    default: return (int)cudaErrorInvalidValue;
  }
}

extern "C" int skl_b200_launch_split_f16(void *dst, uint32_t ld, const void *src, int64_t rs, uint32_t m, uint32_t k,
                                         void *stream) {
  uint64_t grid = ceil_div((uint64_t)m * ld, THREADS * 4);
  if (grid > 148 * 32) grid = 148 * 32;
  return (int)launch(split_f16_kernel, grid, (cudaStream_t)stream, (uint16_t *)dst, ld, (const uint16_t *)src, rs, m, k);
}

extern "C" int skl_b200_launch_align_rows16(void *dst, uint32_t ld, const void *src, int64_t rs, uint32_t m, uint32_t k, void *stream) {
  uint64_t grid = ceil_div((uint64_t)m * (ld / 8u), THREADS);
  if (grid > 148 * 64) grid = 148 * 64;
  return (int)launch(align_rows_kernel, grid, (cudaStream_t)stream, (uint16_t *)dst, ld, (const uint16_t *)src, rs, m, k);
}
