// mxf4_mma.cuh -- the inner step shared by the skinny 16-bit x MX-FP4 product and the experts' layer.
//
// One warp multiplies 16 weight rows by a few activation rows with mma.sync.m16n8k16 (fp16 operands, fp32 sums).  The
// weights stay as they lie in memory: lane (g, t) = (lane / 4, lane % 4) loads the 16 bytes of block t of a 128-element
// chunk of row g (and of row g + 8), i.e. a whole block of 32 elements with one scale, and turns them into fp16 pairs with
// the hardware conversion of E2M1, which is exact.  An mma adds over the four lanes of a quad, whose blocks have different
// scales, so the eight columns of the other operand are used to keep the blocks apart: column 4 * token + b holds the
// token's activations in the k positions of lane b and zeros elsewhere.  After the eight mmas of a chunk the accumulator of
// (row, 4 * token + b) is the unscaled sum of block b, which is multiplied by the weight block's and the activation block's
// scale and added to the running fp32 sum: 4 multiply-adds for 64 weights per lane.  A group of columns thus serves two
// tokens.  Measured: the conversion with the mma behind it runs at 22 T elements/s on the whole chip, against 12 T that HBM
// delivers (17/32 byte per element at 6.4 TB/s); placing the bits of bf16 with integer instructions reached 12 T.
//
// fp16 activations are used as they are.  bf16 activations are brought into fp16's range with one power of two per block of
// 32 that puts the block's largest magnitude into [2^14, 2^15): a bf16 value has 8 significant bits, so every value down to
// 2^-31 of the block's largest stays exact, smaller ones are rounded to a multiple of 2^-38 of it -- far under the rounding
// of the fp32 sums.
#pragma once

#include <cstdint>

#include "loads.cuh"
#include "numerics.cuh"

namespace sklb {
namespace mxmma {

constexpr int STEP = 256;  // elements of k that a warp takes at a time: two chunks, 128 bytes of each of its 16 rows

// 8 E2M1 codes of a word as 4 fp16 pairs
__device__ __forceinline__ void e2m1_to_f16(uint32_t w, uint32_t (&r)[4]) {
  asm("{.reg .b8 a, b, c, d;\n\tmov.b32 {a, b, c, d}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, a;\n\tcvt.rn.f16x2.e2m1x2 %1, b;\n\tcvt.rn.f16x2.e2m1x2 %2, c;\n\tcvt.rn.f16x2.e2m1x2 %3, d;}"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
      : "r"(w));
}
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Two E8M0 scale bytes as fp32 (0 is the subnormal 2^-127, 255 NaN): the hardware widens them to bf16 exactly.
__device__ __forceinline__ void e8m0x2(uint32_t two, float &lo, float &hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.ue8m0x2 %0, %1;" : "=r"(r) : "h"((uint16_t)two));
  lo = u2f(r << 16);
  hi = u2f(r & 0xFFFF0000u);
}

// A warp's ring of steps in shared memory, filled with cp.async so that loads in flight cost no registers: a slot holds the
// 16-byte pieces of its 16 rows in the order of the lanes (lane l's pieces [row half][chunk] at (2 half + chunk) * 512 +
// 16 l, written and read by the same lane without bank conflicts) and the 16 rows' 8 scale bytes of the step.  The experts'
// layer uses the same rings for 16-bit weights, without scales.
constexpr int CODE_BYTES = 4 * 512, SLOT_BYTES = CODE_BYTES + 128;

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async8(uint32_t dst, const void *src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// How a lane addresses the 16 rows of a tile: rows g and g + 8 for the codes, row lane / 2 for the scales.  A row that does
// not exist has null pointers; its codes count as zeros.
struct TileRows {
  const uint8_t *code[2];
  const uint8_t *scale;
};

__device__ __forceinline__ void st_zero16(uint32_t at) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0u) : "memory");
}

// Bytes [128 step, 128 step + 128) of a tile's 16 rows into a slot, and with SCALES the 8 scale bytes of each row.
// `row_bytes`: length of a row (MX-FP4: 16 bytes to a block); what lies behind it, and rows that do not exist, are zeros with
// scale 1.  VEC: rows start on 16 bytes and are whole units of 16; SVEC: scale rows start on 8 bytes.  Without them single
// bytes are loaded, which are in place when the call returns.
template <bool SCALES, bool VEC, bool SVEC>
__device__ __forceinline__ void fill_slot(uint32_t slot, const TileRows &rows, uint32_t step, uint32_t row_bytes, int lane) {
  const int t = lane & 3;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t b = step * 128u + 64u * c + 16u * t, dst = slot + (2 * h + c) * 512 + lane * 16;
      if (rows.code[h] && b < row_bytes) {
        const uint8_t *p = rows.code[h] + b;
        if (VEC) {
          cp_async16(dst, p);
        } else {
          uint32_t q[4] = {0u, 0u, 0u, 0u};
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (b + i < row_bytes) q[i >> 2] |= ld_u8(p + i) << (8 * (i & 3));
          asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]) : "memory");
        }
      } else {
        st_zero16(dst);
      }
    }
  }
  if (SCALES && (lane & 1) == 0) {
    const uint32_t dst = slot + 4 * 512 + lane * 4, b0 = step * 8u, kblocks = row_bytes / 16u;
    if (SVEC && rows.scale && b0 + 8u <= kblocks) {
      cp_async8(dst, rows.scale + b0);
    } else {
      uint32_t q[2] = {0x7F7F7F7Fu, 0x7F7F7F7Fu};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (rows.scale && b0 + i < kblocks) q[i >> 2] = (q[i >> 2] & ~(0xFFu << (8 * (i & 3)))) | ld_u8(rows.scale + b0 + i) << (8 * (i & 3));
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(dst), "r"(q[0]), "r"(q[1]) : "memory");
    }
  }
}

// Activations in shared memory, for TG groups of two tokens: fp16 elements [token][elements] and one fp32 factor per block
// [token][elements / 32].  `x` / `f`: shared addresses of token 0's element / block 0 of the step; the pitches are in bytes.
// `last`: the last token there is; columns of further ones repeat it (columns do not mix) and are ignored by the caller.
// y[group][row half]: the running sums of this lane's token (2 * group + t / 2), over blocks 2 (t % 2) and 2 (t % 2) + 1
// of every chunk: the lanes t and t ^ 1 hold the two halves of a sum.
template <int TG, bool FACTORS>
__device__ __forceinline__ void multiply_step(uint32_t slot, uint32_t x, uint32_t x_pitch, uint32_t f, uint32_t f_pitch,
                                              uint32_t last, uint32_t zeros, int lane, float (&y)[TG][2]) {
  const int g = lane >> 2, t = lane & 3;
  const bool mine = (g & 3) == t;
  uint32_t xrow[TG], frow[TG];
#pragma unroll
  for (int q = 0; q < TG; ++q) {
    xrow[q] = mine ? x + min(2u * q + (uint32_t)(g >> 2), last) * x_pitch + t * 64u : zeros;
    frow[q] = f + min(2u * q + (uint32_t)(t >> 1), last) * f_pitch + (uint32_t)(t & 1) * 8u;
  }
  uint32_t sc[2][2];  // [row half][chunk]: the scale bytes of the chunk's four blocks
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(sc[h][0]), "=r"(sc[h][1]) : "r"(slot + 4 * 512 + (g + 8 * h) * 8));
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float acc[TG][4];
#pragma unroll
    for (int q = 0; q < TG; ++q) acc[q][0] = acc[q][1] = acc[q][2] = acc[q][3] = 0.0f;
    uint32_t lo[4], hi[4];
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(lo[0]), "=r"(lo[1]), "=r"(lo[2]), "=r"(lo[3])
                 : "r"(slot + c * 512 + lane * 16));
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(hi[0]), "=r"(hi[1]), "=r"(hi[2]), "=r"(hi[3])
                 : "r"(slot + (2 + c) * 512 + lane * 16));
    const uint32_t skip = mine ? c * 256u : 0u;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a[4], b[4];
      e2m1_to_f16(lo[j], a);
      e2m1_to_f16(hi[j], b);
#pragma unroll
      for (int q = 0; q < TG; ++q) {
        uint32_t v[4];
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                     : "r"(xrow[q] + skip + 16u * j));
        mma_f16(acc[q], a[0], b[0], a[1], b[1], v[0], v[1]);
        mma_f16(acc[q], a[2], b[2], a[3], b[3], v[2], v[3]);
      }
    }
    float s[2][2];  // [row half][block of this lane's pair]
#pragma unroll
    for (int h = 0; h < 2; ++h) e8m0x2(sc[h][c] >> (16 * (t & 1)), s[h][0], s[h][1]);
#pragma unroll
    for (int q = 0; q < TG; ++q) {
      float f0 = 1.0f, f1 = 1.0f;
      if (FACTORS)
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                     : "=f"(f0), "=f"(f1)
                     : "r"(frow[q] + c * 16u));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float p0 = FACTORS ? acc[q][2 * h] * f0 : acc[q][2 * h], p1 = FACTORS ? acc[q][2 * h + 1] * f1 : acc[q][2 * h + 1];
        y[q][h] = __fmaf_rn(p0, s[h][0], y[q][h]);
        y[q][h] = __fmaf_rn(p1, s[h][1], y[q][h]);
      }
    }
  }
}

// The power of two that brings a block into fp16's range, from the magnitude bits of its largest value (fp32 pattern):
// the largest ends in [2^14, 2^15).  Returns the factor for the elements; `back` undoes it.
__device__ __forceinline__ float block_factor(uint32_t top, float &back) {
  const int ef = (int)(top >> 23);
  int e = 141 - ef;  // 14 - (ef - 127)
  e = e > 126 ? 126 : e;
  back = u2f((uint32_t)(127 - e) << 23);
  return u2f((uint32_t)(127 + e) << 23);
}

}  // namespace mxmma
}  // namespace sklb
