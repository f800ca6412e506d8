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
// tokens; it stays in registers while the warp goes through its tiles (read from shared memory for each, it kept the
// shared-memory pipe busier than the weights did).  Measured: the conversion with the mma behind it runs at 22 T elements/s
// on the whole chip, against 12 T that HBM delivers (17/32 byte per element at 6.4 TB/s); placing the bits of bf16 with
// integer instructions reached 12 T.
//
// Activations are brought into fp16's range with one power of two per block of 32 that puts the block's largest magnitude into
// [2^14, 2^15).  A bf16 value has 8 significant bits, so every value down to 2^-31 of the block's largest stays exact, smaller
// ones are rounded to a multiple of 2^-38 of it -- far under the rounding of the fp32 sums.  fp16 values stay exact, but for
// those under 2^-13 in a block whose largest is 2^15 or more, which is halved: they are rounded to a multiple of 2^-23.
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

__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// `bytes`: how much of the 16 is read, the rest is zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

// How a lane addresses the 16 rows of a tile: rows g and g + 8 for the codes (from byte 16 t on), row lane / 2 for the scales;
// a row that does not exist (has[] false) counts as zeros and its pointer is not followed.
struct TileRows {
  const uint8_t *code[2];
  const uint8_t *scale;
  bool has[2], has_scale;
};

// How rows can be loaded.  WHOLE: rows start on 16 bytes and are whole steps of 128 bytes, scale rows start on 8 bytes: no
// bounds within a row, a dozen instructions for a slot (with the checks of ALIGNED the loads took half the kernel's
// instructions).  ALIGNED: rows start on 16 bytes and are whole units of 16.  BYTES: anything.
enum RowMode { BYTES = 0, ALIGNED = 1, WHOLE = 2 };

// Bytes [128 step, 128 step + 128) of a tile's 16 rows into a slot, and with SCALES the 8 scale bytes of each row.
// `row_bytes`: length of a row (MX-FP4: 16 bytes to a block); what lies behind it counts as zeros (blocks that do not exist
// and rows that do not exist have codes of zero and a scale that is finite).  Single bytes are in place when the call returns.
template <bool SCALES, int MODE>
__device__ __forceinline__ void fill_slot(uint32_t slot, const TileRows &rows, uint32_t step, uint32_t row_bytes, int lane) {
  const uint32_t at = step * 128u, dst = slot + lane * 16;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint8_t *p = rows.code[h] + at;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const uint32_t b = at + 64u * c + 16u * (lane & 3), d = dst + (2 * h + c) * 512;
      if (MODE != BYTES) {
        cp_async16(d, p + 64 * c, rows.has[h] && (MODE == WHOLE || b < row_bytes) ? 16u : 0u);
      } else {
        uint32_t q[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (rows.has[h] && b + i < row_bytes) q[i >> 2] |= ld_u8(p + 64 * c + i) << (8 * (i & 3));
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(d), "r"(q[0]), "r"(q[1]), "r"(q[2]), "r"(q[3]) : "memory");
      }
    }
  }
  if (SCALES) {
    const uint32_t d = slot + CODE_BYTES + lane * 4, b0 = step * 8u, kblocks = row_bytes / 16u;
    if (MODE == WHOLE) {
      asm volatile(
          "{\n\t.reg .pred p;\n\tsetp.eq.u32 p, %3, 0;\n\t"
          "@p cp.async.ca.shared.global [%0], [%1], 8, %2;\n\t}" ::"r"(d), "l"(rows.scale + b0), "r"(rows.has_scale ? 8u : 0u), "r"(lane & 1)
          : "memory");
    } else if ((lane & 1) == 0) {
      uint32_t q[2] = {0u, 0u};
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (rows.has_scale && b0 + i < kblocks) q[i >> 2] |= ld_u8(rows.scale + b0 + i) << (8 * (i & 3));
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(d), "r"(q[0]), "r"(q[1]) : "memory");
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

// One group of two tokens as the mma's second operand, for one step, in registers: lane (g, t) with g % 4 == t holds block t of
// both chunks of token g / 4 as fp16 pairs, every other lane zeros.  factor[chunk][i]: what undoes the block factors of the
// sums this lane ends up with, token t / 2, blocks 2 (t % 2) + i.
//
// A step's sums y are the products' sums divided by `lift`, 1 unless the factors are very large: a block's unscaled sum is below
// 32 * 6 * 2^15 < 2^23, and times a factor above 2^104 (activations from 2^119 on) it may leave fp32's range before the weights'
// scale brings it back.  A lane and its neighbour, which share the token, then take 2^9 off the factors, whose largest is 2^113, and
// `lift` gives it back to the scaled sum.  (Next to such a block the sums of others are exact to 2^-141 times their scale.)
// A branch to another order of the two products instead cost 5 % of the experts' layer.
struct Columns {
  uint32_t v[2][16];
  float factor[2][2], lift;
};
// Chunk c of a group from 8 fp32 elements of every lane: lane L brings elements 8 (L % 4) .. + 7 of block L / 4 % 4 of token
// L / 16 (zeros where there is none).  The four lanes of a quad are the four parts of one block, and the lane that has to hold
// the block is one of them: the block's maximum takes two shuffles, the parts sixteen.
__device__ __forceinline__ void gather_chunk(Columns &x, int c, const float (&e)[8], int lane) {
  const int g = lane >> 2, t = lane & 3;
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = max(top, f2u(e[i]) & 0x7FFFFFFFu);
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
  float back;
  const float factor = block_factor(top, back);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_f16x2_no_nan(e[2 * i] * factor, e[2 * i + 1] * factor);
  const bool mine = (g & 3) == t;
#pragma unroll
  for (int part = 0; part < 4; ++part) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t v = __shfl_sync(0xFFFFFFFFu, w[i], part, 4);
      x.v[c][4 * part + i] = mine ? v : 0u;
    }
  }
  // the factors travel to the lanes whose sums they scale: block b of token h is quad 4 h + b's
#pragma unroll
  for (int i = 0; i < 2; ++i) x.factor[c][i] = __shfl_sync(0xFFFFFFFFu, back, 16 * (t >> 1) + 4 * (2 * (t & 1) + i));
}
// Behind both chunks' gather_chunk: limits the factors.
__device__ __forceinline__ void limit_factors(Columns &x) {
  float most = fmaxf(fmaxf(x.factor[0][0], x.factor[0][1]), fmaxf(x.factor[1][0], x.factor[1][1]));
  most = fmaxf(most, __shfl_xor_sync(0xFFFFFFFFu, most, 1));
  const bool large = most > 0x1p104f;
  x.lift = large ? 512.0f : 1.0f;
  const float down = large ? 1.0f / 512.0f : 1.0f;
#pragma unroll
  for (int i = 0; i < 4; ++i) x.factor[i >> 1][i & 1] *= down;
}
// 8 consecutive 16-bit elements of a row (zeros from `len` on) as packed words
__device__ __forceinline__ void load_row8(uint32_t (&w)[4], const uint16_t *row, uint32_t at, uint32_t len, bool vec) {
  w[0] = w[1] = w[2] = w[3] = 0u;
  if (vec && at + 8u <= len) {
    const uint4 v = ld_v4(row + at);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (at + e < len) w[e >> 1] |= ld_u16(row + at + e) << (16 * (e & 1));
  }
}

// One step: y[group][row half] += the products of this lane's token (2 * group + t / 2) over blocks 2 (t % 2) and
// 2 (t % 2) + 1 of both chunks: the lanes t and t ^ 1 hold the two halves of a sum.
template <int TG>
__device__ __forceinline__ void multiply_step(uint32_t slot, const Columns (&x)[TG], int lane, float (&y)[TG][2]) {
  const int g = lane >> 2, t = lane & 3;
  uint32_t sc[2][2];  // [row half][chunk]: the scale bytes of the chunk's four blocks
#pragma unroll
  for (int h = 0; h < 2; ++h)
    asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(sc[h][0]), "=r"(sc[h][1]) : "r"(slot + CODE_BYTES + (g + 8 * h) * 8));
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    float acc[2][4] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};  // one group: two chains of dependent mmas, too
    uint32_t lo[4], hi[4];
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(lo[0]), "=r"(lo[1]), "=r"(lo[2]), "=r"(lo[3])
                 : "r"(slot + c * 512 + lane * 16));
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                 : "=r"(hi[0]), "=r"(hi[1]), "=r"(hi[2]), "=r"(hi[3])
                 : "r"(slot + (2 + c) * 512 + lane * 16));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t a[4], b[4];
      e2m1_to_f16(lo[j], a);
      e2m1_to_f16(hi[j], b);
#pragma unroll
      for (int q = 0; q < TG; ++q) {
        mma_f16(acc[q], a[0], b[0], a[1], b[1], x[q].v[c][4 * j], x[q].v[c][4 * j + 1]);
        mma_f16(acc[TG == 1 ? 1 : q], a[2], b[2], a[3], b[3], x[q].v[c][4 * j + 2], x[q].v[c][4 * j + 3]);
      }
    }
    if (TG == 1) {
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[0][i] += acc[1][i];
    }
    float s[2][2];  // [row half][block of this lane's pair]
#pragma unroll
    for (int h = 0; h < 2; ++h) e8m0x2(sc[h][c] >> (16 * (t & 1)), s[h][0], s[h][1]);
#pragma unroll
    for (int q = 0; q < TG; ++q) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        y[q][h] = __fmaf_rn(acc[q][2 * h] * x[q].factor[c][0], s[h][0], y[q][h]);
        y[q][h] = __fmaf_rn(acc[q][2 * h + 1] * x[q].factor[c][1], s[h][1], y[q][h]);
      }
    }
  }
}

// y of a tile and step, times lift, into (first) or onto the warp's own sums [2 TG tokens][16 rows]
template <int TG>
__device__ __forceinline__ void keep_sums(float *sums, const Columns (&x)[TG], float (&y)[TG][2], bool first, int lane) {
  const int g = lane >> 2, t = lane & 3;
  const uint32_t at = (uint32_t)__cvta_generic_to_shared(sums + (t >> 1) * 16 + g);
#pragma unroll
  for (int q = 0; q < TG; ++q) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v = y[q][h] + __shfl_xor_sync(0xFFFFFFFFu, y[q][h], 1);
      float old = 0.0f;
      if (!first) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(old) : "r"(at + (32 * q + 8 * h) * 4));
      v = __fmaf_rn(v, x[q].lift, old);
      asm volatile("{\n\t.reg .pred p;\n\tsetp.eq.u32 p, %2, 0;\n\t@p st.shared.f32 [%0], %1;\n\t}" ::"r"(at + (32 * q + 8 * h) * 4), "f"(v), "r"(t & 1)
                   : "memory");
    }
  }
}

}  // namespace mxmma
}  // namespace sklb
