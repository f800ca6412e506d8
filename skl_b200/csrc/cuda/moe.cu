// moe.cu -- a mixture-of-experts layer for few tokens: from the router's logits to the combined output.
//
//   id[j], gate[j]   the topk largest logits of a token (ties to the lowest index) and their softmax
//   h = silu(G_e x) * (U_e x)   for each (token, expert) pair, G_e / U_e the first and last f rows of w1[e]
//   y = sum_j gate[j] * W2_e h
//
// With few tokens the layer is a stream of the met experts' weights from HBM (2 bytes or 17/32 byte per element) with a few
// multiply-adds each; everything is laid out so that each weight is read once and many loads are in flight:
//   route     the pairs sorted by expert: a list of the experts that are met, each with its pairs in token order;
//   up        one CTA for 32 features of one met expert: warps take 8 gate rows with their 8 up rows (one 16-row mma tile) and
//             a part of d; the sums of the parts meet in shared memory, where h is formed; h stays fp32;
//   down      a cluster of CTAs for 16 or 32 rows of W2: its warps take (expert, 256 elements of f) items in turn, each
//             adding gate * product into sums of its own, which are added over warps and CTAs in a fixed order at the end.
// Columns of the mma hold the tokens of an expert.  16-bit weights: mma.sync bf16, eight columns; x enters as it is, h as the
// sum of two bf16 values in two columns (16 significant bits, so that h is not rounded to 8).  4-bit weights: mxf4_mma.cuh;
// h enters as fp16 with a power of two per block of 32 (11 significant bits, against 8 of the result).
#include "mxf4_mma.cuh"

namespace sklb {
namespace {

using namespace mxmma;

constexpr int WARPS = 8, THREADS = 32 * WARPS;
constexpr int UP_TILES = 4, UP_PARTS = WARPS / UP_TILES;  // 8-feature tiles of a CTA, parts of d
constexpr int BSTEP = 128;                                // elements of k of one 16-bit step
constexpr int MAX_TOKENS = 64, MAX_EXPERTS = 1024, MAX_TOPK = 32;

// What route leaves in the workspace: n | expert[n] | first pair[n + 1] | pairs (token * topk + j), sorted by expert
struct Lists {
  int32_t *n, *expert, *first, *pairs;
};
struct MoeParams {
  const float *logits;
  int64_t rsl;
  const uint16_t *x;
  int64_t rsx;
  const uint8_t *w1, *s1, *w2, *s2;
  uint16_t *y;
  int64_t rsy;
  int32_t *ids;
  float *gates, *h;
  Lists list;
  uint32_t m, d, f, experts, topk;
  int renormalise, x_vec, h_vec;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// ------------------------------------------------------------------------------------------------------------ route
// order-preserving key of a logit: larger value, larger key; NaN above everything, -0 equal to +0; 0 is never a value's key
__device__ __forceinline__ uint32_t logit_key(float v) {
  const uint32_t u = f2u(__fadd_rn(v, 0.0f));
  return v != v ? 0xFFFFFFFFu : ((u >> 31) ? ~u : u | 0x80000000u);
}

// One warp, one token: ids and gates to global memory, the ids of the routed slots (-1: a logit of minus infinity, which
// routes nowhere) to `slots`.  keys: `experts` words of this warp's shared memory.
__device__ __forceinline__ void route_token(const MoeParams &p, uint32_t tok, uint32_t *keys, int32_t *slots, int lane) {
  const float *row = p.logits + (int64_t)tok * p.rsl;
  uint32_t best = 0u, at = 0xFFFFFFFFu;  // this lane's largest key and its lowest index
  for (uint32_t e = lane; e < p.experts; e += 32u) {
    const uint32_t key = logit_key(u2f(ld_u32(row + e)));
    keys[e] = key;
    if (key > best) best = key, at = e;
  }
  __syncwarp();
  float top = 0.0f, mine = 0.0f;  // the largest logit; lane j keeps exp(logit_j - top)
  bool routed = false;
  int32_t my_id = -1;
  for (uint32_t j = 0; j < p.topk; ++j) {
    const uint32_t k = __reduce_max_sync(0xFFFFFFFFu, best);
    const uint32_t e = __reduce_min_sync(0xFFFFFFFFu, best == k ? at : 0xFFFFFFFFu);
    const float v = u2f(ld_u32(row + e));
    if (j == 0) top = v;
    if ((uint32_t)lane == j) {
      my_id = (int32_t)e;
      routed = k != 0x007FFFFFu;  // the key of minus infinity
      mine = routed ? expf(__fsub_rn(v, top)) : 0.0f;
    }
    if (at == e) {  // the owner of the winner looks for its next one
      keys[e] = 0u;
      best = 0u, at = 0xFFFFFFFFu;
      for (uint32_t i = lane; i < p.experts; i += 32u) {
        const uint32_t key = keys[i];
        if (key > best) best = key, at = i;
      }
    }
  }
  float sum = 0.0f;
  if (p.renormalise) {
    sum = mine;
  } else {
    for (uint32_t e = lane; e < p.experts; e += 32u) {
      const float v = u2f(ld_u32(row + e));
      sum += v == -INFINITY ? 0.0f : expf(__fsub_rn(v, top));
    }
  }
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xFFFFFFFFu, sum, off));
  if ((uint32_t)lane < p.topk) {
    const uint32_t pair = tok * p.topk + lane;
    slots[pair] = routed ? my_id : -1;
    p.ids[pair] = my_id;
    p.gates[pair] = routed ? __fdiv_rn(mine, sum) : 0.0f;
  }
}

// One CTA: every token's choice, then the lists.  Shared memory: keys [warps][experts] | slots [m * topk] | counts [experts].
__global__ void __launch_bounds__(512) route_kernel(const MoeParams p) {
  extern __shared__ __align__(16) uint32_t rsmem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const uint32_t pairs = p.m * p.topk;
  uint32_t *keys = rsmem + warp * p.experts;
  int32_t *slots = reinterpret_cast<int32_t *>(rsmem + warps * p.experts);
  int32_t *counts = slots + pairs;
  dep_wait();
  for (uint32_t tok = warp; tok < p.m; tok += warps) route_token(p, tok, keys, slots, lane);
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < p.experts; e += blockDim.x) {
    int32_t c = 0;
    for (uint32_t i = 0; i < pairs; ++i) c += slots[i] == (int32_t)e;
    counts[e] = c;
  }
  __syncthreads();
  if (warp == 0) {  // experts in ascending order: position in the list and first pair
    int32_t n = 0, first = 0;
    for (uint32_t e0 = 0; e0 < p.experts; e0 += 32u) {
      const uint32_t e = e0 + lane;
      const int32_t c = e < p.experts ? counts[e] : 0;
      const uint32_t met = __ballot_sync(0xFFFFFFFFu, c > 0);
      int32_t incl = c;
#pragma unroll
      for (int off = 1; off < 32; off <<= 1) {
        const int32_t o = __shfl_up_sync(0xFFFFFFFFu, incl, off);
        if (lane >= off) incl += o;
      }
      if (c > 0) {
        const int32_t a = n + __popc(met & ((1u << lane) - 1u));
        p.list.expert[a] = (int32_t)e;
        p.list.first[a] = first + incl - c;
      }
      if (e < p.experts) counts[e] = first + incl - c;
      n += __popc(met);
      first += __shfl_sync(0xFFFFFFFFu, incl, 31);
    }
    if (lane == 0) {
      *p.list.n = n;
      p.list.first[n] = first;
    }
  }
  __syncthreads();
  for (uint32_t e = threadIdx.x; e < p.experts; e += blockDim.x) {
    int32_t at = counts[e];
    for (uint32_t i = 0; i < pairs; ++i)
      if (slots[i] == (int32_t)e) p.list.pairs[at++] = (int32_t)i;
  }
}

// ------------------------------------------------------------------------------------------------------ 16-bit step
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Lane (g, t) holds 8 consecutive elements of rows g and g + 8 in each 32-element piece of the step: the order of k inside
// an mma does not matter as long as both operands use the same one.
struct Wide {
  uint4 v[2][4];
};
template <bool VEC>
__device__ __forceinline__ void load_wide(Wide &w, const uint16_t *const (&rows)[2], uint32_t step, uint32_t cols, int t) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const uint32_t e = step * BSTEP + c * 32u + t * 8u;
      w.v[h][c] = make_uint4(0u, 0u, 0u, 0u);
      if (VEC) {  // cols is a multiple of 8
        if (e < cols) w.v[h][c] = ld_stream_v4(rows[h] + e);
      } else {
        uint32_t q[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (e + i < cols) q[i >> 1] |= ld_u16(rows[h] + e + i) << (16 * (i & 1));
        w.v[h][c] = make_uint4(q[0], q[1], q[2], q[3]);
      }
    }
  }
}
// x: shared address of column 0 at the step's first element; columns behind `last` repeat it and are ignored by the caller
__device__ __forceinline__ void multiply_wide(const Wide &w, uint32_t x, uint32_t pitch, uint32_t last, int g, int t,
                                              float (&acc)[4]) {
  const uint32_t at = x + min((uint32_t)g, last) * pitch + t * 16u;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    uint32_t b[4];
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(at + 64u * c));
    mma_bf16(acc, w.v[0][c].x, w.v[1][c].x, w.v[0][c].y, w.v[1][c].y, b[0], b[1]);
    mma_bf16(acc, w.v[0][c].z, w.v[1][c].z, w.v[0][c].w, w.v[1][c].w, b[2], b[3]);
  }
}

// --------------------------------------------------------------------------------------------------------------- up
// 8 elements of a bf16 row (zeros behind `cols`) as packed words
__device__ __forceinline__ void load_x8(uint32_t (&w)[4], const uint16_t *row, uint32_t at, uint32_t cols, bool vec) {
  w[0] = w[1] = w[2] = w[3] = 0u;
  if (vec && at + 8u <= cols) {
    const uint4 v = ld_v4(row + at);
    w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (at + e < cols) w[e >> 1] |= ld_u16(row + at + e) << (16 * (e & 1));
  }
}
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// sums[token][16 rows] = this warp's part of the products of up to 2 TG tokens: its steps of d
template <int TG, bool VEC>
__device__ __forceinline__ void up_steps_mx(const RowPair &rows, Weights w, uint32_t step, uint32_t steps, uint32_t kblocks,
                                            uint32_t x, uint32_t x_pitch, uint32_t f, uint32_t f_pitch, uint32_t last,
                                            uint32_t zeros, int g, int t, float *sums) {
  float y[TG][2];
#pragma unroll
  for (int q = 0; q < TG; ++q) y[q][0] = y[q][1] = 0.0f;
  while (step < steps) {
    const uint32_t next = step + UP_PARTS;
    Weights wn;
    if (next < steps) load_step<VEC>(wn, rows, next, kblocks, t);
    multiply_step<TG, true>(w, x + step * (STEP * 2), x_pitch, f + step * (STEP / 8), f_pitch, last, zeros, g, t, y);
    w = wn;
    step = next;
  }
#pragma unroll
  for (int q = 0; q < TG; ++q) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      y[q][h] += __shfl_xor_sync(0xFFFFFFFFu, y[q][h], 1);
      if ((t & 1) == 0) sums[(2 * q + (t >> 1)) * 16 + g + 8 * h] = y[q][h];
    }
  }
}

// Shared memory: 64 bytes of zeros | sums [8 warps][8 tokens][16] | x (4-bit: fp16 [8][steps * 256], then factors
// [8][steps * 8]; 16-bit: bf16 [8][pitch], the pitch 64 bytes more than a multiple of 128 so that the eight rows of an mma
// operand are read without bank conflicts).  A pass takes up to `per_pass` tokens of the expert.
template <bool MX, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) up_kernel(const MoeParams p, uint32_t per_pass) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int tile = warp % UP_TILES, part = warp / UP_TILES;
  const uint32_t steps = MX ? (p.d + STEP - 1) / STEP : (p.d + BSTEP - 1) / BSTEP, kblocks = (p.d + 31u) / 32u;
  const uint32_t x_pitch = MX ? steps * (STEP * 2) : steps * (BSTEP * 2) + 64u, f_pitch = steps * (STEP / 8);
  float *sums = reinterpret_cast<float *>(smem + 64);
  const uint32_t zeros = smem_addr(smem), x = zeros + 64u + WARPS * 8 * 16 * 4, f = x + per_pass * x_pitch;
  const uint32_t feature0 = blockIdx.x * (8u * UP_TILES);
  if (threadIdx.x < 16) reinterpret_cast<uint32_t *>(smem)[threadIdx.x] = 0u;

  dep_wait();
  if ((int32_t)blockIdx.y >= *p.list.n) return;
  const uint32_t e = (uint32_t)p.list.expert[blockIdx.y];
  const int32_t first = p.list.first[blockIdx.y], last = p.list.first[blockIdx.y + 1];

  const uint32_t feat = min(feature0 + 8u * tile + g, p.f - 1u);  // features behind the last are not stored
  RowPair rows;
  const uint16_t *wide[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint64_t r = (uint64_t)e * 2u * p.f + (h ? p.f : 0u) + feat;
    if (MX) {
      rows.code[h] = p.w1 + r * kblocks * 16u;
      rows.scale[h] = p.s1 + r * kblocks;
    } else {
      wide[h] = reinterpret_cast<const uint16_t *>(p.w1) + r * p.d;
    }
  }
  for (int32_t at = first; at < last; at += (int32_t)per_pass) {
    const uint32_t cnt = min((uint32_t)(last - at), per_pass);
    Weights w;
    Wide wb;
    if ((uint32_t)part < steps) {
      if (MX) load_step<VEC>(w, rows, part, kblocks, t);
      else load_wide<VEC>(wb, wide, part, p.d, t);
    }
    // the tokens' activations; four lanes share a block of 32
    const uint32_t groups = steps * (MX ? STEP / 8 : BSTEP / 8), total = cnt * groups;
    for (uint32_t i0 = 0; i0 < total; i0 += THREADS) {
      const uint32_t i = i0 + threadIdx.x;
      const bool in = i < total;
      const uint32_t j = in ? i / groups : 0u, gr = in ? i - j * groups : 0u;
      uint32_t v[4];
      const uint32_t tok = (uint32_t)p.list.pairs[at + j] / p.topk;
      load_x8(v, p.x + (int64_t)tok * p.rsx, gr * 8u, in ? p.d : 0u, p.x_vec);
      if (MX) {
        uint32_t top = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) top = max(top, max(v[q] << 16 & 0x7FFFFFFFu, v[q] & 0x7FFF0000u));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        float back;
        const float factor = block_factor(top, back);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = pack_f16x2_no_nan(dec_bf16(v[q] & 0xFFFFu) * factor, u2f(v[q] & 0xFFFF0000u) * factor);
        if (in && (gr & 3u) == 0u) asm volatile("st.shared.f32 [%0], %1;" ::"r"(f + j * f_pitch + gr), "f"(back) : "memory");
      }
      if (in) st_shared_v4(x + j * x_pitch + gr * 16u, v[0], v[1], v[2], v[3]);
    }
    __syncthreads();
    float *own = sums + warp * (8 * 16);
    if (MX) {
      if (cnt <= 2) up_steps_mx<1, VEC>(rows, w, part, steps, kblocks, x, x_pitch, f, f_pitch, cnt - 1u, zeros, g, t, own);
      else if (cnt <= 4) up_steps_mx<2, VEC>(rows, w, part, steps, kblocks, x, x_pitch, f, f_pitch, cnt - 1u, zeros, g, t, own);
      else up_steps_mx<4, VEC>(rows, w, part, steps, kblocks, x, x_pitch, f, f_pitch, cnt - 1u, zeros, g, t, own);
    } else {
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (uint32_t step = part; step < steps;) {
        const uint32_t next = step + UP_PARTS;
        Wide wn;
        if (next < steps) load_wide<VEC>(wn, wide, next, p.d, t);
        multiply_wide(wb, x + step * (BSTEP * 2), x_pitch, cnt - 1u, g, t, acc);
        wb = wn;
        step = next;
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) own[(2 * t + (q & 1)) * 16 + g + 8 * (q >> 1)] = acc[q];
    }
    __syncthreads();
    {  // one (token, feature) per thread: h = silu(gate) * up
      const uint32_t j = threadIdx.x / 32u, c = threadIdx.x & 31u, feature = feature0 + c;
      if (j < cnt && feature < p.f) {
        const float *s = sums + (c / 8u) * (8 * 16) + j * 16 + (c & 7u);
        float gate = 0.0f, up = 0.0f;
#pragma unroll
        for (int q = 0; q < UP_PARTS; ++q) {
          gate += s[q * UP_TILES * (8 * 16)];
          up += s[q * UP_TILES * (8 * 16) + 8];
        }
        p.h[(uint64_t)p.list.pairs[at + j] * p.f + feature] = __fmul_rn(__fmul_rn(logistic_f32(1.0f, gate), gate), up);
      }
    }
    // the next pass writes x and sums again: x only after this pass's multiplications, which the barrier above ended; the
    // sums only after its own first barrier
  }
}

// ------------------------------------------------------------------------------------------------------------- down
constexpr int DOWN_K = 256;  // elements of f of one item

// Shared memory: 64 bytes of zeros | per warp: h of the item (4-bit: fp16 [4][256], factors [4][8]; 16-bit: bf16 hi of four
// tokens, then lo, [8][256] with a pitch of 576 bytes) | per warp: sums [m][rows]
template <bool MX>
struct Down {
  static constexpr int RT = MX ? 2 : 1;  // 16-row tiles of a warp
  static constexpr int ROWS = 16 * RT;
  static constexpr int PASS = 4;         // tokens at a time
  static constexpr int PITCH = MX ? DOWN_K * 2 : DOWN_K * 2 + 64;
  static constexpr int STAGE = MX ? PASS * PITCH + PASS * (DOWN_K / 32) * 4 : 2 * PASS * PITCH;
  static constexpr size_t smem(uint32_t m) { return 64 + (size_t)WARPS * STAGE + (size_t)WARPS * m * ROWS * 4; }
};

template <bool MX, bool VEC>
__global__ void __launch_bounds__(THREADS, 2) down_kernel(const MoeParams p) {
  using D = Down<MX>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const uint32_t row0 = (blockIdx.x / ranks) * D::ROWS;
  const uint32_t zeros = smem_addr(smem), stage = zeros + 64u + warp * D::STAGE, factors = stage + D::PASS * D::PITCH;
  float *all = reinterpret_cast<float *>(smem + 64 + WARPS * D::STAGE);  // [warp][m][ROWS]
  float *own = all + (size_t)warp * p.m * D::ROWS;
  if (threadIdx.x < 16) reinterpret_cast<uint32_t *>(smem)[threadIdx.x] = 0u;
  for (uint32_t i = lane; i < p.m * D::ROWS; i += 32u) own[i] = 0.0f;
  __syncthreads();
  dep_wait();

  const uint32_t kblocks = (p.f + 31u) / 32u, parts = (p.f + DOWN_K - 1) / DOWN_K;
  const uint32_t items = (uint32_t)*p.list.n * parts;
  for (uint32_t item = rank * WARPS + warp; item < items; item += ranks * WARPS) {
    const uint32_t a = item / parts, k0 = (item - a * parts) * DOWN_K;
    const uint32_t e = (uint32_t)p.list.expert[a];
    const int32_t first = p.list.first[a], last = p.list.first[a + 1];
    Weights w[D::RT];
    Wide wb[2];
#pragma unroll
    for (int r = 0; r < D::RT; ++r) {
      RowPair rows;
      const uint16_t *wide[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t row = min(row0 + 16u * r + g + 8u * h, p.d - 1u);
        const uint64_t at = (uint64_t)e * p.d + row;
        if (MX) {
          rows.code[h] = p.w2 + at * kblocks * 16u;
          rows.scale[h] = p.s2 + at * kblocks;
        } else {
          wide[h] = reinterpret_cast<const uint16_t *>(p.w2) + at * p.f;
        }
      }
      if (MX) {
        load_step<VEC>(w[r], rows, k0 / STEP, kblocks, t);
      } else {
        load_wide<VEC>(wb[0], wide, k0 / BSTEP, p.f, t);
        load_wide<VEC>(wb[1], wide, k0 / BSTEP + 1u, p.f, t);
      }
    }
    for (int32_t at = first; at < last; at += D::PASS) {
      const uint32_t cnt = min((uint32_t)(last - at), (uint32_t)D::PASS);
      __syncwarp();  // the pass before has read its h
      for (uint32_t j = 0; j < cnt; ++j) {  // lane: 8 consecutive elements of f
        const float *src = p.h + (uint64_t)p.list.pairs[at + j] * p.f;
        const uint32_t col = k0 + lane * 8u;
        float v[8];
        if (p.h_vec && col + 8u <= p.f) {
          const float4 v0 = __ldcg(reinterpret_cast<const float4 *>(src + col)), v1 = __ldcg(reinterpret_cast<const float4 *>(src + col) + 1);
          v[0] = v0.x, v[1] = v0.y, v[2] = v0.z, v[3] = v0.w, v[4] = v1.x, v[5] = v1.y, v[6] = v1.z, v[7] = v1.w;
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) v[q] = col + q < p.f ? __ldcg(src + col + q) : 0.0f;
        }
        if (MX) {
          uint32_t top = 0;
#pragma unroll
          for (int q = 0; q < 8; ++q) top = max(top, f2u(v[q]) & 0x7FFFFFFFu);
          top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
          top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
          float back;
          const float factor = block_factor(top, back);
          st_shared_v4(stage + j * D::PITCH + lane * 16u, pack_f16x2_no_nan(v[0] * factor, v[1] * factor),
                       pack_f16x2_no_nan(v[2] * factor, v[3] * factor), pack_f16x2_no_nan(v[4] * factor, v[5] * factor),
                       pack_f16x2_no_nan(v[6] * factor, v[7] * factor));
          if (t == 0) asm volatile("st.shared.f32 [%0], %1;" ::"r"(factors + j * (DOWN_K / 32) * 4u + g * 4u), "f"(back) : "memory");
        } else {
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            hi[q] = pack_bf16x2_no_nan(v[2 * q], v[2 * q + 1]);
            const float a0 = u2f(hi[q] << 16), a1 = u2f(hi[q] & 0xFFFF0000u);
            // an infinity or NaN stays in the first part
            lo[q] = pack_bf16x2_no_nan(fabsf(a0) < INFINITY ? v[2 * q] - a0 : 0.0f, fabsf(a1) < INFINITY ? v[2 * q + 1] - a1 : 0.0f);
          }
          st_shared_v4(stage + j * D::PITCH + lane * 16u, hi[0], hi[1], hi[2], hi[3]);
          st_shared_v4(stage + (j + D::PASS) * D::PITCH + lane * 16u, lo[0], lo[1], lo[2], lo[3]);
        }
      }
      __syncwarp();
      if (MX) {
#pragma unroll
        for (int r = 0; r < D::RT; ++r) {
          float y[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
          if (cnt <= 2) {
            float(&y1)[1][2] = reinterpret_cast<float(&)[1][2]>(y);
            multiply_step<1, true>(w[r], stage, D::PITCH, factors, DOWN_K / 32 * 4, cnt - 1u, zeros, g, t, y1);
          } else {
            multiply_step<2, true>(w[r], stage, D::PITCH, factors, DOWN_K / 32 * 4, cnt - 1u, zeros, g, t, y);
          }
#pragma unroll
          for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float v = y[q][h] + __shfl_xor_sync(0xFFFFFFFFu, y[q][h], 1);
              const uint32_t j = 2u * q + (uint32_t)(t >> 1);
              if ((t & 1) == 0 && j < cnt) {
                const uint32_t pair = (uint32_t)p.list.pairs[at + j];
                float *o = own + (pair / p.topk) * D::ROWS + 16 * r + g + 8 * h;
                *o = __fmaf_rn(p.gates[pair], v, *o);
              }
            }
          }
        }
      } else {
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        multiply_wide(wb[0], stage, D::PITCH, 7u, g, t, acc);
        multiply_wide(wb[1], stage + BSTEP * 2, D::PITCH, 7u, g, t, acc);
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // columns 2 t, 2 t + 1: the first part of tokens 0..3 in lanes t = 0, 1, the second in 2, 3
          const float v = acc[q] + __shfl_xor_sync(0xFFFFFFFFu, acc[q], 2);
          const uint32_t j = 2u * t + (q & 1);
          if (t < 2 && j < cnt) {
            const uint32_t pair = (uint32_t)p.list.pairs[at + j];
            float *o = own + (pair / p.topk) * D::ROWS + g + 8 * (q >> 1);
            *o = __fmaf_rn(p.gates[pair], v, *o);
          }
        }
      }
    }
  }
  __syncthreads();
  // over the warps, then over the cluster's CTAs, in order
  const uint32_t outs = p.m * D::ROWS;
  for (uint32_t i = threadIdx.x; i < outs; i += THREADS) {
    float v = all[i];
#pragma unroll
    for (int q = 1; q < WARPS; ++q) v += all[(size_t)q * outs + i];
    all[i] = v;
  }
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
  for (uint32_t i = rank * THREADS + threadIdx.x; i < outs; i += ranks * THREADS) {
    float v = 0.0f;
    const uint32_t at = smem_addr(all + i);
    for (uint32_t r = 0; r < ranks; ++r) {
      uint32_t remote;
      float part;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(r));
      asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(remote) : "memory");
      v += part;
    }
    const uint32_t tok = i / D::ROWS, row = row0 + i % D::ROWS;
    if (row < p.d) p.y[(int64_t)tok * p.rsy + row] = (uint16_t)enc_bf16(v);
  }
  // no CTA leaves while its shared memory may still be read
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename... P, typename... A>
cudaError_t launch(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, unsigned ranks, cudaStream_t s, A... args) {
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SKLB_COUNT_LAUNCH();
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
}

constexpr size_t UP_BUDGET = 96 * 1024;  // activations of one pass: two CTAs on an SM

template <bool MX, bool VEC>
cudaError_t launch_moe(const MoeParams &p, cudaStream_t s) {
  const uint32_t pairs = p.m * p.topk, met = pairs < p.experts ? pairs : p.experts;
  const unsigned warps = p.m < 16 ? p.m : 16;
  cudaError_t e = launch(route_kernel, dim3(1), 32 * warps, ((size_t)warps * p.experts + pairs + p.experts) * 4, 1, s, p);
  if (e != cudaSuccess) return e;
  const uint32_t steps = MX ? (p.d + STEP - 1) / STEP : (p.d + BSTEP - 1) / BSTEP;
  const size_t per_token = MX ? (size_t)steps * (STEP * 2 + STEP / 8) : (size_t)steps * (BSTEP * 2) + 64;
  uint32_t per_pass = p.m < 8 ? p.m : 8;
  while (per_pass > 1 && per_pass * per_token > UP_BUDGET) --per_pass;
  e = launch(up_kernel<MX, VEC>, dim3((p.f + 31) / 32, met), THREADS, 64 + WARPS * 8 * 16 * 4 + per_pass * per_token, 1, s, p,
             per_pass);
  if (e != cudaSuccess) return e;
  // CTAs of a cluster: as many as find an item for each warp, at most 8
  const uint32_t items = met * ((p.f + DOWN_K - 1) / DOWN_K);
  unsigned ranks = 1;
  while (ranks < 8 && items > ranks * WARPS) ranks *= 2;
  const uint32_t tiles = (p.d + Down<MX>::ROWS - 1) / Down<MX>::ROWS;
  return launch(down_kernel<MX, VEC>, dim3(tiles * ranks), THREADS, Down<MX>::smem(p.m), ranks, s, p);
}

}  // namespace
}  // namespace sklb

using namespace sklb;

extern "C" int skl_b200_moe_supported(uint64_t m, uint64_t d, uint64_t f, uint64_t experts, uint64_t topk) {
  return m <= MAX_TOKENS && d <= 32768 && f <= 32768 && experts <= MAX_EXPERTS && topk <= MAX_TOPK;
}

// h [m * topk][f] fp32, then n, expert[], first[], pairs[]
extern "C" size_t skl_b200_moe_scratch_bytes(uint64_t m, uint64_t f, uint64_t experts, uint64_t topk) {
  const size_t pairs = (size_t)(m * topk), met = pairs < experts ? pairs : (size_t)experts;
  return (pairs * (size_t)f + 1 + met + met + 1 + pairs) * 4;
}

extern "C" int skl_b200_launch_moe(const skl_b200_moe_args *q, void *stream) {
  MoeParams p;
  p.logits = (const float *)q->logits, p.rsl = q->rsl;
  p.x = (const uint16_t *)q->x, p.rsx = q->rsx;
  p.w1 = (const uint8_t *)q->w1, p.s1 = (const uint8_t *)q->s1, p.w2 = (const uint8_t *)q->w2, p.s2 = (const uint8_t *)q->s2;
  p.y = (uint16_t *)q->y, p.rsy = q->rsy;
  p.ids = (int32_t *)q->ids, p.gates = (float *)q->gates;
  p.m = q->m, p.d = q->d, p.f = q->f, p.experts = q->experts, p.topk = q->topk, p.renormalise = q->renormalise;
  p.x_vec = (reinterpret_cast<uintptr_t>(p.x) & 15u) == 0 && (p.m == 1 || p.rsx % 8 == 0);
  const size_t pairs = (size_t)p.m * p.topk, met = pairs < p.experts ? pairs : p.experts;
  p.h = (float *)q->workspace;
  p.h_vec = (reinterpret_cast<uintptr_t>(p.h) & 15u) == 0 && p.f % 4 == 0;
  p.list.n = (int32_t *)(p.h + pairs * p.f);
  p.list.expert = p.list.n + 1;
  p.list.first = p.list.expert + met;
  p.list.pairs = p.list.first + met + 1;
  cudaStream_t s = (cudaStream_t)stream;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(p.w1) | reinterpret_cast<uintptr_t>(p.w2);
  if (q->mx) {
    // 16-byte loads of codes, 8-byte loads of scales: packed rows are always whole blocks of 16 bytes
    const bool vec = (bases & 15u) == 0 && ((reinterpret_cast<uintptr_t>(p.s1) | reinterpret_cast<uintptr_t>(p.s2)) & 7u) == 0 &&
                     (p.d + 31) / 32 % 8 == 0 && (p.f + 31) / 32 % 8 == 0;
    return (int)(vec ? launch_moe<true, true>(p, s) : launch_moe<true, false>(p, s));
  }
  const bool vec = (bases & 15u) == 0 && p.d % 8 == 0 && p.f % 8 == 0;
  return (int)(vec ? launch_moe<false, true>(p, s) : launch_moe<false, false>(p, s));
}
