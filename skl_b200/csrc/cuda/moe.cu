// moe.cu -- a mixture-of-experts layer for few tokens: from the router's logits to the combined output.
//
//   id[j], gate[j]   the topk largest logits of a token (ties to the lowest index) and their softmax
//   h = silu(G_e x) * (U_e x)   for each (token, expert) pair, G_e / U_e the first and last f rows of w1[e]
//   y = sum_j gate[j] * W2_e h
//
// With few tokens the layer is a stream of the met experts' weights from HBM (2 bytes or 17/32 byte per element) with a few
// multiply-adds each.  Two kernels of one CTA of 16 warps per SM; each warp streams 16-row pieces of the weights through a
// ring in shared memory (mxf4_mma.cuh), so that about 100 KB are in flight on an SM; weights are read once for up to 4 tokens of an
// expert, and in `down` for any number:
//   up     every CTA finds the routing itself (a warp per token; cheaper than a kernel before it) and takes an equal run of the
//          tiles of all met experts, 8 gate rows with their 8 up rows to a tile, so that both sums of a feature end in the
//          same CTA.  Warps split d, their sums meet in shared memory, where h is formed.
//   down   a CTA owns up to 16 rows of W2 of every expert, so nothing has to be added across CTAs; its warps take (expert,
//          piece of f) items in turn, each adding gate * product to sums of its own, which are added in order at the end.
// Columns of the mma hold the tokens of an expert, at most 4 at a time.  16-bit weights: mma.sync bf16; x enters as it is, h as
// the sum of two bf16 values in two columns (16 significant bits, so that h is not rounded to 8).  4-bit weights:
// mxf4_mma.cuh; h is kept as fp16 with a power of two per block of 32 (11 significant bits, against 8 of the result; elements
// below 2^-28 of their block's largest have fewer), which every CTA of `down` can copy as it is: converting fp32 there took as
// many instructions as the products.  Against h in fp32 a tenth of the results differ in their last bit, 8.6e-4 in the 2-norm,
// half of bf16's own rounding (1.65e-3 either way against 64 bits).
//
// d 2048, f 1024, 8 of 64 experts, in a graph over three sets of weights: one token, bf16 weights (100 MB), 28.5 us: the routing
// (about 5 us) and two streams, each with its start and end; MX-FP4 17.0.  16 tokens, MX-FP4 (187 MB): 74 us, two thirds of them
// `up`; bound by the issue slots (half busy) and the latency of dependent instructions, about 400 instructions of a warp for
// 16 x 256 weights.  16 tokens, bf16: 145 us, 4.8 TB/s.
#include "mxf4_mma.cuh"

namespace sklb {
namespace {

using namespace mxmma;

constexpr int WARPS = 16, THREADS = 32 * WARPS;
constexpr int PASS = 4;  // tokens of an expert at a time
constexpr int MAX_TOKENS = 64, MAX_EXPERTS = 1024, MAX_TOPK = 32;
constexpr size_t MAX_SMEM = 226 * 1024;

// 4-bit weights: the factors of h's blocks reach 2^113, and a block's sum of 2^23 times that would leave fp32's range before the
// weights' scale brings it back (see Columns).  They are kept divided by this, and the gates multiplied by it; a block's sum is then
// exact to 2^-141 times its scale.
constexpr float H_LIFT = 512.0f;

// The routed pairs (token * topk + j) sorted by expert: n experts met, in ascending order, expert[a] with the pairs
// pairs[first[a]] .. pairs[first[a + 1] - 1], in token order; they are taken `per_pass` at a time, passes before expert a: turn[a].
// turn[] only in the first kernel; token[], gate[]: of the pairs, in the same order, only in the workspace for the second.
struct Lists {
  int32_t *n, *expert, *first, *turn, *pairs, *token;
  float *gate;
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
  float *gates;
  float *h;        // 16-bit weights: [pairs][f]
  uint16_t *h16;   // 4-bit weights: [pairs][f up to a multiple of 32] and a factor per block [pairs][blocks]
  float *hf;
  Lists list;  // in the workspace, for the second kernel
  uint32_t m, d, f, experts, topk, met;  // met: the most experts that can be met
  uint32_t per_pass, k_warps, down_rows;
  int renormalise, x_vec, h_vec;
};

// What differs between the two weight formats: elements of a 128-byte step and bytes of a slot.
template <bool MX>
struct Format {
  static constexpr uint32_t K = MX ? 256 : 64;
  static constexpr uint32_t SLOT = MX ? SLOT_BYTES : CODE_BYTES;
  static __host__ __device__ uint32_t row_bytes(uint32_t cols) { return MX ? (cols + 31u) / 32u * 16u : cols * 2u; }
  static __host__ __device__ uint32_t steps(uint32_t cols) { return (cols + K - 1u) / K; }
  // a token's bf16 activations in shared memory: a pitch 64 bytes more than a multiple of 128, so that the rows of an mma
  // operand are read without bank conflicts
  static __host__ __device__ uint32_t x_pitch(uint32_t steps) { return steps * (K * 2u) + 64u; }
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__host__ __device__ __forceinline__ uint32_t h_pitch(uint32_t f) { return (f + 31u) / 32u * 32u; }

// ------------------------------------------------------------------------------------------------------------ route
// order-preserving key of a logit: larger value, larger key; NaN above everything, -0 equal to +0; 0 is never a value's key
__device__ __forceinline__ uint32_t logit_key(float v) {
  const uint32_t u = f2u(__fadd_rn(v, 0.0f));
  return v != v ? 0xFFFFFFFFu : ((u >> 31) ? ~u : u | 0x80000000u);
}
__device__ __forceinline__ float key_logit(uint32_t key) { return u2f((key >> 31) ? key & 0x7FFFFFFFu : ~key); }

// One warp, one token: the routed slots (-1: a logit of minus infinity, which routes nowhere), the token's bit for each of its
// experts (tokens[2][experts]) and, with `write`, ids and gates to global memory.  The keys stay in registers up to 128 experts, above that in `keys`, `experts` words of this warp's
// shared memory.
__device__ __forceinline__ void route_token(const MoeParams &p, uint32_t tok, uint32_t *keys, int32_t *slots, uint32_t *tokens, int lane,
                                            bool write) {
  const float *row = p.logits + (int64_t)tok * p.rsl;
  const bool small = p.experts <= 128u;
  uint32_t reg[4];  // experts lane, lane + 32, ...
#pragma unroll
  for (int i = 0; i < 4; ++i) reg[i] = lane + 32u * i < p.experts && small ? logit_key(u2f(ld_u32(row + lane + 32 * i))) : 0u;
  uint32_t best = 0u, at = 0xFFFFFFFFu;  // this lane's largest key and its lowest index
  if (!small) {
    for (uint32_t e = lane; e < p.experts; e += 32u) {
      const uint32_t key = logit_key(u2f(ld_u32(row + e)));
      keys[e] = key;
      if (key > best) best = key, at = e;
    }
  }
  auto scan = [&]() {
    best = 0u, at = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (reg[i] > best) best = reg[i], at = lane + 32u * i;
  };
  if (small) scan();
  float top = 0.0f, mine = 0.0f, all = 0.0f;  // the largest logit; lane j keeps exp(logit_j - top)
  bool routed = false;
  int32_t my_id = -1;
  for (uint32_t j = 0; j < p.topk; ++j) {
    const uint32_t k = __reduce_max_sync(0xFFFFFFFFu, best);
    const uint32_t e = __reduce_min_sync(0xFFFFFFFFu, best == k ? at : 0xFFFFFFFFu);
    const float v = key_logit(k);
    if (j == 0) {
      top = v;
      if (write && !p.renormalise) {
        for (uint32_t i = lane; i < p.experts; i += 32u) {
          const float w = u2f(ld_u32(row + i));
          all += w == -INFINITY ? 0.0f : expf(__fsub_rn(w, top));
        }
      }
    }
    if ((uint32_t)lane == j) {
      my_id = (int32_t)e;
      routed = v != -INFINITY;
      mine = routed ? expf(__fsub_rn(v, top)) : 0.0f;
    }
    // the owner of the winner looks for its next one
    if (small) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (lane + 32u * i == e) reg[i] = 0u;
      scan();
    } else if (at == e) {
      keys[e] = 0u;
      best = 0u, at = 0xFFFFFFFFu;
      for (uint32_t i = lane; i < p.experts; i += 32u) {
        const uint32_t key = keys[i];
        if (key > best) best = key, at = i;
      }
    }
  }
  if ((uint32_t)lane < p.topk) slots[tok * p.topk + lane] = routed ? my_id : -1;
  if (routed) atomicOr(tokens + (tok >> 5) * p.experts + my_id, 1u << (tok & 31u));
  if (!write) return;
  float sum = p.renormalise ? mine : all;
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) sum = __fadd_rn(sum, __shfl_xor_sync(0xFFFFFFFFu, sum, off));
  if ((uint32_t)lane < p.topk) {
    p.ids[tok * p.topk + lane] = my_id;
    p.gates[tok * p.topk + lane] = routed ? __fdiv_rn(mine, sum) : 0.0f;
  }
}

// The whole CTA: every token's choice, then the lists.  A token has an expert at most once, so 64 bits tell an expert's tokens,
// how many there are and which comes when; one scan over the experts places them.  (Comparing every pair with every other took
// several times as long from 16 tokens on.)  scratch, in words: totals of the warps [32] | tokens [2][experts] | first pair of an
// expert [experts] | slots [pairs] | with more than 128 experts keys [warps][experts].
__device__ void route(const MoeParams &p, uint32_t *scratch, const Lists &out, bool mx, bool write) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t pairs = p.m * p.topk;
  unsigned long long *totals = reinterpret_cast<unsigned long long *>(scratch);
  uint32_t *tokens = scratch + 32, *base = tokens + 2u * p.experts, *keys = base + p.experts + pairs;
  int32_t *slots = reinterpret_cast<int32_t *>(base + p.experts);
  for (uint32_t i = threadIdx.x; i < 2u * p.experts; i += THREADS) tokens[i] = 0u;
  __syncthreads();
  dep_wait();
  for (uint32_t tok = warp; tok < p.m; tok += WARPS) route_token(p, tok, keys + warp * p.experts, slots, tokens, lane, write);
  __syncthreads();
  // experts 2 tid and 2 tid + 1: pairs | met << 16 | passes << 32 (at most 2048, 1024 and 2048), summed up over the experts
  unsigned long long own[2], sum;
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint32_t e = 2u * threadIdx.x + q;
    const uint32_t c = e < p.experts ? __popc(tokens[e]) + __popc(tokens[p.experts + e]) : 0u;
    own[q] = (unsigned long long)((c + p.per_pass - 1u) / p.per_pass) << 32 | (c != 0u ? 0x10000u : 0u) | c;
  }
  sum = own[0] + own[1];
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const unsigned long long o = __shfl_up_sync(0xFFFFFFFFu, sum, off);
    if (lane >= off) sum += o;
  }
  if (lane == 31) totals[warp] = sum;
  __syncthreads();
  unsigned long long before = sum - own[0] - own[1], all = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += totals[w];
    all += totals[w];
  }
  const int32_t n = (int32_t)(all >> 16 & 0xFFFFu);
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const uint32_t e = 2u * threadIdx.x + q;
    if (own[q] != 0) {
      const uint32_t a = (uint32_t)(before >> 16) & 0xFFFFu, first = (uint32_t)before & 0xFFFFu;
      base[e] = first;
      out.expert[a] = (int32_t)e;
      out.first[a] = (int32_t)first;
      out.turn[a] = (int32_t)(before >> 32);
      if (write) {
        p.list.expert[a] = (int32_t)e;
        p.list.first[a] = (int32_t)first;
      }
    }
    before += own[q];
  }
  if (threadIdx.x == 0) {
    *out.n = n;
    out.first[n] = (int32_t)(all & 0xFFFFu);
    out.turn[n] = (int32_t)(all >> 32);
    if (write) {
      *p.list.n = n;
      p.list.first[n] = (int32_t)(all & 0xFFFFu);
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < pairs; i += THREADS) {
    const int32_t e = slots[i];
    if (e < 0) continue;
    const uint32_t tok = i / p.topk, low = tokens[e], high = tokens[p.experts + e], bits = (1u << (tok & 31u)) - 1u;
    const uint32_t at = base[e] + (tok < 32u ? __popc(low & bits) : __popc(low) + __popc(high & bits));
    out.pairs[at] = (int32_t)i;
    if (write) {
      p.list.pairs[at] = (int32_t)i;
      p.list.token[at] = (int32_t)tok;
      p.list.gate[at] = p.gates[i] * (mx ? H_LIFT : 1.0f);  // written by this CTA, before a barrier
    }
  }
  __syncthreads();
}

// ------------------------------------------------------------------------------------------------------ 16-bit step
__device__ __forceinline__ void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// Lane (g, t)'s pieces are 8 consecutive elements of rows g and g + 8 in each 32-element chunk: the order of k inside an mma
// does not matter as long as both operands use the same one.  x: shared address of column 0 at the step's first element;
// columns behind `last` repeat it and are ignored by the caller.
__device__ __forceinline__ void multiply_wide(uint32_t slot, uint32_t x, uint32_t pitch, uint32_t last, int lane, float (&acc)[4]) {
  const uint32_t at = x + min((uint32_t)(lane >> 2), last) * pitch + (lane & 3) * 16u;
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t lo[4], hi[4], b[4];
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(lo[0]), "=r"(lo[1]), "=r"(lo[2]), "=r"(lo[3]) : "r"(slot + c * 512 + lane * 16));
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(hi[0]), "=r"(hi[1]), "=r"(hi[2]), "=r"(hi[3]) : "r"(slot + (2 + c) * 512 + lane * 16));
    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(b[0]), "=r"(b[1]), "=r"(b[2]), "=r"(b[3]) : "r"(at + 64u * c));
    mma_bf16(acc, lo[0], hi[0], lo[1], hi[1], b[0], b[1]);
    mma_bf16(acc, lo[2], hi[2], lo[3], hi[3], b[2], b[3]);
  }
}

// --------------------------------------------------------------------------------------------------------------- up
__device__ __forceinline__ void st_shared_v4(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

constexpr uint32_t UP_DEPTH = 4;   // slots of a ring
template <bool MX>
constexpr uint32_t UP_ROUND = MX ? 8 : 4;  // tiles of a warp between two barriers (16-bit weights: x takes the room)

// Shared memory: rings (before them, for a moment, the routing's scratch) | 16-bit weights: x of a pass, bf16 [tokens][pitch]
// | sums [2][round][warps along d][tokens][16] | lists
template <bool MX>
struct UpLayout {
  uint32_t x, sums, sums_half, lists, total;
  // long rows of 16-bit weights leave room for fewer tokens
  static __host__ __device__ uint32_t sums_of_tile(uint32_t per_pass) { return (MX ? (uint32_t)PASS : per_pass) * 16u; }
  __host__ __device__ UpLayout(const MoeParams &p) {
    using F = Format<MX>;
    const uint32_t steps = F::steps(p.d), pairs = p.m * p.topk;
    const uint32_t ring = WARPS * UP_DEPTH * F::SLOT, scratch = (32u + 3u * p.experts + pairs + (p.experts > 128u ? WARPS * p.experts : 0u)) * 4u;
    x = ((ring > scratch ? ring : scratch) + 15u) / 16u * 16u;
    sums = x + (MX ? 0u : p.per_pass * F::x_pitch(steps));
    sums_half = UP_ROUND<MX> * WARPS * sums_of_tile(p.per_pass);
    lists = sums + 2u * sums_half * 4u;
    total = lists + (1u + p.met + 2u * (p.met + 1u) + pairs) * 4u;
  }
};

// This CTA's run of tiles [u0, u1), tile = pass over an expert * tiles of an expert + tile.  It is taken in rounds that do not
// leave a pass, of UP_ROUND tiles of each group of warps; 4-bit weights: in a round a warp goes through its steps and for
// each through its tiles, so that its activations stay in registers; 16-bit weights: through its tiles and for each through
// its steps, so that the sums do.  The cursor names the warp's next item in that order, for the loads that run ahead.
template <bool MX>
struct Cursor {
  uint32_t r0, r1, step, v, v0;  // the round, the warp's next item, its first tile in the round
  __device__ __forceinline__ void round(const uint32_t start, uint32_t u0, uint32_t u1, uint32_t tiles, uint32_t TW, uint32_t tw, uint32_t kw) {
    r0 = start;
    r1 = min(min(u1, r0 + UP_ROUND<MX> * TW), (r0 / tiles + 1u) * tiles);
    v = v0 = r0 + ((tw - (r0 - u0)) & (TW - 1u));  // TW is a power of two
    step = kw;
  }
  __device__ __forceinline__ void next(uint32_t u0, uint32_t u1, uint32_t tiles, uint32_t steps, uint32_t KW, uint32_t TW, uint32_t kw, uint32_t tw) {
    if (MX) {
      v += TW;
      if (v < r1) return;
      v = v0;
      step += KW;
      if (step < steps) return;
    } else {
      step += KW;
      if (step < steps) return;
      step = kw;
      v += TW;
      if (v < r1) return;
    }
    do round(r1, u0, u1, tiles, TW, tw, kw);
    while (r0 < u1 && v >= r1);
  }
};

// The activations of a step as the columns of TG groups
template <int TG>
__device__ __forceinline__ void up_columns(const MoeParams &p, const int32_t *pairs, uint32_t cnt, uint32_t step, int lane, Columns (&x)[TG]) {
#pragma unroll
  for (int q = 0; q < TG; ++q) {
    const uint32_t j = 2u * q + (uint32_t)(lane >> 4);
    const uint16_t *row = p.x + (int64_t)((uint32_t)pairs[min(j, cnt - 1u)] / p.topk) * p.rsx;
    uint32_t w[2][4];
#pragma unroll
    for (int c = 0; c < 2; ++c) load_row8(w[c], row, step * STEP + 128u * c + 8u * (lane & 15), j < cnt ? p.d : 0u, p.x_vec);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float e[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) e[2 * i] = dec_bf16(w[c][i] & 0xFFFFu), e[2 * i + 1] = u2f(w[c][i] & 0xFFFF0000u);
      gather_chunk(x[q], c, e, lane);
    }
    limit_factors(x[q]);
  }
}

template <bool MX, int MODE>
__global__ void __launch_bounds__(THREADS, 1) up_kernel(const MoeParams p) {
  using F = Format<MX>;
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const UpLayout<MX> at(p);
  const uint32_t steps = F::steps(p.d), row_bytes = F::row_bytes(p.d), kblocks = (p.d + 31u) / 32u;
  const uint32_t tiles = MX ? (p.f + 31u) / 32u * 4u : (p.f + 7u) / 8u;  // 4-bit weights: whole blocks of 32 features
  const uint32_t x = smem_addr(smem) + at.x, x_pitch = F::x_pitch(steps), ring = smem_addr(smem) + warp * (UP_DEPTH * F::SLOT);
  float *sums = reinterpret_cast<float *>(smem + at.sums);
  Lists list;
  list.n = reinterpret_cast<int32_t *>(smem + at.lists);
  list.expert = list.n + 1;
  list.first = list.expert + p.met;
  list.turn = list.first + p.met + 1;
  list.pairs = list.turn + p.met + 1;

  route(p, reinterpret_cast<uint32_t *>(smem), list, MX, blockIdx.x == 0);
  const int32_t n = *list.n;
  constexpr uint32_t UNIT = MX ? 4 : 1;  // tiles that stay together
  const uint64_t total = (uint64_t)list.turn[n] * (tiles / UNIT);  // every pass over an expert counts
  const uint32_t u0 = (uint32_t)(total * blockIdx.x / gridDim.x) * UNIT, u1 = (uint32_t)(total * (blockIdx.x + 1) / gridDim.x) * UNIT;
  __syncthreads();  // the routing's scratch becomes the rings

  const uint32_t KW = p.k_warps, TW = WARPS / KW, kw = warp % KW, tw = warp / KW;
  TileRows rows;
  int32_t aim_a = 0;
  // a row that does not exist may lie outside the matrix, its pointer is never followed
  const uint64_t tile_by = (uint64_t)(8u * TW) * row_bytes, up_by = (uint64_t)p.f * row_bytes;
  const uint32_t srow = lane >> 1;
  uint32_t feature0 = 0;
  auto mark = [&]() {
    rows.has[0] = rows.has[1] = feature0 + g < p.f;
    if (MX) rows.has_scale = feature0 + (srow & 7u) < p.f;
  };
  auto aim = [&](uint32_t u) {
    const uint32_t turn = u / tiles;
    feature0 = (u - turn * tiles) * 8u;
    while ((int32_t)turn >= list.turn[aim_a + 1]) ++aim_a;
    const uint64_t base = (uint64_t)list.expert[aim_a] * 2u * p.f + feature0;
    rows.code[0] = p.w1 + (base + g) * row_bytes + 16 * t;
    rows.code[1] = rows.code[0] + up_by;
    if (MX) rows.scale = p.s1 + (base + (srow >= 8u ? p.f : 0u) + (srow & 7u)) * kblocks;
    mark();
  };
  Cursor<MX> ahead = {};
  uint32_t fill_at = 0;
  auto fill = [&]() {
    if (ahead.r0 < u1) {
      fill_slot<MX, MODE>(ring + fill_at * F::SLOT, rows, ahead.step, row_bytes, lane);
      const uint32_t v = ahead.v, r0 = ahead.r0;
      ahead.next(u0, u1, tiles, steps, KW, TW, kw, tw);
      if (ahead.v != v) {
        if (ahead.r0 == r0 && ahead.v > v) {  // the group's next tile of the same expert
          rows.code[0] += tile_by, rows.code[1] += tile_by, feature0 += 8u * TW;
          if (MX) rows.scale += (uint64_t)(8u * TW) * kblocks;
          mark();
        } else if (ahead.r0 < u1) {
          aim(ahead.v);
        }
      }
    }
    cp_commit();
    fill_at = fill_at + 1 == UP_DEPTH ? 0 : fill_at + 1;
  };
  ahead.round(u0, u0, u1, tiles, TW, tw, kw);
  while (ahead.r0 < u1 && ahead.v >= ahead.r1) ahead.round(ahead.r1, u0, u1, tiles, TW, tw, kw);
  if (ahead.r0 < u1) aim(ahead.v);
#pragma unroll
  for (uint32_t i = 0; i < UP_DEPTH - 1; ++i) fill();

  uint32_t slot = 0, half = 0;
  int32_t a = 0;
  uint32_t held = 0xFFFFFFFFu;  // the pass whose x is at hand
  Columns cols[2];
  for (uint32_t r0 = u0; r0 < u1;) {
    Cursor<MX> now;
    now.round(r0, u0, u1, tiles, TW, tw, kw);
    const uint32_t r1 = now.r1, turn = r0 / tiles;
    while ((int32_t)turn >= list.turn[a + 1]) ++a;
    const uint32_t pair0 = (uint32_t)list.first[a] + (turn - (uint32_t)list.turn[a]) * p.per_pass;
    const uint32_t cnt = min(p.per_pass, (uint32_t)list.first[a + 1] - pair0);
    float *round = sums + half * at.sums_half;
    const uint32_t tile_sums = UpLayout<MX>::sums_of_tile(p.per_pass);
    if (MX) {
      if (now.v < r1) {
        for (uint32_t step = kw; step < steps; step += KW) {
          // the activations of this step, unless they are the same as in the round before
          const bool fresh = held != turn || steps > KW;
          if (cnt <= 2) {
            Columns(&one)[1] = reinterpret_cast<Columns(&)[1]>(cols);
            if (fresh) up_columns<1>(p, list.pairs + pair0, cnt, step, lane, one);
            for (uint32_t v = now.v; v < r1; v += TW) {
              float y[1][2] = {{0.0f, 0.0f}};
              cp_wait<UP_DEPTH - 2>();
              __syncwarp();  // the slot's scales came through other lanes, and the slot filled next has been read by all
              fill();
              multiply_step<1>(ring + slot * F::SLOT, one, lane, y);
              slot = slot + 1 == UP_DEPTH ? 0 : slot + 1;
              keep_sums<1>(round + ((v - r0) * KW + kw) * (PASS * 16), one, y, step == kw, lane);
            }
          } else {
            if (fresh) up_columns<2>(p, list.pairs + pair0, cnt, step, lane, cols);
            for (uint32_t v = now.v; v < r1; v += TW) {
              float y[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
              cp_wait<UP_DEPTH - 2>();
              __syncwarp();
              fill();
              multiply_step<2>(ring + slot * F::SLOT, cols, lane, y);
              slot = slot + 1 == UP_DEPTH ? 0 : slot + 1;
              keep_sums<2>(round + ((v - r0) * KW + kw) * (PASS * 16), cols, y, step == kw, lane);
            }
          }
        }
        held = turn;
      }
    } else {
      if (held != turn) {  // x of the pass (the one before was last read before the barrier of its last round)
        const uint32_t groups = steps * (F::K / 8u), all = cnt * groups;
        for (uint32_t i = threadIdx.x; i < all; i += THREADS) {
          const uint32_t j = i / groups, gr = i - j * groups;
          uint32_t v[4];
          load_row8(v, p.x + (int64_t)((uint32_t)list.pairs[pair0 + j] / p.topk) * p.rsx, gr * 8u, p.d, p.x_vec);
          st_shared_v4(x + j * x_pitch + gr * 16u, v[0], v[1], v[2], v[3]);
        }
        held = turn;
        __syncthreads();
      }
      for (uint32_t v = now.v; v < r1; v += TW) {
        float *own = round + ((v - r0) * KW + kw) * tile_sums;
        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (uint32_t step = kw; step < steps; step += KW) {
          cp_wait<UP_DEPTH - 2>();
          __syncwarp();
          fill();
          multiply_wide(ring + slot * F::SLOT, x + step * (F::K * 2u), x_pitch, cnt - 1u, lane, acc);
          slot = slot + 1 == UP_DEPTH ? 0 : slot + 1;
        }
        if (t < 2) {  // columns 2 t and 2 t + 1 of the four tokens
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (2u * t + (q & 1) < cnt) own[(2 * t + (q & 1)) * 16 + g + 8 * (q >> 1)] = acc[q];
        }
      }
    }
    __syncthreads();
    // h = silu(gate) * up; the other half of the sums is written meanwhile
    const uint32_t feats = 8u * (r1 - r0);
    for (uint32_t i = threadIdx.x; i < feats * cnt; i += THREADS) {
      const uint32_t j = i / feats, c = i - j * feats;
      const uint32_t feature = (r0 - turn * tiles) * 8u + c, pair = (uint32_t)list.pairs[pair0 + j];
      const float *s = round + (c >> 3) * KW * tile_sums + j * 16 + (c & 7u);
      float gate = 0.0f, up = 0.0f;
      for (uint32_t q = 0; q < KW; ++q) {
        gate += s[q * tile_sums];
        up += s[q * tile_sums + 8];
      }
      float h = __fmul_rn(__fmul_rn(logistic_f32(1.0f, gate), gate), up);
      if (MX) {  // a warp has a block of 32 features (feats is a multiple of 32)
        if (feature >= p.f) h = 0.0f;
        const uint32_t top = __reduce_max_sync(0xFFFFFFFFu, f2u(h) & 0x7FFFFFFFu);
        float back;
        const float factor = block_factor(top, back);
        p.h16[(uint64_t)pair * h_pitch(p.f) + feature] = (uint16_t)(pack_f16x2_no_nan(h * factor, 0.0f) & 0xFFFFu);
        if (lane == 0) p.hf[(uint64_t)pair * (h_pitch(p.f) / 32u) + feature / 32u] = back * (1.0f / H_LIFT);
      } else if (feature < p.f) {
        p.h[(uint64_t)pair * p.f + feature] = h;
      }
    }
    half ^= 1u;
    r0 = r1;
  }
}

// ------------------------------------------------------------------------------------------------------------- down
// The warps' sums [warp][m][16], in order, into y
__device__ __forceinline__ void add_up(const MoeParams &p, const float *sums, uint32_t row0, uint32_t nrows) {
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < p.m * 16u; i += THREADS) {
    const uint32_t tok = i >> 4, r = i & 15u;
    float s = sums[i];
#pragma unroll
    for (int q = 1; q < WARPS; ++q) s += sums[(size_t)q * p.m * 16 + i];
    if (r < nrows) p.y[(int64_t)tok * p.rsy + row0 + r] = (uint16_t)enc_bf16(s);
  }
}

// 4-bit weights.  A slot of a ring holds an item: 16 rows x 256 elements of W2 and the h of up to PASS of the expert's pairs, fp16
// [4][256] and factors [4][8], all by cp.async, so that a warp does little more than multiply.  Shared memory: rings | per warp:
// sums [m][16]
constexpr uint32_t H_BYTES = PASS * 512 + PASS * 32, DOWN_SLOT = SLOT_BYTES + H_BYTES;

template <int MODE, int DEPTH>
__global__ void __launch_bounds__(THREADS, 1) down_mx_kernel(const MoeParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t row0 = blockIdx.x * p.down_rows, nrows = min(p.down_rows, p.d - row0);
  const uint32_t kblocks = (p.f + 31u) / 32u, row_bytes = kblocks * 16u, pitch = kblocks * 32u;
  const uint32_t ring = smem_addr(smem) + warp * (DEPTH * DOWN_SLOT);
  float *sums = reinterpret_cast<float *>(smem + WARPS * DEPTH * DOWN_SLOT), *own = sums + (size_t)warp * p.m * 16;
  for (uint32_t i = lane; i < p.m * 16u; i += 32u) own[i] = 0.0f;
  __syncwarp();
  dep_wait();

  const uint32_t parts = (p.f + STEP - 1u) / STEP, items = (uint32_t)*p.list.n * parts;
  // a row that does not exist may lie outside the matrix, its pointer is never followed
  TileRows rows;
  rows.has[0] = g < nrows, rows.has[1] = g + 8u < nrows, rows.has_scale = (uint32_t)(lane >> 1) < nrows;
  const uint64_t expert_by = (uint64_t)p.d * row_bytes, first_row = (uint64_t)(row0 + g) * row_bytes + 16 * t;
  const uint32_t by_a = WARPS / parts, by_part = WARPS % parts;  // an item ahead: WARPS parts further
  // h of the pairs `at` .. `last` - 1, at most PASS, elements 256 part ..
  auto load_h = [&](uint32_t slot, int32_t at, int32_t last, uint32_t part) {
    const uint32_t h = slot + SLOT_BYTES, col = part * STEP + lane * 8u;
#pragma unroll
    for (int j = 0; j < PASS; ++j)
      if (at + j < last) cp_async16(h + j * 512 + lane * 16, p.h16 + (uint64_t)p.list.pairs[at + j] * pitch + min(col, pitch - 8u), col < pitch ? 16u : 0u);
    const int32_t j = lane >> 3;  // the factors: 8 lanes to a pair
    const uint32_t blk = part * 8u + (lane & 7);
    if (at + j < last)
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(h + PASS * 512 + lane * 4),
                   "l"(p.hf + (uint64_t)p.list.pairs[at + j] * kblocks + min(blk, kblocks - 1u)), "r"(blk < kblocks ? 4u : 0u)
                   : "memory");
  };
  uint32_t fill_item = warp, fill_a = warp / parts, fill_part = warp % parts, fill_at = 0;
  auto fill = [&]() {
    if (fill_item < items) {
      const uint32_t slot = ring + fill_at * DOWN_SLOT;
      const uint64_t e = (uint64_t)p.list.expert[fill_a];
      rows.code[0] = p.w2 + e * expert_by + first_row;
      rows.code[1] = rows.code[0] + 8u * row_bytes;
      rows.scale = p.s2 + (e * p.d + row0 + (lane >> 1)) * kblocks;
      fill_slot<true, MODE>(slot, rows, fill_part, row_bytes, lane);
      load_h(slot, p.list.first[fill_a], p.list.first[fill_a + 1], fill_part);
      fill_item += WARPS, fill_a += by_a, fill_part += by_part;
      if (fill_part >= parts) fill_part -= parts, ++fill_a;
    }
    cp_commit();
    fill_at = fill_at + 1 == DEPTH ? 0 : fill_at + 1;
  };
#pragma unroll
  for (int i = 0; i < DEPTH - 1; ++i) fill();

  uint32_t a = warp / parts, part = warp % parts, at_slot = 0;
  for (uint32_t item = warp; item < items; item += WARPS) {
    const uint32_t slot = ring + at_slot * DOWN_SLOT, h = slot + SLOT_BYTES;
    const int32_t first = p.list.first[a], last = p.list.first[a + 1];
    cp_wait<DEPTH - 2>();
    __syncwarp();
    fill();
    for (int32_t at = first; at < last; at += PASS) {
      const uint32_t cnt = min((uint32_t)(last - at), (uint32_t)PASS);
      if (at != first) {  // more pairs than a slot holds: fetched when they are needed
        __syncwarp();
        load_h(slot, at, last, part);
        cp_commit();
        cp_wait<0>();
        __syncwarp();
      }
      // where this lane's sums go: tokens t / 2 and 2 + t / 2 of the pass
      const int32_t at0 = at + (int32_t)min((uint32_t)(t >> 1), cnt - 1u), at1 = at + (int32_t)min(2u + (uint32_t)(t >> 1), cnt - 1u);
      float *own0 = own + p.list.token[at0] * 16 + g, *own1 = own + p.list.token[at1] * 16 + g;
      const float gate0 = p.list.gate[at0], gate1 = p.list.gate[at1];
      // tokens 2 q and 2 q + 1 of the pass as the columns of a group
      auto columns = [&](Columns &c, int q) {
        const uint32_t j = 2u * q + (uint32_t)(g >> 2);
#pragma unroll
        for (int ch = 0; ch < 2; ++ch) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            uint32_t *w = c.v[ch] + 4 * i;
            w[0] = w[1] = w[2] = w[3] = 0u;
            if ((g & 3) == t && j < cnt)
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                           : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3])
                           : "r"(h + j * 512 + ch * 256u + t * 64u + 16u * i));
          }
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];"
                       : "=f"(c.factor[ch][0]), "=f"(c.factor[ch][1])
                       : "r"(h + PASS * 512 + min(2u * q + (uint32_t)(t >> 1), cnt - 1u) * 32u + ch * 16u + (uint32_t)(t & 1) * 8u));
        }
      };
      float y[2][2] = {{0.0f, 0.0f}, {0.0f, 0.0f}};
      if (cnt <= 2) {
        Columns x[1];
        float y1[1][2] = {{0.0f, 0.0f}};
        columns(x[0], 0);
        multiply_step<1>(slot, x, lane, y1);
        y[0][0] = y1[0][0], y[0][1] = y1[0][1];
      } else {
        Columns x[2];
        columns(x[0], 0);
        columns(x[1], 1);
        multiply_step<2>(slot, x, lane, y);
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        if (q == 1 && cnt <= 2) break;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const float s = y[q][i] + __shfl_xor_sync(0xFFFFFFFFu, y[q][i], 1);
          if ((t & 1) == 0 && 2u * q + (uint32_t)(t >> 1) < cnt) {
            float *o = (q ? own1 : own0) + 8 * i;
            *o = __fmaf_rn(q ? gate1 : gate0, s, *o);
          }
        }
      }
    }
    at_slot = at_slot + 1 == DEPTH ? 0 : at_slot + 1;
    a += by_a, part += by_part;
    if (part >= parts) part -= parts, ++a;
  }
  add_up(p, sums, row0, nrows);
}

// 16-bit weights.  An item is 16 rows x 128 elements of W2, two slots of a ring; h is fetched an item ahead into registers and
// split into two bf16 parts.  Shared memory: rings | per warp: h of an item, bf16, the first parts of four tokens, then the
// second parts, [8][128] with a pitch of 320 bytes | per warp: sums [m][16]
constexpr uint32_t WIDE_PITCH = 320, WIDE_STAGE = 2 * PASS * WIDE_PITCH;

template <int MODE, int DEPTH>
__global__ void __launch_bounds__(THREADS, 1) down_wide_kernel(const MoeParams p) {
  using F = Format<false>;
  constexpr uint32_t ITEM = 128, SLOTS = ITEM / F::K;
  constexpr int PER = ITEM / 32;  // elements of an item that a lane converts
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t row0 = blockIdx.x * p.down_rows, nrows = min(p.down_rows, p.d - row0), row_bytes = F::row_bytes(p.f);
  const uint32_t ring = smem_addr(smem) + warp * (DEPTH * F::SLOT);
  const uint32_t stage = smem_addr(smem) + WARPS * DEPTH * F::SLOT + warp * WIDE_STAGE;
  float *sums = reinterpret_cast<float *>(smem + WARPS * (DEPTH * F::SLOT + WIDE_STAGE)), *own = sums + (size_t)warp * p.m * 16;
  for (uint32_t i = lane; i < p.m * 16u; i += 32u) own[i] = 0.0f;
  __syncwarp();
  dep_wait();

  const uint32_t parts = (p.f + ITEM - 1u) / ITEM, items = (uint32_t)*p.list.n * parts;
  // a row that does not exist may lie outside the matrix, its pointer is never followed
  TileRows rows;
  rows.has[0] = g < nrows, rows.has[1] = g + 8u < nrows, rows.has_scale = false;
  rows.scale = nullptr;
  const uint64_t expert_by = (uint64_t)p.d * row_bytes, first_row = (uint64_t)(row0 + g) * row_bytes + 16 * t;
  auto aim = [&](uint32_t a) {
    rows.code[0] = p.w2 + (uint64_t)p.list.expert[a] * expert_by + first_row;
    rows.code[1] = rows.code[0] + 8u * row_bytes;
  };
  const uint32_t by_a = WARPS / parts, by_part = WARPS % parts;  // an item ahead: WARPS parts further
  uint32_t fill_item = warp, fill_a = warp / parts, fill_part = warp % parts, fill_sub = 0, fill_at = 0;
  auto fill = [&]() {
    if (fill_item < items) {
      fill_slot<false, MODE>(ring + fill_at * F::SLOT, rows, fill_part * SLOTS + fill_sub, row_bytes, lane);
      if (++fill_sub == SLOTS) {
        fill_sub = 0;
        fill_item += WARPS, fill_a += by_a, fill_part += by_part;
        if (fill_part >= parts) fill_part -= parts, ++fill_a;
        if (fill_item < items) aim(fill_a);
      }
    }
    cp_commit();
    fill_at = fill_at + 1 == DEPTH ? 0 : fill_at + 1;
  };
  // h of up to PASS pairs from `at` on: PER elements of each to a lane
  auto load_h = [&](float (&v)[PASS][PER], int32_t at, int32_t last, uint32_t k0) {
    const uint32_t col = k0 + lane * PER;
#pragma unroll
    for (int j = 0; j < PASS; ++j) {
#pragma unroll
      for (int q = 0; q < PER; ++q) v[j][q] = 0.0f;
      if (at + j < last) {
        const float *src = p.h + (uint64_t)p.list.pairs[at + j] * p.f + col;
        if (p.h_vec && col + PER <= p.f) {
          const float4 w = __ldcg(reinterpret_cast<const float4 *>(src));
          v[j][0] = w.x, v[j][1] = w.y, v[j][2] = w.z, v[j][3] = w.w;
        } else {
#pragma unroll
          for (int q = 0; q < PER; ++q)
            if (col + q < p.f) v[j][q] = __ldcg(src + q);
        }
      }
    }
  };
  auto store_h = [&](const float (&v)[PASS][PER], uint32_t cnt) {
#pragma unroll
    for (int j = 0; j < PASS; ++j) {
      if ((uint32_t)j >= cnt) break;
      uint32_t hi[2], lo[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float a = v[j][2 * q], b = v[j][2 * q + 1];
        hi[q] = pack_bf16x2_no_nan(a, b);
        const float a0 = u2f(hi[q] << 16), b0 = u2f(hi[q] & 0xFFFF0000u);
        // an infinity or NaN stays in the first part
        lo[q] = pack_bf16x2_no_nan(fabsf(a0) < INFINITY ? a - a0 : 0.0f, fabsf(b0) < INFINITY ? b - b0 : 0.0f);
      }
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(stage + j * WIDE_PITCH + lane * 8u), "r"(hi[0]), "r"(hi[1]) : "memory");
      asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(stage + (j + PASS) * WIDE_PITCH + lane * 8u), "r"(lo[0]), "r"(lo[1]) : "memory");
    }
  };
  if (fill_item < items) aim(fill_a);
#pragma unroll
  for (int i = 0; i < DEPTH - 1; ++i) fill();

  float v[PASS][PER];
  uint32_t a = warp / parts, part = warp % parts, slot = 0;
  int32_t first = 0, last = 0;
  if ((uint32_t)warp < items) {
    first = p.list.first[a], last = p.list.first[a + 1];
    load_h(v, first, last, part * ITEM);
  }
  for (uint32_t item = warp; item < items; item += WARPS) {
    uint32_t next_a = a + by_a, next_part = part + by_part;
    if (next_part >= parts) next_part -= parts, ++next_a;
    const bool more = item + WARPS < items;
    const int32_t next_first = more ? p.list.first[next_a] : 0, next_last = more ? p.list.first[next_a + 1] : 0;
    cp_wait<DEPTH - 1 - (int)SLOTS>();  // all slots of the item
    for (int32_t at = first; at < last; at += PASS) {
      const uint32_t cnt = min((uint32_t)(last - at), (uint32_t)PASS);
      if (at != first) load_h(v, at, last, part * ITEM);
      // where this lane's sums go: tokens 2 t and 2 t + 1 of the pass
      const uint32_t j0 = 2u * (t & 1);
      const int32_t at0 = at + (int32_t)min(j0, cnt - 1u), at1 = at + (int32_t)min(j0 + 1u, cnt - 1u);
      float *own0 = own + p.list.token[at0] * 16 + g, *own1 = own + p.list.token[at1] * 16 + g;
      const float gate0 = p.list.gate[at0], gate1 = p.list.gate[at1];
      __syncwarp();  // the h before has been read
      store_h(v, cnt);
      if (at + PASS >= last && more) load_h(v, next_first, next_last, next_part * ITEM);
      __syncwarp();
      float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (uint32_t s = 0; s < SLOTS; ++s) {
        const uint32_t i = slot + s >= DEPTH ? slot + s - DEPTH : slot + s;
        multiply_wide(ring + i * F::SLOT, stage + s * (F::K * 2u), WIDE_PITCH, 7u, lane, acc);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {  // columns 2 t, 2 t + 1: the first parts of the four tokens in lanes t = 0, 1, the second in 2, 3
        const float s = acc[q] + __shfl_xor_sync(0xFFFFFFFFu, acc[q], 2);
        if (t < 2 && j0 + (q & 1) < cnt) {
          float *o = (q & 1 ? own1 : own0) + 8 * (q >> 1);
          *o = __fmaf_rn(q & 1 ? gate1 : gate0, s, *o);
        }
      }
    }
    __syncwarp();  // every lane has read the item's slots
#pragma unroll
    for (uint32_t s = 0; s < SLOTS; ++s) fill();
    slot += SLOTS;
    if (slot >= DEPTH) slot -= DEPTH;
    a = next_a, part = next_part, first = next_first, last = next_last;
  }
  add_up(p, sums, row0, nrows);
}

template <auto KERNEL>
cudaError_t launch(unsigned grid, size_t smem, cudaStream_t s, const MoeParams &p) {
  static bool ready[64];  // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!__atomic_load_n(&ready[dev & 63], __ATOMIC_ACQUIRE)) {  // threads that meet here do the same
    e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MAX_SMEM);
    if (e != cudaSuccess) return e;
    __atomic_store_n(&ready[dev & 63], true, __ATOMIC_RELEASE);
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SKLB_COUNT_LAUNCH();
  return cudaLaunchKernelEx(&cfg, KERNEL, p);
}

template <bool MX, int MODE>
cudaError_t launch_moe(MoeParams &p, cudaStream_t s) {
  using F = Format<MX>;
  const uint32_t pairs = p.m * p.topk;
  p.met = pairs < p.experts ? pairs : p.experts;
  const uint32_t steps = F::steps(p.d);
  p.k_warps = 1;
  while (p.k_warps < (uint32_t)WARPS && p.k_warps * 2u <= steps) p.k_warps *= 2u;
  p.per_pass = p.m < PASS ? p.m : PASS;
  while (p.per_pass > 1 && UpLayout<MX>(p).total > MAX_SMEM) --p.per_pass;
  const UpLayout<MX> up(p);
  if (up.total > MAX_SMEM) return cudaErrorInvalidConfiguration;
  // an SM has room for one CTA; never more CTAs than tiles that can exist
  const uint64_t most = (uint64_t)p.met * ((p.m + p.per_pass - 1) / p.per_pass) * (MX ? (p.f + 31) / 32 : (p.f + 7) / 8);
  cudaError_t e = launch<up_kernel<MX, MODE>>((unsigned)(most < 148 ? most : 148), up.total, s, p);
  if (e != cudaSuccess) return e;
  const uint32_t rounds = (p.d + 148u * 16u - 1u) / (148u * 16u), ctas = 148u * rounds;
  p.down_rows = (p.d + ctas - 1u) / ctas;
  const unsigned grid = (p.d + p.down_rows - 1u) / p.down_rows;
  const size_t sums = (size_t)WARPS * p.m * 16 * 4;
  if constexpr (MX) {
    const size_t slot = (size_t)WARPS * DOWN_SLOT;
    if (3 * slot + sums <= MAX_SMEM) return launch<down_mx_kernel<MODE, 3>>(grid, 3 * slot + sums, s, p);
    return launch<down_mx_kernel<MODE, 2>>(grid, 2 * slot + sums, s, p);
  } else {
    // An item of `down` is two steps: rows of whole steps may still end in the middle of an item (f an odd multiple of 64), and
    // what lies behind a row is not the row's (nor, behind the last one, the caller's).
    constexpr int SAFE = MODE == WHOLE ? (int)ALIGNED : MODE;
    const size_t slot = (size_t)WARPS * F::SLOT, stage = (size_t)WARPS * WIDE_STAGE;
    const bool deep = 4 * slot + stage + sums <= MAX_SMEM, safe = p.f % 128u != 0;
    const size_t smem = (deep ? 4 : 3) * slot + stage + sums;
    if (safe) return deep ? launch<down_wide_kernel<SAFE, 4>>(grid, smem, s, p) : launch<down_wide_kernel<SAFE, 3>>(grid, smem, s, p);
    return deep ? launch<down_wide_kernel<MODE, 4>>(grid, smem, s, p) : launch<down_wide_kernel<MODE, 3>>(grid, smem, s, p);
  }
}

}  // namespace
}  // namespace sklb

using namespace sklb;

extern "C" int skl_b200_moe_supported(uint64_t m, uint64_t d, uint64_t f, uint64_t experts, uint64_t topk) {
  return m <= MAX_TOKENS && d <= 32768 && f <= 32768 && experts <= MAX_EXPERTS && topk <= MAX_TOPK;
}

// Up to 12 bytes that bring the workspace to a 16-byte boundary, h, either [pairs][f] fp32 or [pairs][f up to a multiple of 32] fp16 with a factor per block, then n, expert[], first[], pairs[],
// token[], gate[]; a multiple of 16 bytes up to the lists
static size_t h_bytes(uint64_t pairs, uint64_t f) {
  const size_t wide = (size_t)(pairs * f) * 4, blocks = (size_t)pairs * ((f + 31) / 32), packed = blocks * (32 * 2 + 4);
  return ((wide > packed ? wide : packed) + 15) / 16 * 16;
}
extern "C" size_t skl_b200_moe_scratch_bytes(uint64_t m, uint64_t f, uint64_t experts, uint64_t topk) {
  const size_t pairs = (size_t)(m * topk), met = pairs < experts ? pairs : (size_t)experts;
  return 12 + h_bytes(pairs, f) + (1 + met + met + 1 + 3 * pairs) * 4;
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
  uint8_t *work = (uint8_t *)((reinterpret_cast<uintptr_t>(q->workspace) + 15u) / 16u * 16u);
  p.h = (float *)work;
  p.h16 = (uint16_t *)work;
  p.hf = (float *)(p.h16 + pairs * h_pitch(p.f));
  p.h_vec = p.f % 4 == 0;
  p.list.n = (int32_t *)(work + h_bytes(pairs, p.f));
  p.list.expert = p.list.n + 1;
  p.list.first = p.list.expert + met;
  p.list.turn = nullptr;
  p.list.pairs = p.list.first + met + 1;
  p.list.token = p.list.pairs + pairs;
  p.list.gate = (float *)(p.list.token + pairs);
  cudaStream_t s = (cudaStream_t)stream;
  const uintptr_t bases = reinterpret_cast<uintptr_t>(p.w1) | reinterpret_cast<uintptr_t>(p.w2);
  const uint32_t row1 = q->mx ? Format<true>::row_bytes(p.d) : Format<false>::row_bytes(p.d);
  const uint32_t row2 = q->mx ? Format<true>::row_bytes(p.f) : Format<false>::row_bytes(p.f);
  const uintptr_t scales = q->mx ? reinterpret_cast<uintptr_t>(p.s1) | reinterpret_cast<uintptr_t>(p.s2) : 0;
  const int mode = (bases & 15u) || ((row1 | row2) & 15u) ? BYTES : ((row1 | row2) % 128 == 0 && (scales & 7u) == 0 ? WHOLE : ALIGNED);
  if (q->mx) {
    if (mode == WHOLE) return (int)launch_moe<true, WHOLE>(p, s);
    return (int)(mode == ALIGNED ? launch_moe<true, ALIGNED>(p, s) : launch_moe<true, BYTES>(p, s));
  }
  if (mode == WHOLE) return (int)launch_moe<false, WHOLE>(p, s);
  return (int)(mode == ALIGNED ? launch_moe<false, ALIGNED>(p, s) : launch_moe<false, BYTES>(p, s));
}
