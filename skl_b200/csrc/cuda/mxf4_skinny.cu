// mxf4_skinny.cu -- C = alpha * A W^T + beta * C for few rows of A (bf16 / fp16) and MX-FP4 weights W [n][k]: the decode case.
//
// Bound by HBM: the weights are read once, 17/32 byte per element.  One CTA of 16 warps per SM owns an equal run of weight
// rows (tiles of 16, the last one short, so that all SMs read the same amount); its warps split k, then tiles, and stream
// their steps of 16 rows x 256 elements through rings in shared memory (mxf4_mma.cuh).  The partial sums of the warps meet
// in shared memory once, at the end, and are added in a fixed order, so results do not change from run to run.
#include "mxf4_mma.cuh"

namespace sklb {
namespace {

using namespace mxmma;

constexpr int WARPS = 16;

struct SkinnyParams {
  const uint8_t *b, *sb;
  const void *a;
  void *c;
  int64_t csb, cssb, rsa, rsc;
  uint32_t m, n, k, kblocks, steps;
  uint32_t cta_rows, k_warps;  // rows of a CTA; warps that split k (a power of two)
  float alpha, beta;
  int ta, tc, a_vec;
  int static_b;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Elements [first, first + count) of the activation rows into shared memory as fp16 with their blocks' factors; elements
// behind k are zeros.  Four lanes share a block of 32.
template <bool BF16>
__device__ __forceinline__ void stage_rows(const SkinnyParams &p, uint32_t tokens, uint32_t first, uint32_t count, uint32_t x,
                                           uint32_t x_pitch, uint32_t f, uint32_t f_pitch) {
  const uint32_t groups = count / 8u, total = tokens * groups;
  for (uint32_t i0 = 0; i0 < total; i0 += blockDim.x) {  // whole warps stay together for the shuffles
    const uint32_t i = i0 + threadIdx.x;
    const bool in = i < total;
    const uint32_t tok = in ? i / groups : 0u, gr = in ? i - tok * groups : 0u, kk = first + gr * 8u;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (in && tok < p.m && kk < p.k) {
      const uint16_t *src = (const uint16_t *)p.a + (int64_t)tok * p.rsa + kk;
      if (p.a_vec && kk + 8u <= p.k) {
        const uint4 v = ld_v4(src);
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (kk + e < p.k) w[e >> 1] |= ld_u16(src + e) << (16 * (e & 1));
      }
    }
    if (BF16) {
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) top = max(top, max(w[e] << 16 & 0x7FFFFFFFu, w[e] & 0x7FFF0000u));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
      top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
      float back;
      const float factor = block_factor(top, back);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        w[e] = pack_f16x2_no_nan(dec_bf16(w[e] & 0xFFFFu) * factor, u2f(w[e] & 0xFFFF0000u) * factor);
      if (in && (gr & 3u) == 0u) asm volatile("st.shared.f32 [%0], %1;" ::"r"(f + tok * f_pitch + (gr >> 2) * 4u), "f"(back) : "memory");
    }
    if (in)
      asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(x + tok * x_pitch + gr * 16u), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                   "r"(w[3])
                   : "memory");
  }
}

// Shared memory: 64 bytes of zeros | activations fp16 [m][steps * 256] | factors [m][steps * 8] | rings [16][DEPTH] |
// partial sums [tile][warps along k][2 TG][16]
template <int TG, bool BF16, bool VEC, bool SVEC, int DEPTH>
__global__ void __launch_bounds__(32 * WARPS, 1) skinny_kernel(const SkinnyParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t row0 = blockIdx.x * p.cta_rows, rows = min(p.cta_rows, p.n - row0), tiles = (rows + 15u) / 16u;
  const uint32_t x_pitch = p.steps * (STEP * 2), f_pitch = p.steps * (STEP / 8);
  const uint32_t zeros = smem_addr(smem), x = zeros + 64u, f = x + p.m * x_pitch;
  const uint32_t rings = f + (BF16 ? p.m * f_pitch : 0u), ring = rings + warp * (DEPTH * SLOT_BYTES);
  float *part = reinterpret_cast<float *>(smem + (rings - zeros) + WARPS * DEPTH * SLOT_BYTES);

  // this warp's items: steps kw, kw + KW, ... of tiles tw, tw + TW, ...
  const uint32_t KW = p.k_warps, TW = WARPS / KW, kw = warp % KW, tw = warp / KW;
  TileRows at;
  auto aim = [&](uint32_t tile) {
    const uint32_t r = tile * 16u;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t i = r + g + 8u * h;
      at.code[h] = i < rows ? p.b + (int64_t)(row0 + i) * p.csb : nullptr;
    }
    const uint32_t i = r + (lane >> 1);
    at.scale = i < rows ? p.sb + (int64_t)(row0 + i) * p.cssb : nullptr;
  };
  uint32_t fill_tile = tw, fill_step = kw, fill_at = 0;  // the next item to load and its slot
  auto fill = [&]() {
    if (fill_tile < tiles) {
      fill_slot<true, VEC, SVEC>(ring + fill_at * SLOT_BYTES, at, fill_step, p.kblocks * 16u, lane);
      fill_step += KW;
      if (fill_step >= p.steps) {
        fill_step = kw;
        fill_tile += TW;
        if (fill_tile < tiles) aim(fill_tile);
      }
    }
    cp_commit();
    fill_at = fill_at + 1 == DEPTH ? 0 : fill_at + 1;
  };
  if (fill_tile < tiles) aim(fill_tile);
  if (!p.static_b) dep_wait();
#pragma unroll
  for (int i = 0; i < DEPTH - 1; ++i) fill();
  if (p.static_b) dep_wait();
  if (threadIdx.x < 16) reinterpret_cast<uint32_t *>(smem)[threadIdx.x] = 0u;
  stage_rows<BF16>(p, p.m, 0, p.steps * STEP, x, x_pitch, f, f_pitch);
  __syncthreads();

  uint32_t slot = 0;
  for (uint32_t tile = tw; tile < tiles; tile += TW) {
    float y[TG][2];
#pragma unroll
    for (int q = 0; q < TG; ++q) y[q][0] = y[q][1] = 0.0f;
    for (uint32_t step = kw; step < p.steps; step += KW) {
      cp_wait<DEPTH - 2>();
      __syncwarp();  // the slot's scales came through other lanes, and the slot filled next has been read by all
      fill();
      multiply_step<TG, BF16>(ring + slot * SLOT_BYTES, x + step * (STEP * 2), x_pitch, f + step * (STEP / 8), f_pitch, p.m - 1u,
                              zeros, lane, y);
      slot = slot + 1 == DEPTH ? 0 : slot + 1;
    }
#pragma unroll
    for (int q = 0; q < TG; ++q) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        y[q][h] += __shfl_xor_sync(0xFFFFFFFFu, y[q][h], 1);
        if ((t & 1) == 0) part[((tile * KW + kw) * 2 * TG + 2 * q + (t >> 1)) * 16 + g + 8 * h] = y[q][h];
      }
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < rows * p.m; i += 32u * WARPS) {
    const uint32_t tok = i / rows, r = i - tok * rows;
    const float *s = part + ((r >> 4) * KW * 2 * TG + tok) * 16 + (r & 15u);
    float v = 0.0f;
    for (uint32_t q = 0; q < KW; ++q) v += s[q * 2 * TG * 16];
    const int64_t o = (int64_t)tok * p.rsc + row0 + r;
    v = __fmul_rn(p.alpha, v);
    if (p.beta != 0.0f) v = __fadd_rn(__fmul_rn(p.beta, load_c_f32(p.tc, p.c, o)), v);
    store_c_f32(p.tc, p.c, o, v);
  }
}

constexpr size_t MAX_SMEM = 226 * 1024;
constexpr uint32_t MAX_ROWS = 128;  // of a CTA: bounds its partial sums; longer matrices take several rounds of CTAs

struct Shape {
  uint32_t steps, cta_rows, k_warps;
  size_t fixed;  // shared memory without the rings
};
Shape shape_of(uint32_t m, uint32_t n, uint32_t k, int tg, bool factors) {
  Shape s;
  s.steps = (k + STEP - 1) / STEP;
  const uint32_t rounds = (n + 148u * MAX_ROWS - 1u) / (148u * MAX_ROWS), ctas = 148u * rounds;
  s.cta_rows = (n + ctas - 1u) / ctas;
  s.k_warps = 1;
  while (s.k_warps < (uint32_t)WARPS && s.k_warps * 2u <= s.steps) s.k_warps *= 2u;
  s.fixed = 64 + (size_t)m * s.steps * (STEP * 2 + (factors ? STEP / 8 : 0)) +
            (size_t)((s.cta_rows + 15u) / 16u) * s.k_warps * 2 * tg * 16 * 4;
  return s;
}

template <int TG, bool BF16, bool VEC, bool SVEC, int DEPTH>
cudaError_t launch_depth(const SkinnyParams &p, size_t smem, cudaStream_t s) {
  auto kernel = skinny_kernel<TG, BF16, VEC, SVEC, DEPTH>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MAX_SMEM);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((p.n + p.cta_rows - 1u) / p.cta_rows);
  cfg.blockDim = dim3(32u * WARPS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SKLB_COUNT_LAUNCH();
  return cudaLaunchKernelEx(&cfg, kernel, (const SkinnyParams)p);
}

template <int TG, bool BF16, bool VEC, bool SVEC>
cudaError_t launch_skinny(SkinnyParams &p, cudaStream_t s) {
  const Shape h = shape_of(p.m, p.n, p.k, TG, BF16);
  p.steps = h.steps, p.cta_rows = h.cta_rows, p.k_warps = h.k_warps;
  // four slots to a ring (100 KB in flight on an SM) where the activations leave room, else two
  const size_t slot = (size_t)WARPS * SLOT_BYTES;
  if (h.fixed + 4 * slot <= MAX_SMEM) return launch_depth<TG, BF16, VEC, SVEC, 4>(p, h.fixed + 4 * slot, s);
  if (h.fixed + 2 * slot <= MAX_SMEM) return launch_depth<TG, BF16, VEC, SVEC, 2>(p, h.fixed + 2 * slot, s);
  return cudaErrorInvalidConfiguration;
}

template <int TG, bool BF16>
cudaError_t dispatch(SkinnyParams &p, bool vec, bool svec, cudaStream_t s) {
  if (vec && svec) return launch_skinny<TG, BF16, true, true>(p, s);
  return vec ? launch_skinny<TG, BF16, true, false>(p, s) : launch_skinny<TG, BF16, false, false>(p, s);
}

int group_count(uint32_t m) { return m <= 2 ? 1 : (m <= 4 ? 2 : 4); }

}  // namespace
}  // namespace sklb

using namespace sklb;

// up to 8 rows whose activations fit into shared memory beside two slots per warp
extern "C" int skl_b200_mxf4_skinny_supported(uint64_t m, uint64_t n, uint64_t k, int ta) {
  if (m < 1 || m > 8 || n < 1 || k < 1 || n >= (1ull << 31) || k >= (1ull << 22)) return 0;
  const Shape h = shape_of((uint32_t)m, (uint32_t)n, (uint32_t)k, group_count((uint32_t)m), ta == SKL_DT_BF16);
  return h.fixed + 2 * (size_t)WARPS * SLOT_BYTES <= MAX_SMEM;
}

extern "C" int skl_b200_launch_mxf4_skinny(uint32_t m, uint32_t n, uint32_t k, float alpha, const void *a, int ta, int64_t rsa,
                                           const void *b, int64_t csb, const void *sb, int64_t cssb, float beta, void *c,
                                           int tc, int64_t rsc, int static_b, void *stream) {
  SkinnyParams p;
  p.a = a, p.b = (const uint8_t *)b, p.sb = (const uint8_t *)sb, p.c = c;
  p.rsa = rsa, p.csb = csb, p.cssb = cssb, p.rsc = rsc;
  p.m = m, p.n = n, p.k = k, p.kblocks = (k + 31) / 32;
  p.alpha = alpha, p.beta = beta, p.ta = ta, p.tc = tc, p.static_b = static_b;
  p.a_vec = (reinterpret_cast<uintptr_t>(a) & 15u) == 0 && (m == 1 || rsa % 8 == 0);
  const bool vec = (reinterpret_cast<uintptr_t>(b) & 15u) == 0 && (n == 1 || csb % 16 == 0);
  const bool svec = (reinterpret_cast<uintptr_t>(sb) & 7u) == 0 && (n == 1 || cssb % 8 == 0);
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf = ta == SKL_DT_BF16;
  switch (group_count(m)) {
    case 1: return (int)(bf ? dispatch<1, true>(p, vec, svec, s) : dispatch<1, false>(p, vec, svec, s));
    case 2: return (int)(bf ? dispatch<2, true>(p, vec, svec, s) : dispatch<2, false>(p, vec, svec, s));
    default: return (int)(bf ? dispatch<4, true>(p, vec, svec, s) : dispatch<4, false>(p, vec, svec, s));
  }
}
