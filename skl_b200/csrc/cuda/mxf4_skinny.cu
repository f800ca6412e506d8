// mxf4_skinny.cu -- C = alpha * A W^T + beta * C for few rows of A (bf16 / fp16) and MX-FP4 weights W [n][k]: the decode case.
//
// Bound by HBM: the weights are read once, 17/32 byte per element.  A tile of 16 weight rows belongs to one CTA, or to a
// cluster of CTAs where n is small; its warps take the steps of 256 elements of k in turn (mxf4_mma.cuh), keeping one step's
// loads in flight while they multiply the one before.  The partial sums of the warps, then of the cluster's CTAs (through
// distributed shared memory), are added in a fixed order, so results do not change from run to run.
#include "mxf4_mma.cuh"

namespace sklb {
namespace {

using namespace mxmma;

struct SkinnyParams {
  const uint8_t *b, *sb;
  const void *a;
  void *c;
  int64_t csb, cssb, rsa, rsc;
  uint32_t m, n, k, kblocks, steps, cta_steps;  // cta_steps: steps of one CTA of the cluster
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

template <int TG, bool BF16, bool VEC>
__global__ void __launch_bounds__(512) skinny_kernel(const SkinnyParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warps = blockDim.x >> 5;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const uint32_t row0 = (blockIdx.x / ranks) * 16u;
  const uint32_t first_step = rank * p.cta_steps;
  const uint32_t last_step = min(first_step + p.cta_steps, p.steps);

  // layout: 64 bytes of zeros | activations fp16 [2 TG][cta_steps * 256] | factors [2 TG][cta_steps * 8] | sums
  const uint32_t x_pitch = p.cta_steps * (STEP * 2), f_pitch = p.cta_steps * (STEP / 8);
  const uint32_t zeros = smem_addr(smem), x = zeros + 64u, f = x + 2 * TG * x_pitch;
  float *sums = reinterpret_cast<float *>(smem + 64 + 2 * TG * (x_pitch + (BF16 ? f_pitch : 0u)));  // [warp][2 TG][16]

  RowPair rows;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t r = min(row0 + g + 8u * h, p.n - 1u);  // rows behind the last are read again and not stored
    rows.code[h] = p.b + (int64_t)r * p.csb;
    rows.scale[h] = p.sb + (int64_t)r * p.cssb;
  }
  Weights w;
  uint32_t step = first_step + warp;
  if (p.static_b && step < last_step) load_step<VEC>(w, rows, step, p.kblocks, t);
  dep_wait();
  if (!p.static_b && step < last_step) load_step<VEC>(w, rows, step, p.kblocks, t);
  if (threadIdx.x < 16) reinterpret_cast<uint32_t *>(smem)[threadIdx.x] = 0u;
  stage_rows<BF16>(p, 2 * TG, first_step * STEP, p.cta_steps * STEP, x, x_pitch, f, f_pitch);
  __syncthreads();

  float y[TG][2];
#pragma unroll
  for (int q = 0; q < TG; ++q) y[q][0] = y[q][1] = 0.0f;
  while (step < last_step) {
    const uint32_t next = step + warps;
    Weights wn;
    if (next < last_step) load_step<VEC>(wn, rows, next, p.kblocks, t);
    const uint32_t s = step - first_step;
    multiply_step<TG, BF16>(w, x + s * (STEP * 2), x_pitch, f + s * (STEP / 8), f_pitch, 2 * TG - 1, zeros,
                                   g, t, y);
    w = wn;
    step = next;
  }
#pragma unroll
  for (int q = 0; q < TG; ++q) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      y[q][h] += __shfl_xor_sync(0xFFFFFFFFu, y[q][h], 1);
      if ((t & 1) == 0) sums[(warp * 2 * TG + 2 * q + (t >> 1)) * 16 + g + 8 * h] = y[q][h];
    }
  }
  __syncthreads();
  const int out = (int)threadIdx.x;  // one (token, row) per thread
  float v = 0.0f;
  const bool mine = out < 32 * TG;
  if (mine)
    for (int i = 0; i < warps; ++i) v += sums[i * 32 * TG + out];
  if (ranks > 1) {
    // the CTA's sum goes to the front of its own sums, rank 0 collects
    __syncthreads();
    if (mine) sums[out] = v;
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && mine) {
      const uint32_t at = smem_addr(sums + out);
      v = 0.0f;
      for (uint32_t r = 0; r < ranks; ++r) {
        uint32_t remote;
        float part;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(r));
        asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(part) : "r"(remote) : "memory");
        v += part;
      }
    }
    // no CTA leaves while its shared memory may still be read
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank != 0) return;
  }
  const uint32_t tok = (uint32_t)out >> 4, row = row0 + (out & 15);
  if (mine && tok < p.m && row < p.n) {
    const int64_t at = (int64_t)tok * p.rsc + row;
    v = __fmul_rn(p.alpha, v);
    if (p.beta != 0.0f) v = __fadd_rn(__fmul_rn(p.beta, load_c_f32(p.tc, p.c, at)), v);
    store_c_f32(p.tc, p.c, at, v);
  }
}

constexpr int MAX_SMEM = 200 * 1024;

template <int TG, bool BF16, bool VEC>
cudaError_t launch_skinny(SkinnyParams &p, cudaStream_t s) {
  // Warps for one tile of 16 rows: enough that the whole chip holds about 24 per SM, at most one per step.  Up to 8 (16 for
  // small grids) of them make a CTA, the rest become further CTAs of a cluster, which also shortens the run of activations
  // that a CTA has to stage.
  const uint32_t tiles = (p.n + 15u) / 16u;
  uint32_t want = (148u * 24u + tiles - 1u) / tiles;
  if (want > p.steps) want = p.steps;
  uint32_t ranks = 1;
  const uint32_t per_cta = tiles >= 148u ? 16u : 8u;
  while (ranks < 8u && want > ranks * per_cta) ranks *= 2u;
  auto bytes = [&](uint32_t r, uint32_t warps) {
    const uint64_t st = (p.steps + r - 1u) / r;
    return 64 + (uint64_t)2 * TG * st * (STEP * 2 + (BF16 ? STEP / 8 : 0)) + (uint64_t)warps * 2 * TG * 16 * 4;
  };
  while (ranks < 8u && bytes(ranks, 16) > 64 * 1024) ranks *= 2u;
  p.cta_steps = (p.steps + ranks - 1u) / ranks;
  uint32_t warps = (want + ranks - 1u) / ranks;
  if (warps > 16u) warps = 16u;
  if (warps > p.cta_steps) warps = p.cta_steps;
  if (warps < TG) warps = TG;  // a thread per (token, row) of the tile
  const uint64_t smem = bytes(ranks, warps);
  if (smem > MAX_SMEM) return cudaErrorInvalidConfiguration;
  auto kernel = skinny_kernel<TG, BF16, VEC>;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  cfg.gridDim = dim3(tiles * ranks);
  cfg.blockDim = dim3(32u * warps);
  cfg.dynamicSmemBytes = (size_t)smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  SKLB_COUNT_LAUNCH();
  return cudaLaunchKernelEx(&cfg, kernel, (const SkinnyParams)p);
}

template <int TG>
cudaError_t dispatch(SkinnyParams &p, bool vec, cudaStream_t s) {
  if (p.ta == SKL_DT_BF16) return vec ? launch_skinny<TG, true, true>(p, s) : launch_skinny<TG, true, false>(p, s);
  return vec ? launch_skinny<TG, false, true>(p, s) : launch_skinny<TG, false, false>(p, s);
}

int group_count(uint32_t m) { return m <= 2 ? 1 : (m <= 4 ? 2 : (m <= 8 ? 4 : 8)); }

}  // namespace
}  // namespace sklb

using namespace sklb;

// m <= 16, and the activations of an eighth of k fit into shared memory
extern "C" int skl_b200_mxf4_skinny_supported(uint64_t m, uint64_t n, uint64_t k) {
  if (m < 1 || m > 16 || n < 1 || k < 1 || n >= (1ull << 31) || k >= (1ull << 31)) return 0;
  const uint64_t steps = (k + STEP - 1) / STEP, per = (steps + 7) / 8, tg = (uint64_t)group_count((uint32_t)m);
  return n <= (1ull << 30) && 64 + 2 * tg * per * (STEP * 2 + STEP / 8) + 16 * 2 * tg * 64 <= (uint64_t)MAX_SMEM;
}

extern "C" int skl_b200_launch_mxf4_skinny(uint32_t m, uint32_t n, uint32_t k, float alpha, const void *a, int ta, int64_t rsa,
                                           const void *b, int64_t csb, const void *sb, int64_t cssb, float beta, void *c,
                                           int tc, int64_t rsc, int static_b, void *stream) {
  SkinnyParams p;
  p.a = a, p.b = (const uint8_t *)b, p.sb = (const uint8_t *)sb, p.c = c;
  p.rsa = rsa, p.csb = csb, p.cssb = cssb, p.rsc = rsc;
  p.m = m, p.n = n, p.k = k, p.kblocks = (k + 31) / 32, p.steps = (k + STEP - 1) / STEP;
  p.alpha = alpha, p.beta = beta, p.ta = ta, p.tc = tc, p.static_b = static_b;
  p.a_vec = (reinterpret_cast<uintptr_t>(a) & 15u) == 0 && (m == 1 || rsa % 8 == 0);
  const bool vec = (reinterpret_cast<uintptr_t>(b) & 15u) == 0 && (reinterpret_cast<uintptr_t>(sb) & 7u) == 0 &&
                   (n == 1 || (csb % 16 == 0 && cssb % 8 == 0));
  cudaStream_t s = (cudaStream_t)stream;
  switch (group_count(m)) {
    case 1: return (int)dispatch<1>(p, vec, s);
    case 2: return (int)dispatch<2>(p, vec, s);
    case 4: return (int)dispatch<4>(p, vec, s);
    default: return (int)dispatch<8>(p, vec, s);
  }
}
