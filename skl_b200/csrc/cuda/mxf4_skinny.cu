// mxf4_skinny.cu -- C = alpha * A W^T + beta * C for few rows of A (bf16 / fp16) and MX-FP4 weights W [n][k]: the decode case.
//
// Bound by HBM: the weights are read once, 17/32 byte per element.  One CTA of 16 warps per SM owns an equal run of weight
// rows (tiles of 16, the last one short, so that all SMs read the same amount); its warps split k, then tiles, and stream
// their steps of 16 rows x 256 elements through rings in shared memory (mxf4_mma.cuh).  The partial sums of the warps meet
// in shared memory once, at the end, and are added in a fixed order, so results do not change from run to run.
//
// 14336 x 4096, in a graph: 1 or 2 rows 8.9 us, 3 or 4 rows 11.7 (31 MB: 4.9 us of HBM; about 2 us pass until the first weights
// arrive, the rest is the stream and the join); 4096 x 14336 (fp16) 11.2 and 15.4; 4096 x 4096 4.5 and 6.0; 1024 x 1024 2.7 and 3.2.
// Plain loads into registers instead of the rings: 18.0 us for the first.
#include "mxf4_mma.cuh"

namespace sklb {
namespace {

using namespace mxmma;

constexpr int WARPS = 16, DEPTH = 4;  // four slots to a ring: up to 100 KB in flight on an SM
constexpr int MAX_SMEM = WARPS * DEPTH * SLOT_BYTES + 8 * WARPS * 4 * 16 * 4;  // eight tiles, four tokens

struct SkinnyParams {
  const uint8_t *b, *sb;
  const void *a;
  void *c;
  int64_t csb, cssb, rsa, rsc;
  uint32_t m, n, k, kblocks, steps;
  uint32_t cta_rows, k_warps;  // rows of a CTA; warps that split k (a power of two)
  float alpha, beta;
  int tc, a_vec;
  int static_b;
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// Shared memory: rings [16][DEPTH] | sums [tile][warps along k][2 TG][16]
template <int TG, bool BF16, int MODE>
__global__ void __launch_bounds__(32 * WARPS, 1) skinny_kernel(const SkinnyParams p) {
  extern __shared__ __align__(16) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t row0 = blockIdx.x * p.cta_rows, rows = min(p.cta_rows, p.n - row0), tiles = (rows + 15u) / 16u;
  const uint32_t ring = smem_addr(smem) + warp * (DEPTH * SLOT_BYTES);
  float *sums = reinterpret_cast<float *>(smem + WARPS * DEPTH * SLOT_BYTES);

  // this warp's items: for each of the steps kw, kw + KW, ... the tiles tw, tw + TW, ...
  const uint32_t KW = p.k_warps, TW = WARPS / KW, kw = warp % KW, tw = warp / KW;
  TileRows at;
  const int64_t code_by = p.csb * (16 * TW), scale_by = p.cssb * (16 * TW);
  uint32_t fill_tile = tw, fill_step = tw < tiles ? kw : p.steps, fill_at = 0;  // the next item to load and its slot
  auto mark = [&]() {
    const uint32_t r = fill_tile * 16u;
    at.has[0] = r + g < rows, at.has[1] = r + g + 8u < rows, at.has_scale = r + (lane >> 1) < rows;
  };
  auto aim = [&]() {  // at the first tile; a row that does not exist may lie outside the matrix, its pointer is never followed
    at.code[0] = p.b + (int64_t)(row0 + tw * 16u + g) * p.csb + 16 * t;
    at.code[1] = at.code[0] + 8 * p.csb;
    at.scale = p.sb + (int64_t)(row0 + tw * 16u + (lane >> 1)) * p.cssb;
    mark();
  };
  auto fill = [&]() {
    if (fill_step < p.steps) {
      fill_slot<true, MODE>(ring + fill_at * SLOT_BYTES, at, fill_step, p.kblocks * 16u, lane);
      fill_tile += TW;
      if (fill_tile >= tiles) {
        fill_tile = tw;
        fill_step += KW;
        aim();
      } else {
        at.code[0] += code_by, at.code[1] += code_by, at.scale += scale_by;
        mark();
      }
    }
    cp_commit();
    fill_at = fill_at + 1 == DEPTH ? 0 : fill_at + 1;
  };
  aim();
  if (!p.static_b) dep_wait();
#pragma unroll
  for (int i = 0; i < DEPTH - 1; ++i) fill();
  if (p.static_b) dep_wait();

  uint32_t slot = 0;
  for (uint32_t step = kw; step < p.steps && tw < tiles; step += KW) {
    Columns x[TG];
    uint32_t w[TG][2][4];
#pragma unroll
    for (int q = 0; q < TG; ++q) {
      const uint32_t tok = 2u * q + (uint32_t)(lane >> 4);
#pragma unroll
      for (int c = 0; c < 2; ++c)
        load_row8(w[q][c], (const uint16_t *)p.a + (int64_t)min(tok, p.m - 1u) * p.rsa, step * STEP + 128u * c + 8u * (lane & 15),
                  tok < p.m ? p.k : 0u, p.a_vec);
    }
#pragma unroll
    for (int q = 0; q < TG; ++q) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float e[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          e[2 * i] = BF16 ? dec_bf16(w[q][c][i] & 0xFFFFu) : dec_f16(w[q][c][i] & 0xFFFFu);
          e[2 * i + 1] = BF16 ? u2f(w[q][c][i] & 0xFFFF0000u) : dec_f16(w[q][c][i] >> 16);
        }
        gather_chunk(x[q], c, e, lane);
      }
      limit_factors(x[q]);
    }
    for (uint32_t tile = tw; tile < tiles; tile += TW) {
      float y[TG][2];
#pragma unroll
      for (int q = 0; q < TG; ++q) y[q][0] = y[q][1] = 0.0f;
      cp_wait<DEPTH - 2>();
      __syncwarp();  // the slot's scales came through other lanes, and the slot filled next has been read by all
      fill();
      multiply_step<TG>(ring + slot * SLOT_BYTES, x, lane, y);
      slot = slot + 1 == DEPTH ? 0 : slot + 1;
      keep_sums<TG>(sums + (tile * KW + kw) * (2 * TG * 16), x, y, step == kw, lane);
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < rows * p.m; i += 32u * WARPS) {
    const uint32_t tok = i / rows, r = i - tok * rows;
    const float *s = sums + ((r >> 4) * KW * 2 * TG + tok) * 16 + (r & 15u);
    float v = 0.0f;
    for (uint32_t q = 0; q < KW; ++q) v += s[q * 2 * TG * 16];
    const int64_t o = (int64_t)tok * p.rsc + row0 + r;
    v = __fmul_rn(p.alpha, v);
    if (p.beta != 0.0f) v = __fadd_rn(__fmul_rn(p.beta, load_c_f32(p.tc, p.c, o)), v);
    store_c_f32(p.tc, p.c, o, v);
  }
}

constexpr uint32_t MAX_ROWS = 128;  // of a CTA: bounds its sums; longer matrices take several rounds of CTAs

template <int TG, bool BF16, int MODE>
cudaError_t launch_skinny(SkinnyParams &p, cudaStream_t s) {
  p.steps = (p.k + STEP - 1) / STEP;
  const uint32_t ctas = 148u * ((p.n + 148u * MAX_ROWS - 1u) / (148u * MAX_ROWS));
  p.cta_rows = (p.n + ctas - 1u) / ctas;
  p.k_warps = 1;
  while (p.k_warps < (uint32_t)WARPS && p.k_warps * 2u <= p.steps) p.k_warps *= 2u;
  const size_t smem = WARPS * DEPTH * SLOT_BYTES + (size_t)((p.cta_rows + 15u) / 16u) * p.k_warps * (2 * TG * 16) * 4;
  auto kernel = skinny_kernel<TG, BF16, MODE>;
  static bool ready[64];  // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (!__atomic_load_n(&ready[dev & 63], __ATOMIC_ACQUIRE)) {  // threads that meet here do the same
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MAX_SMEM);
    if (e != cudaSuccess) return e;
    __atomic_store_n(&ready[dev & 63], true, __ATOMIC_RELEASE);
  }
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

template <int TG, bool BF16>
cudaError_t dispatch(SkinnyParams &p, int mode, cudaStream_t s) {
  if (mode == WHOLE) return launch_skinny<TG, BF16, WHOLE>(p, s);
  return mode == ALIGNED ? launch_skinny<TG, BF16, ALIGNED>(p, s) : launch_skinny<TG, BF16, BYTES>(p, s);
}

}  // namespace
}  // namespace sklb

using namespace sklb;

extern "C" int skl_b200_mxf4_skinny_supported(uint64_t m, uint64_t n, uint64_t k) {
  return m >= 1 && m <= 4 && n >= 1 && k >= 1 && n < (1ull << 31) && k < (1ull << 31);
}

extern "C" int skl_b200_launch_mxf4_skinny(uint32_t m, uint32_t n, uint32_t k, float alpha, const void *a, int ta, int64_t rsa,
                                           const void *b, int64_t csb, const void *sb, int64_t cssb, float beta, void *c,
                                           int tc, int64_t rsc, int static_b, void *stream) {
  SkinnyParams p;
  p.a = a, p.b = (const uint8_t *)b, p.sb = (const uint8_t *)sb, p.c = c;
  p.rsa = rsa, p.csb = csb, p.cssb = cssb, p.rsc = rsc;
  p.m = m, p.n = n, p.k = k, p.kblocks = (k + 31) / 32;
  p.alpha = alpha, p.beta = beta, p.tc = tc, p.static_b = static_b;
  p.a_vec = (reinterpret_cast<uintptr_t>(a) & 15u) == 0 && (m == 1 || rsa % 8 == 0);
  const bool vec = (reinterpret_cast<uintptr_t>(b) & 15u) == 0 && (n == 1 || csb % 16 == 0);
  const bool svec = (reinterpret_cast<uintptr_t>(sb) & 7u) == 0 && (n == 1 || cssb % 8 == 0);
  const int mode = !vec ? BYTES : (svec && p.kblocks % 8 == 0 ? WHOLE : ALIGNED);
  cudaStream_t s = (cudaStream_t)stream;
  const bool bf = ta == SKL_DT_BF16;
  if (m <= 2) return (int)(bf ? dispatch<1, true>(p, mode, s) : dispatch<1, false>(p, mode, s));
  return (int)(bf ? dispatch<2, true>(p, mode, s) : dispatch<2, false>(p, mode, s));
}
