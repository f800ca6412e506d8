// mxf4_planes.cu -- C = alpha * A W^T + beta * C for a batch of rows of A (bf16 / fp16) and MX-FP4 weights W [n][k], on the
// block-scaled tensor-core instruction: tcgen05.mma.kind::mxf8f6f4.block_scale takes E2M1 weights with their E8M0 scales as
// they are, next to an E5M2 operand with scales of its own.
//
// A enters as a sum of E5M2 matrices ("planes").  In a block of 32 with largest magnitude in [2^e, 2^(e+1)) the first plane
// is a / 2^(e - 14) rounded to E5M2 (3 significant bits), the next the remainder / 2^(e - 17), and so on, each remainder exact
// in fp32.  bf16 has 8 significant bits, fp16 11: after three and four planes nothing is left of a value down to 2^-29 of its
// block's largest, and less than 2^-36 of the largest is left of smaller ones.  (E4M3 planes, 4 bits each, would be two and
// three, but their range of exponents rounds what is 2^-20 of a block's largest.)  Products with E2M1 are exact, sums fp32.
// A block with an infinity or a NaN gets NaN scales: the row's results are NaN.
//
// planes_kernel writes the planes, below each other, and lays their scales out the way tcgen05.cp takes them (512 bytes for
// 128 rows and 4 blocks of k: row r at (r % 32) * 16 + (r / 32) * 4).  The product kernel: one tile of 128 rows by up to 256
// rows of W per CTA, k split over a cluster of CTAs so that the chip is full.  A stage holds as few tiles of A as the planes of
// its rows need: all planes below each other in one (42 bf16, 32 fp16 rows), pairs of planes (64 rows), or each plane its own;
// the MMAs add over the tiles, the epilogue over the planes of a tile.  Warp 0 loads planes and scales by TMA; eight warps bring
// the packed weights through registers to where the instruction wants them, 16 elements to 16 bytes, and their scales (the
// TMA's own spreading copy of 4-bit elements took 1.1 us for a stage's 256 x 128, several times what HBM needs for them);
// warp 1 copies the scales to TMEM and issues the MMAs (K = 32 each, 4 to a stage and tile).  At the end all warps read the
// accumulator, the cluster adds its parts through distributed shared memory in a fixed order, and every CTA stores a share of
// the rows.  Every wait is bounded.
//
// 14336 x 4096, both kernels, in a graph: 5 rows 19.9 us, 32 rows 22.3, 61 rows 26.7, 128 rows 31.8 (31 MB: 4.9 us of HBM; W
// widened to bf16 and multiplied: 64 rows 50 us); 4096 x 4096 with 5 rows 12.8, 1024 x 1024 9.0, which is what the two launches, filling
// and emptying cost.  Beyond that a stage takes about 0.7 us: the hand-over from the loaders to the MMAs, not HBM.
#include <cuda.h>

#include "loads.cuh"
#include "numerics.cuh"

namespace sklb {
namespace {

constexpr int BM = 128, BN = 256, BK = 128;  // largest tile; elements of k of a stage, one byte each in shared memory
constexpr int AHEAD = 2;                      // stages of packed weights that a loader holds in registers (3 to 6: 1 to 2 us slower)
constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
constexpr int SF_BYTES = 512;  // scales of 128 rows and one stage
constexpr int LOADERS = 8, THREADS = 64 + 32 * LOADERS;  // warp 0: TMA, warp 1: MMA, then the loaders
constexpr uint32_t ERR_EMPTY = 0x401, ERR_FULL = 0x402, ERR_DONE = 0x403;

// PLANES: tiles of A to a stage
template <int PLANES>
struct Cfg {
  static constexpr int TX = PLANES * (A_BYTES + SF_BYTES);                                          // bytes that the TMA brings
  static constexpr int STAGE = (PLANES * A_BYTES + B_BYTES + (PLANES + 2) * SF_BYTES + 1023) / 1024 * 1024;  // tiles start on 1024 bytes
  static constexpr int STAGES = PLANES == 1 ? 4 : (PLANES == 2 ? 3 : 2);
  static constexpr int SMEM = 1024 + STAGES * STAGE + 256;
  static_assert(SMEM <= 227 * 1024, "exceeds the shared memory one CTA can have");
  static_assert(STAGES * STAGE >= BM * BN * 4, "the accumulator is staged where the operands were");
};

struct PlanesParams {
  const uint8_t *sfa;  // [row tile of all planes][stage][512]
  const uint8_t *b, *sb;
  int64_t csb, cssb;
  void *c;
  int64_t rsc;
  int m, n, stages, tiles_m, row_bytes, bn;  // row_bytes: of a packed row; bn: rows of W of a tile, a multiple of 16
  int plane_tiles;                       // row tiles from a stage's tile of A to its next
  int fold;                              // planes of m rows in a tile
  float alpha, beta;
  int tc, c_vec, b_vec, s_vec;
  uint64_t wait_ns;
  uint32_t *status;
  int skip_loads;  // testing aid: loads are announced, not issued
};

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait: false when it ran out or another thread of the CTA gave up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile uint32_t *abort_flag, uint32_t *status, uint32_t code,
                                         uint64_t limit_ns) {
  uint64_t t0 = 0;
  for (uint32_t spins = 0;; ++spins) {
    if (bar_try(bar, parity)) return true;
    if ((spins & 63u) == 63u) {
      if (*abort_flag) return false;
      uint64_t now;
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
      if (t0 == 0) t0 = now;
      if (now - t0 > limit_ns) {
        *abort_flag = 1u;
        atomicCAS(status, 0u, code);
        return false;
      }
    }
  }
}
// For a warp's own copies in flight: nobody to tell, nothing to give up.  t0: when the first such wait began.
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity, uint64_t &t0, uint64_t limit_ns) {
  for (uint32_t spins = 0; !bar_try(bar, parity); ++spins) {
    if ((spins & 63u) != 63u) continue;
    uint64_t now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (t0 == 0) t0 = now;
    if (now - t0 > limit_ns) return;
  }
}
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap *tm, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst), "l"(tm),
               "r"(bar), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void bulk(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
               : "memory");
}
// k-major operand, 128-byte rows with the 128-byte swizzle, 8-row groups 1024 bytes apart
__device__ __forceinline__ uint64_t operand_desc(uint32_t at) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)(16u >> 4) << 16 | (uint64_t)(1024u >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// 32 rows x 16 bytes of scales, no swizzle, 8-row groups 128 bytes apart
__device__ __forceinline__ uint64_t scale_desc(uint32_t at) {
  return (uint64_t)((at >> 4) & 0x3FFFu) | (uint64_t)(128u >> 4) << 32 | 1ull << 46;
}
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// ------------------------------------------------------------------------------------------------------------ planes
// One thread for 8 elements of k, four lanes to a block; plane p of row r is row (p / fold) * tile_span + (p % fold) * m + r.
// PLANES fills whole tiles: planes that are not needed (their elements come out as zeros) are written like the others.  Rows
// that no plane has are not written, nor are their scales: whatever lies there only reaches accumulator rows that are not
// used.  `stages` * 128 is the k of the planes; the elements behind k are zeros.
template <int PLANES>
__global__ void __launch_bounds__(256)
    planes_kernel(uint8_t *__restrict__ planes, uint8_t *__restrict__ sfa, const uint16_t *a, int64_t rsa, int m, int k, int stages,
                  int bf16, int a_vec, int fold, int tile_span) {
  dep_wait();
  const int64_t kp = (int64_t)stages * BK;
  const int64_t groups = kp / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  const int64_t row64 = i / groups;
  const bool in = row64 < m;
  const int row = in ? (int)row64 : 0, g = in ? (int)(i - row64 * groups) : 0, kk = g * 8;
  float x[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = 0.0f;
  if (in) {
    const uint16_t *src = a + (int64_t)row * rsa + kk;
    uint32_t w[4] = {0u, 0u, 0u, 0u};
    if (a_vec && kk + 8 <= k) {
      const uint4 v = ld_v4(src);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (kk + e < k) w[e >> 1] |= ld_u16(src + e) << (16 * (e & 1));
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      x[2 * q] = bf16 ? dec_bf16(w[q] & 0xFFFFu) : dec_f16(w[q] & 0xFFFFu);
      x[2 * q + 1] = bf16 ? u2f(w[q] & 0xFFFF0000u) : dec_f16(w[q] >> 16);
    }
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, f2u(x[e]) & 0x7FFFFFFFu);
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
  top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
  const int ef = (int)(top >> 23);
  // scale byte of the first plane: 2^(ef - 127 - 14), then 3 less for each further one, not below 2^-127 (E8M0's smallest; every
  // bf16 and fp16 value is a multiple of 2^-133, so nothing is lost there)
#pragma unroll
  for (int p = 0; p < PLANES; ++p) {
    int s = ef - 14 - 3 * p;
    s = s < 0 ? 0 : s;
    const float up = u2f((uint32_t)(254 - s) << 23), down = s == 0 ? u2f(0x00400000u) : u2f((uint32_t)s << 23);  // 2^(127 - s), 2^(s - 127)
    uint32_t w[2];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const uint32_t lo = hw_e5m2x2(x[4 * q] * up, x[4 * q + 1] * up), hi = hw_e5m2x2(x[4 * q + 2] * up, x[4 * q + 3] * up);
      w[q] = lo | hi << 16;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[4 * q + e] = __fmaf_rn(-dec_e5m2((w[q] >> (8 * e)) & 0xFFu), down, x[4 * q + e]);
    }
    if (ef == 255) s = 255, w[0] = w[1] = 0u;
    if (in) {
      const int64_t at = (int64_t)(p / fold) * tile_span + (int64_t)(p % fold) * m + row;
      *reinterpret_cast<uint2 *>(planes + at * kp + kk) = make_uint2(w[0], w[1]);
      if ((g & 3) == 0) {
        const int r = (int)(at % BM), blk = g >> 2;
        sfa[(at / BM * stages + (blk >> 2)) * SF_BYTES + (r % 32) * 16 + (r / 32) * 4 + (blk & 3)] = (uint8_t)s;
      }
    }
  }
}

// ----------------------------------------------------------------------------------------------------------- product
template <int PLANES>
__global__ void __launch_bounds__(THREADS, 1)
    product_kernel(const __grid_constant__ CUtensorMap tma, const PlanesParams p) {
  using C = Cfg<PLANES>;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw), tiles = (raw + 1023u) & ~1023u, bars = tiles + C::STAGES * C::STAGE;
  const uint32_t full = bars, empty = bars + 8 * C::STAGES, done = bars + 16 * C::STAGES;
  uint8_t *gen = smem_raw + (bars - raw);
  volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(gen + 16 * C::STAGES + 8), *abort_flag = tmem_slot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t rank, ranks;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ranks));
  const int tile = (int)(blockIdx.x / ranks), mi = tile % p.tiles_m, ni = tile / p.tiles_m;
  const int k0 = (int)((int64_t)p.stages * rank / ranks), k1 = (int)((int64_t)p.stages * (rank + 1) / ranks);

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      bar_init(full + 8 * s, 1 + LOADERS);
      bar_init(empty + 8 * s, 1);
    }
    bar_init(done, 1);
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_addr((const void *)tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;
  dep_wait();

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int s = k0; s < k1; ++s, ++issued) {
        const int i = s - k0, st = i % C::STAGES;
        if (i >= C::STAGES && !bar_wait(empty + 8 * st, (uint32_t)(i / C::STAGES - 1) & 1u, abort_flag, p.status, ERR_EMPTY, p.wait_ns)) break;
        const uint32_t at = tiles + st * C::STAGE, fb = full + 8 * st, sf = at + PLANES * A_BYTES + B_BYTES;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(fb), "r"((uint32_t)C::TX) : "memory");
        if (p.skip_loads) continue;
#pragma unroll
        for (int q = 0; q < PLANES; ++q) {
          const int row_tile = q * p.plane_tiles + mi;
          tma_2d(at + q * A_BYTES, &tma, fb, s * BK, row_tile * BM);
          bulk(sf + q * SF_BYTES, p.sfa + ((int64_t)row_tile * p.stages + s) * SF_BYTES, SF_BYTES, fb);
        }
      }
      // the copies of the last stages land before the memory is used for anything else; after a wait has run out their barriers miss
      // the loaders' arrivals, and one limit for all of them is long past the time that a copy takes
      uint64_t t0 = 0;
      for (int i = issued > C::STAGES ? issued - C::STAGES : 0; i < issued && !p.skip_loads; ++i)
        bar_drain(full + 8 * (i % C::STAGES), (uint32_t)(i / C::STAGES) & 1u, t0, p.wait_ns);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true;
      for (int s = k0; s < k1; ++s) {
        const int i = s - k0, st = i % C::STAGES;
        if (!bar_wait(full + 8 * st, (uint32_t)(i / C::STAGES) & 1u, abort_flag, p.status, ERR_FULL, p.wait_ns)) {
          ok = false;
          break;
        }
        // scales of the stage: plane q at columns 256 + 32 (i % 2) + 4 q, W at + 16 (rows 0..127) and + 20 (128..255).  A copy is
        // ordered before later MMAs of its thread, not behind earlier ones: the MMAs of stage i - 2, which read the region
        // this stage overwrites, have to be done (those of stage i - 1 keep the tensor core busy meanwhile).
        if (i >= 2 &&
            !bar_wait(empty + 8 * ((i - 2) % C::STAGES), (uint32_t)((i - 2) / C::STAGES) & 1u, abort_flag, p.status, ERR_EMPTY, p.wait_ns)) {
          ok = false;
          break;
        }
        fence_after();
        const uint32_t at = tiles + st * C::STAGE, sf = at + PLANES * A_BYTES + B_BYTES;
        const uint32_t tsf = tmem + 256u + (uint32_t)(i & 1) * 32u;
#pragma unroll
        for (int q = 0; q < PLANES; ++q)
          asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tsf + 4u * q), "l"(scale_desc(sf + q * SF_BYTES)) : "memory");
#pragma unroll
        for (int q = 0; q < 2; ++q)
          asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tsf + 16u + 4u * q), "l"(scale_desc(sf + (PLANES + q) * SF_BYTES)) : "memory");
        const uint64_t db = operand_desc(at + PLANES * A_BYTES);
#pragma unroll
        for (int q = 0; q < PLANES; ++q) {
          const uint64_t da = operand_desc(at + q * A_BYTES);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            // E5M2 x E2M1 with E8M0 scales, byte j of the scales' 4-byte columns; M = 128, N = p.bn
            const uint32_t idesc = (uint32_t)j << 4 | 1u << 7 | 5u << 10 | (uint32_t)(p.bn >> 3) << 17 | 1u << 23 | (uint32_t)(BM >> 4) << 24 |
                                   (uint32_t)j << 29;
            const uint32_t accumulate = (i | q | j) != 0;
            asm volatile(
                "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(tmem),
                "l"(da + (uint64_t)(2 * j)), "l"(db + (uint64_t)(2 * j)), "r"(idesc), "r"(accumulate), "r"(tsf + 4u * q), "r"(tsf + 16u)
                : "memory");
          }
        }
        commit(empty + 8 * st);
      }
      if (ok) commit(done);
    }
  } else {
    // packed weights: 4 lanes to a row, 16 bytes (32 elements) each, a warp takes 8 rows at a time, AHEAD stages of loads in flight;
    // the halves of lane c's piece go to the 16-byte chunks 2 c and 2 c + 1 of row r, chunk i at i ^ (r % 8): the 128-byte swizzle.
    // Scales: one row to a thread, 16 blocks (four stages) to a load where they are aligned.
    constexpr int PIECES = BN / (8 * LOADERS);
    const int lw = warp - 2, sub = lane >> 2, c = lane & 3;
    uint4 w[AHEAD][PIECES];
    auto load = [&](uint4 (&v)[PIECES], int s) {
      const int byte = s * (BK / 2) + 16 * c;
#pragma unroll
      for (int q = 0; q < PIECES; ++q) {
        const int r = q * 8 * LOADERS + 8 * lw + sub, row = ni * p.bn + r;
        v[q] = make_uint4(0u, 0u, 0u, 0u);
        if (s < k1 && r < p.bn && row < p.n && byte < p.row_bytes) {
          const uint8_t *src = p.b + (int64_t)row * p.csb + byte;
          if (p.b_vec) {
            v[q] = ld_stream_v4(src);
          } else {
            const uint2 lo = ld_v2(src), hi = ld_v2(src + 8);
            v[q] = make_uint4(lo.x, lo.y, hi.x, hi.y);
          }
        }
      }
    };
    const int srow = 32 * lw + lane, wrow = ni * p.bn + srow;
    const bool has_scale = srow < p.bn && wrow < p.n;
    const uint8_t *ssrc = p.sb + (has_scale ? (int64_t)wrow * p.cssb : 0);
    const uint32_t sdst = (uint32_t)((srow / 128) * SF_BYTES + (srow % 32) * 16 + (srow % 128 / 32) * 4);
    const int kblocks = p.row_bytes / 16;
    uint4 sc = make_uint4(0u, 0u, 0u, 0u), sc_next = sc;
    // the scales of stages s & ~3 .. s | 3; blocks and rows that do not exist get 0, a scale that is finite
    auto load_scales = [&](uint4 &v, int s) {
      const int b0 = (s & ~3) * 4;
      v = make_uint4(0u, 0u, 0u, 0u);
      if (!has_scale || s >= k1) return;
      if (p.s_vec && b0 + 16 <= kblocks) {
        v = ld_v4(ssrc + b0);
      } else {
        uint32_t q[4] = {0u, 0u, 0u, 0u};
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (b0 + e < kblocks) q[e >> 2] |= ld_u8(ssrc + b0 + e) << (8 * (e & 3));
        v = make_uint4(q[0], q[1], q[2], q[3]);
      }
    };
    load_scales(sc, k0);
#pragma unroll
    for (int j = 0; j < AHEAD; ++j) load(w[j], k0 + j);
    load_scales(sc_next, (k0 | 3) + 1);
    bool ok = true;
    for (int i0 = 0; ok && k0 + i0 < k1; i0 += AHEAD) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int i = i0 + j, s = k0 + i, st = i % C::STAGES;
        if (s >= k1) break;
        if (i >= C::STAGES) ok = bar_wait(empty + 8 * st, (uint32_t)(i / C::STAGES - 1) & 1u, abort_flag, p.status, ERR_EMPTY, p.wait_ns);
        if (!__all_sync(0xFFFFFFFFu, ok)) {
          ok = false;
          break;
        }
        const uint32_t at = tiles + st * C::STAGE + PLANES * A_BYTES;
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
          const int r = q * 8 * LOADERS + 8 * lw + sub;
          if (r < p.bn) {
            const uint32_t row = at + (uint32_t)r * 128u;
            asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(row + (uint32_t)(((2 * c) ^ (r & 7)) << 4)), "r"(w[j][q].x), "r"(w[j][q].y) : "memory");
            asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(row + (uint32_t)(((2 * c + 1) ^ (r & 7)) << 4)), "r"(w[j][q].z), "r"(w[j][q].w) : "memory");
          }
        }
        const uint32_t word = (s & 3) == 0 ? sc.x : ((s & 3) == 1 ? sc.y : ((s & 3) == 2 ? sc.z : sc.w));
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(at + B_BYTES + PLANES * SF_BYTES + sdst), "r"(word) : "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // visible to the tensor core, then counted
        __syncwarp();
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(full + 8 * st) : "memory");
        load(w[j], s + AHEAD);
        if ((s & 3) == 3) {
          sc = sc_next;
          load_scales(sc_next, s + 5);
        }
      }
    }
  }
  // every MMA has finished: the accumulator is whole and the stages are free to hold it
  __syncwarp();
  const bool whole = k1 > k0 && bar_wait(done, 0u, abort_flag, p.status, ERR_DONE, p.wait_ns);
  __syncthreads();
  fence_after();
  const int rows = min(BM, p.m - mi * BM), cols = min(p.bn, p.n - ni * p.bn), used = p.fold > 1 ? p.fold * p.m : rows;  // folded: m <= 64, one row tile
  float *acc = reinterpret_cast<float *>(smem_raw + (tiles - raw));  // [row][256], 16-byte groups rotated by the row
  if (warp >= 2) {
    const int quad = warp & 3, half = (warp - 2) >> 2, row = quad * 32 + lane;
    float4 *out = reinterpret_cast<float4 *>(acc + row * BN);
#pragma unroll
    for (int ch = 0; ch < 4; ++ch) {
      uint32_t r[32];
      const uint32_t at = tmem + (uint32_t)(half * 128 + ch * 32) + ((uint32_t)(quad * 32) << 16);
      asm volatile(
          "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
          "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
          "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
          : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
            "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
            "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
            "=r"(r[31])
          : "r"(at));
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        const int gq = half * 32 + ch * 8 + q;
        float4 v = make_float4(u2f(r[4 * q]), u2f(r[4 * q + 1]), u2f(r[4 * q + 2]), u2f(r[4 * q + 3]));
        if (!whole) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // a share of k without a stage, or a wait that ran out
        if (row < used) out[(gq & ~7) | ((gq + row) & 7)] = v;
      }
    }
  }
  fence_before();
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
  // rows rank, rank + ranks, ...: a warp takes a row, a lane 4 columns at a time
  for (int row = (int)rank + (int)ranks * warp; row < rows; row += (int)ranks * (THREADS / 32)) {
    const int64_t c0 = (int64_t)(mi * BM + row) * p.rsc + (int64_t)ni * p.bn;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int gq = h * 32 + lane, col = gq * 4;
      if (col >= cols) continue;
      float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int q = 0; q < p.fold; ++q) {
        const int from = row + q * p.m;  // the row's planes
        const uint32_t at = smem_addr(acc + from * BN + (((gq & ~7) | ((gq + from) & 7)) * 4));
        for (uint32_t r = 0; r < ranks; ++r) {
          uint32_t remote;
          float4 w;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(at), "r"(r));
          asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(w.x), "=f"(w.y), "=f"(w.z), "=f"(w.w) : "r"(remote) : "memory");
          v[0] += w.x, v[1] += w.y, v[2] += w.z, v[3] += w.w;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = __fmul_rn(p.alpha, v[e]);
        if (p.beta != 0.0f && col + e < cols) v[e] = __fadd_rn(__fmul_rn(p.beta, load_c_f32(p.tc, p.c, c0 + col + e)), v[e]);
      }
      if (p.c_vec && col + 4 <= cols) {
        if (p.tc == SKL_DT_F32) {
          *reinterpret_cast<float4 *>((float *)p.c + c0 + col) = make_float4(v[0], v[1], v[2], v[3]);
        } else {
          const bool bf = p.tc == SKL_DT_BF16;
          const uint32_t lo = bf ? pack_bf16x2_no_nan(v[0], v[1]) : pack_f16x2_no_nan(v[0], v[1]);
          const uint32_t hi = bf ? pack_bf16x2_no_nan(v[2], v[3]) : pack_f16x2_no_nan(v[2], v[3]);
          *reinterpret_cast<uint2 *>((uint16_t *)p.c + c0 + col) = make_uint2(lo, hi);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (col + e < cols) store_c_f32(p.tc, p.c, c0 + col + e, v[e]);
      }
    }
  }
  // no CTA leaves while its shared memory may still be read
  if (ranks > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

typedef CUresult (*EncodeFn)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                             const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                             CUtensorMapFloatOOBfill);
EncodeFn encoder() {
  static EncodeFn fn = [] {
    void *sym = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) {
      (void)cudaGetLastError();
      return (EncodeFn) nullptr;
    }
    return (EncodeFn)sym;
  }();
  return fn;
}

int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }

struct Layout {
  int planes, fold, tiles;  // planes; planes to a tile; tiles of A to a stage
  int64_t stages, tile_span, tile_rows, kp, sfa_at, total;
};
Layout layout(uint64_t m, uint64_t k, int ta) {
  Layout l;
  l.planes = ta == SKL_DT_BF16 ? 3 : 4;
  l.fold = l.planes * m <= BM ? l.planes : (2 * m <= BM ? 2 : 1);
  l.tiles = (l.planes + l.fold - 1) / l.fold;
  l.stages = up((int64_t)k, BK) / BK;
  l.kp = l.stages * BK;
  l.tile_span = up((int64_t)m, BM);
  l.tile_rows = l.tiles * l.tile_span;
  l.sfa_at = l.tile_rows * l.kp;
  l.total = l.sfa_at + l.tile_rows / 128 * l.stages * SF_BYTES;
  return l;
}

cudaLaunchConfig_t product_config(unsigned grid, unsigned ranks, size_t smem, cudaStream_t s, cudaLaunchAttribute *attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cfg;
}

// Rows of W to a tile and CTAs to a cluster: the pair whose longest CTA has the fewest stages x rows, with all tiles on the chip
// at once if they fit.  How many clusters of a size fit is asked of the driver: with one CTA to an SM some SMs have no
// partners left for clusters of 4 and 8, and a second round costs as much as the first.
template <int PLANES>
cudaError_t launch_product(const CUtensorMap &tma, PlanesParams &p, cudaStream_t s) {
  struct Device {
    bool ready;
    int fit[4];  // clusters of 1, 2, 4, 8
  };
  static Device devices[64];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  Device &d = devices[dev & 63];
  cudaLaunchAttribute attr[2];
  if (!__atomic_load_n(&d.ready, __ATOMIC_ACQUIRE)) {  // threads that meet here find the same values
    e = cudaFuncSetAttribute(product_kernel<PLANES>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<PLANES>::SMEM);
    if (e != cudaSuccess) return e;
    for (int i = 0; i < 4; ++i) {
      cudaLaunchConfig_t q = product_config(1u << i, 1u << i, Cfg<PLANES>::SMEM, s, attr);
      q.numAttrs = 1;
      int n = 0;
      if (cudaOccupancyMaxActiveClusters(&n, product_kernel<PLANES>, &q) != cudaSuccess) {
        (void)cudaGetLastError();
        n = 0;
      }
      d.fit[i] = n;
    }
    if (d.fit[0] < 1) d.fit[0] = 1;
    __atomic_store_n(&d.ready, true, __ATOMIC_RELEASE);
  }
  unsigned ranks = 1;
  int64_t best = INT64_MAX, tiles = 0;
  for (int i = 0; i < 4; ++i) {
    const int64_t r = 1ll << i, fit = d.fit[i];
    if (fit < 1 || r > p.stages) break;
    const int64_t room = fit / p.tiles_m;  // tiles along n that fit
    int64_t bn = room > 0 ? up((p.n + room - 1) / room, 16) : BN;
    bn = bn > BN ? BN : (bn < 64 ? 64 : bn);
    const int64_t all = p.tiles_m * ((p.n + bn - 1) / bn), rounds = (all + fit - 1) / fit;
    const int64_t cost = rounds * ((p.stages + r - 1) / r) * (bn + 64);  // 64: a stage's part that does not shrink with bn
    if (cost < best) best = cost, ranks = (unsigned)r, p.bn = (int)bn, tiles = all;
  }
  if (tiles * ranks > 0x7FFFFFFFll) return cudaErrorInvalidValue;
  const cudaLaunchConfig_t cfg = product_config((unsigned)(tiles * ranks), ranks, Cfg<PLANES>::SMEM, s, attr);
  SKLB_COUNT_LAUNCH();
  return cudaLaunchKernelEx(&cfg, product_kernel<PLANES>, tma, (const PlanesParams)p);
}

}  // namespace
}  // namespace sklb

using namespace sklb;

// packed rows on 8 bytes
extern "C" int skl_b200_mxf4_planes_supported(uint64_t m, uint64_t n, uint64_t k, const void *b, int64_t csb) {
  return m >= 1 && n >= 1 && k >= 1 && m < (1ull << 22) && n < (1ull << 30) && k < (1ull << 30) &&
         (reinterpret_cast<uintptr_t>(b) & 7u) == 0 && (n == 1 || csb % 8 == 0) && encoder() != nullptr;
}

extern "C" size_t skl_b200_mxf4_planes_scratch(uint64_t m, uint64_t k, int ta) { return (size_t)layout(m, k, ta).total; }

extern "C" int skl_b200_launch_mxf4_planes(uint32_t m, uint32_t n, uint32_t k, float alpha, const void *a, int ta, int64_t rsa,
                                           const void *b, int64_t csb, const void *sb, int64_t cssb, float beta, void *c, int tc,
                                           int64_t rsc, void *scratch, uint32_t wait_limit_ms, int debug_skip_loads,
                                           uint32_t *dev_status, void *before_product, void *stream) {
  EncodeFn enc = encoder();
  if (!enc) return (int)cudaErrorNotSupported;
  const Layout l = layout(m, k, ta);
  cudaStream_t s = (cudaStream_t)stream;
  uint8_t *base = (uint8_t *)scratch;
  CUtensorMap tma;
  {
    cuuint64_t dims[2] = {(cuuint64_t)l.kp, (cuuint64_t)l.tile_rows}, strides[1] = {(cuuint64_t)l.kp};
    cuuint32_t box[2] = {BK, BM}, step[2] = {1, 1};
    if (enc(&tma, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return (int)cudaErrorInvalidValue;
  }
  const int es = tc == SKL_DT_F32 ? 4 : 2;
  {
    const int64_t blocks = ((int64_t)m * (l.kp / 8) + 255) / 256;
    if (blocks > 0x7FFFFFFFll) return (int)cudaErrorInvalidValue;
    const int a_vec = (reinterpret_cast<uintptr_t>(a) & 15u) == 0 && (m == 1 || rsa % 8 == 0);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    cfg.gridDim = dim3((unsigned)blocks);
    cfg.blockDim = dim3(256);
    cfg.stream = s;
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    SKLB_COUNT_LAUNCH();
    const int bf = ta == SKL_DT_BF16;
    // planes written: whole tiles
    const auto kernel = l.fold * l.tiles == 3 ? planes_kernel<3> : planes_kernel<4>;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, base, base + l.sfa_at, (const uint16_t *)a, rsa, (int)m,
                                       (int)k, (int)l.stages, bf, a_vec, l.fold, (int)l.tile_span);
    if (e != cudaSuccess) return (int)e;
  }
  PlanesParams p;
  p.sfa = base + l.sfa_at, p.c = c, p.rsc = rsc;
  p.b = (const uint8_t *)b, p.csb = csb, p.sb = (const uint8_t *)sb, p.cssb = cssb;
  p.b_vec = (reinterpret_cast<uintptr_t>(b) & 15u) == 0 && (n == 1 || csb % 16 == 0);
  p.s_vec = (reinterpret_cast<uintptr_t>(sb) & 15u) == 0 && (n == 1 || cssb % 16 == 0);
  p.m = (int)m, p.n = (int)n, p.stages = (int)l.stages, p.tiles_m = (int)((m + BM - 1) / BM);
  p.row_bytes = (int)((k + 31) / 32 * 16), p.plane_tiles = (int)(l.tile_span / BM), p.fold = l.fold;
  p.alpha = alpha, p.beta = beta, p.tc = tc;
  p.c_vec = (reinterpret_cast<uintptr_t>(c) & 15u) == 0 && (m == 1 || rsc * es % 16 == 0);
  p.wait_ns = (uint64_t)(wait_limit_ms ? wait_limit_ms : 2000u) * 1000000ull;
  p.status = dev_status, p.skip_loads = debug_skip_loads;
  if (before_product) (void)cudaEventRecord((cudaEvent_t)before_product, s);
  switch (l.tiles) {
    case 1: return (int)launch_product<1>(tma, p, s);
    case 2: return (int)launch_product<2>(tma, p, s);
    case 3: return (int)launch_product<3>(tma, p, s);
    default: return (int)launch_product<4>(tma, p, s);
  }
}
