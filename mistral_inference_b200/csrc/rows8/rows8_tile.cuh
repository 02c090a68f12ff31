// y[t, n] = sum over blocks b of 2^(ex[t, b] + ew[n, b]) sum over the block of cx[t, k] cw[n, k]: products of 8-bit rows on tcgen05.mma.kind::mxf8f6f4, which multiplies
// by both powers as it adds to the fp32 accumulator in tensor memory.
//
// The simplest form: a CTA computes 128 tokens x 256 features over all of K.  Warp 0 copies (128 bytes of 128 token rows and 256 feature rows a stage, and every fourth stage the
// scales of four blocks), warp 1 multiplies, warps 2-5 store, a token a thread.
#pragma once
#include "rows8_common.cuh"

namespace mb200 {

enum { R8_OUT_BF16 = 0, R8_OUT_F32 = 1, R8_OUT_GATE = 2 };
struct ProductParams {
  int T, N, K;  // N: rows of the weights
  int64_t ld;   // of `out`, in elements
  void* out;    // [T, N] bf16 or fp32
  uint8_t *codes, *scales;  // of gated units
  int width, quads;         // of gated units: bytes of a row of codes, quads of blocks
};

// 4 K = 32 steps of a block; a, b: lower words of the tiles' descriptors, sa, sb: tensor memory of their scales, block: which byte of four
constexpr uint32_t R8_IDESC = 1u << 23;  // e4m3 by e4m3, scales e8m0
__device__ __forceinline__ uint32_t r8_idesc(int rows, int columns, uint32_t block) { return R8_IDESC | (uint32_t)(columns >> 3) << 17 | (uint32_t)(rows >> 4) << 24 | block << 29 | block << 4; }
__device__ __forceinline__ void umma_mx8(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 da, db;\n"
      "mov.b64 da, {%1, %7};\n"
      "mov.b64 db, {%2, %7};\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %3, [%4], [%5], p;\n"
      "}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "n"(UMMA_DESC_HI)
      : "memory");
}
// 512 bytes of scales (32 lanes x 16 bytes) to four columns of tensor memory, in every quarter of its lanes
constexpr uint32_t R8_SCALE_DESC_HI = (128u >> 4) | (1u << 14);  // no swizzle, eight rows of 16 bytes side by side
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t smem_addr) {
  asm volatile(
      "{\n"
      ".reg .b64 d;\n"
      "mov.b64 d, {%1, %2};\n"
      "tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n"
      "}\n" ::"r"(taddr),
      "r"((smem_addr & 0x3ffff) >> 4), "n"(R8_SCALE_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)), "l"(map), "r"(smem_u32(bar)),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ float silu_times(float gate, float up) {  // within 2^-20: e4m3 keeps 2^-4
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(gate * -1.4426950408889634f));
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return gate * r * up;
}

// 32 features n .. of token t
template <int OUT>
__device__ __forceinline__ void r8_store32(const ProductParams& p, int64_t t, int n, const uint32_t (&v)[32]) {
  using O = std::conditional_t<OUT == R8_OUT_F32, float, bf16>;
  O* to = reinterpret_cast<O*>(p.out) + t * p.ld + n;
  if (n + 32 <= p.N && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
    if constexpr (OUT == R8_OUT_F32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) reinterpret_cast<uint4*>(to)[i] = make_uint4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack_bf16x2(__uint_as_float(v[8 * i + 2 * j]), __uint_as_float(v[8 * i + 2 * j + 1]));
        reinterpret_cast<uint4*>(to)[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (n + i < p.N) to[i] = (O)__uint_as_float(v[i]);
}

constexpr int RT_ROWS = 128, RT_COLS = 256, RT_STAGES = 4, RT_THREADS = 192;
constexpr int RT_A = RT_ROWS * R8_BLOCK, RT_B = RT_COLS * R8_BLOCK, RT_SCALES = 3 * R8_TILE, RT_STAGE = RT_A + RT_B + 2048 /* scales; stages start on 1024 bytes */;
constexpr int RT_SMEM = RT_STAGES * RT_STAGE + 1024;

template <int OUT>
__global__ void __launch_bounds__(RT_THREADS, 1) rows8_tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sx,
                                                                   const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ ProductParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[RT_STAGES], empty[RT_STAGES], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int gave_up;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_n = (p.N + RT_COLS - 1) / RT_COLS, num_k = (p.K + R8_BLOCK - 1) / R8_BLOCK;
  const int n0 = (int)(blockIdx.x % num_n) * RT_COLS, t0 = (int)(blockIdx.x / num_n) * RT_ROWS;
  if (threadIdx.x == 0) {
    for (int i = 0; i < RT_STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    mbar_init(&done, 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot, ts_x = tmem + RT_COLS, ts_w = ts_x + 4;
  pdl_trigger();
  pdl_wait();
  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      for (int kb = 0; kb < num_k; ++kb) {
        const int s = kb % RT_STAGES;
        if (!bounded_wait(&empty[s], ((kb / RT_STAGES) & 1) ^ 1, &gave_up)) break;
        uint8_t* st = smem + s * RT_STAGE;
        const bool scales = kb % 4 == 0;
        mbar_arrive_expect_tx(&full[s], RT_A + RT_B + (scales ? RT_SCALES : 0));
        tma_load_2d(st, &map_x, &full[s], kb * R8_BLOCK, t0);
        tma_load_2d(st + RT_A, &map_w, &full[s], kb * R8_BLOCK, n0);
        if (scales) {
          tma_load_3d(st + RT_A + RT_B, &map_sx, &full[s], 0, kb / 4, t0 / 128);
          tma_load_3d(st + RT_A + RT_B + R8_TILE, &map_sw, &full[s], 0, kb / 4, n0 / 128);
        }
        issued = kb + 1;
      }
      if (gave_up)  // this CTA's copies land before it leaves
        for (int kb = issued > RT_STAGES ? issued - RT_STAGES : 0; kb < issued; ++kb) {
          int zero = 0;
          bounded_wait(&full[kb % RT_STAGES], (kb / RT_STAGES) & 1, &zero);
        }
    }
  } else if (warp == 1) {
    const uint32_t ring = umma_desc_lo(smem_u32(smem));
    bool fine = true;
    for (int kb = 0; kb < num_k && fine; ++kb) {
      const int s = kb % RT_STAGES;
      fine = bounded_wait(&full[s], (kb / RT_STAGES) & 1, &gave_up);
      fine = __all_sync(0xffffffffu, fine);
      if (!fine) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t a = ring + s * (RT_STAGE >> 4), b = a + (RT_A >> 4);
        if (kb % 4 == 0) {
          const uint32_t src = smem_u32(smem + s * RT_STAGE + RT_A + RT_B);
          copy_scales(ts_x, src);
          copy_scales(ts_w, src + R8_TILE);
          copy_scales(ts_w + 4, src + 2 * R8_TILE);
        }
        const uint32_t idesc = r8_idesc(RT_ROWS, RT_COLS, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_mx8(tmem, a + 2 * k, b + 2 * k, idesc, ts_x, ts_w, (kb > 0 || k > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
        if (kb == num_k - 1) umma_commit(&done);
      }
      __syncwarp();
    }
  } else {
    const bool fine = bounded_wait(&done, 0, &gave_up);
    tc_fence_after();
    const bool whole = __all_sync(0xffffffffu, fine);
    const int row = (warp & 3) * 32 + lane;
    const int64_t t = (int64_t)t0 + row;
    const uint32_t at = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t none = 0x7fffffffu;  // where the wait ran out
    if constexpr (OUT != R8_OUT_GATE) {
#pragma unroll 1
      for (int c = 0; c < RT_COLS; c += 32) {
        uint32_t v[32];
        if (whole) {
          tmem_ld_32x32b_x32(at + c, v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = none;
        }
        if (t < p.T) r8_store32<OUT>(p, t, n0 + c, v);
      }
    } else {
      float g[128];
      uint32_t amax = 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t v[32];
        if (whole) {
          tmem_ld_32x32b_x32(at + 32 * c, v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = none;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          g[16 * c + i] = silu_times(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
          amax = max(amax, r8_bits(g[16 * c + i]));
        }
      }
      const uint32_t byte = r8_byte(amax);
      const int block = n0 / RT_COLS;
      if (t < p.T) {
        uint4* to = reinterpret_cast<uint4*>(p.codes + t * p.width + (int64_t)block * R8_BLOCK);
        const float inverse = r8_inverse(byte);
#pragma unroll
        for (int c = 0; c < 8; ++c) {
          float x[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = g[16 * c + i];
          to[c] = r8_codes16(x, amax, inverse);
        }
      }
      uint8_t* sc = p.scales + r8_scale_at(t, block >> 2, p.quads);
      sc[block & 3] = (uint8_t)(t < p.T ? byte : 127u);
      if (block == num_n - 1)
        for (int b = (block & 3) + 1; b < 4; ++b) sc[b] = 127;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, 512);
}

// ---- host ----
template <int OUT>
int launch_rows8_tile(const ProductParams& p, const void* xc, const void* xs, const void* wc, const void* ws, cudaStream_t st) {
  CUtensorMap mx, mw, msx, msw;
  const int64_t width = r8_width(p.K), quads = r8_quads(p.K);
  int rc = r8_code_map(&mx, xc, p.T, width, RT_ROWS);
  if (!rc) rc = r8_code_map(&mw, wc, p.N, width, RT_COLS);
  if (!rc) rc = r8_scale_map(&msx, xs, p.T, quads, 1);
  if (!rc) rc = r8_scale_map(&msw, ws, p.N, quads, 2);
  if (rc) return rc;
  const int64_t tiles = (int64_t)((p.N + RT_COLS - 1) / RT_COLS) * ((p.T + RT_ROWS - 1) / RT_ROWS);
  MB_CHECK_CUDA(device_info::allow_shared<rows8_tile_kernel<OUT>>(RT_SMEM));
  MB_CHECK_CUDA(launch_pdl(rows8_tile_kernel<OUT>, dim3((unsigned)tiles), dim3(RT_THREADS), RT_SMEM, st, mx, mw, msx, msw, p));
  return MB200_OK;
}

}  // namespace mb200
