// Products of 8-bit rows for prompts: pairs of CTAs share MMAs (cta_group::2), 256 tokens x 256 features a tile, persistent.
//
// Bound by the tensor pipe under the power cap.  A k-block of 128 takes the pair 512 clocks; each CTA copies 128 token rows and 128 feature rows of it, 32 KB, where a CTA
// by itself would copy 48 KB for the same products: L2 gives an SM some 64 bytes a clock.  Tokens are the MMA's rows (lanes), features its columns, so that a thread has a
// token's features next to one another and, of gated units, half of a block of 128 that share a power.
//
// Two accumulators of 256 columns and the scales' 12 do not fit the 512 columns of tensor memory: the second accumulator begins 16 columns inside the first.  An epilogue reads
// these first and says so (overlap), and the next tile's MMAs begin, some hundred clocks behind the last one's.  Tiles begin at multiples of 128 rows: scales of 128 rows fill four
// columns, and an MMA takes them from a multiple of four.
//
// 4096 tokens 28672 x 4096 (gate): 335 us in bursts of milliseconds, 2.87 PFLOP/s, 398 in loops of seconds; a k-block takes some 600 clocks, of which operands out of L2 and a tile's two ends are
// the rest.  With one accumulator and a tile a CTA of its own (128 tokens, 48 KB a k-block) 756.
// Tiles are dealt in rounds of the chip's pairs.  A last round that is at most half full is cut along K (pair_cut): its parts leave fp32 sums in scratch memory, which a second kernel, launched
// programmatically, adds in the order of k and finishes.  Nobody waits for another cluster.
//
// Warps: 0 copies, 1 multiplies (in the first CTA, for both), 2-9 epilogue, two to a quarter of the lanes, each 128 columns.  Waits are bounded; results of a tile whose wait ran out are NaN.
#pragma once
#include "../gemm_pair.cuh"
#include "rows8_product.cuh"

namespace mb200 {

constexpr int RP_ROWS = 256, RP_COLS = 256, RP_EPI_WARPS = 8, RP_THREADS = 64 + 32 * RP_EPI_WARPS;
constexpr int RP_HALF = 128 * R8_BLOCK, RP_STAGE = 2 * RP_HALF + 2048 /* 3 * R8_TILE of scales; stages start on 1024 bytes */, RP_STAGES = 6;
constexpr int RP_TURN = 2048;  // of an epilogue warp
constexpr int RP_SMEM = RP_STAGES * RP_STAGE + RP_EPI_WARPS * RP_TURN + 1024;
constexpr uint32_t RP_SECOND = 240, RP_SCALES_X = 496, RP_SCALES_W = 500;

__device__ __forceinline__ void umma_mx8_pair(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t sa, uint32_t sb, uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      ".reg .b64 da, db;\n"
      "mov.b64 da, {%1, %7};\n"
      "mov.b64 db, {%2, %7};\n"
      "setp.ne.b32 p, %6, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], da, db, %3, [%4], [%5], p;\n"
      "}\n" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(sa), "r"(sb), "r"(accumulate), "n"(UMMA_DESC_HI)
      : "memory");
}
// copy_scales in both CTAs, each from its own shared memory at this offset
__device__ __forceinline__ void copy_scales_pair(uint32_t taddr, uint32_t smem_addr) {
  asm volatile(
      "{\n"
      ".reg .b64 d;\n"
      "mov.b64 d, {%1, %2};\n"
      "tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n"
      "}\n" ::"r"(taddr),
      "r"((smem_addr & 0x3ffff) >> 4), "n"(R8_SCALE_DESC_HI)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)), "l"(map), "r"(bar),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}

// The cut of a last round: `rest` tiles behind `whole` ones, each in `cut` parts (no cut: 0, 1)
constexpr int RP_MAX_CUT = 4;
constexpr int64_t RP_PART = (int64_t)RP_ROWS * RP_COLS * sizeof(float);
struct PairCut {
  int rest, cut;
};
// Cut where the k-blocks saved (some 0.3 us each) are more than what the parts cost: their way through L2 and the second launch.  us of a call, uncut and cut: 256 tokens 4096 x 4096 15.7, 13.3;
// 777 tokens 6144 x 4096 27.2, 25.7; 130 tokens 4096 x 14336 38.7, 21.3; 400 tokens 40.0, 30.3; 4096 tokens 179, 174.
inline PairCut pair_cut(int64_t tiles, int num_k, int pairs) {
  const int rest = (int)(tiles % pairs);
  int cut = rest ? pairs / rest : 1;
  if (cut > RP_MAX_CUT) cut = RP_MAX_CUT;
  while (cut > 1 && num_k < 4 * cut) --cut;
  return cut > 1 && num_k - (num_k + cut - 1) / cut >= 16 ? PairCut{rest, cut} : PairCut{0, 1};
}
struct Pair8Params {
  ProductParams o;
  PairCut cut;
  int whole;       // tiles that are not cut
  float4* parts;   // [rest][cut][2 CTAs][64 quads of columns][128 rows]
};
struct PairItem {
  int tile, kb0, kb1, part, slot;  // part -1: a whole tile
};
__device__ __forceinline__ PairItem pair_item(const Pair8Params& p, int i, int num_k) {
  if (i < p.whole) return {i, 0, num_k, -1, 0};
  const int s = i - p.whole, part = s / p.cut.rest, slot = s % p.cut.rest;
  return {p.whole + slot, num_k * part / p.cut.cut, num_k * (part + 1) / p.cut.cut, part, slot};
}
__device__ __forceinline__ float4* pair_part(const Pair8Params& p, int slot, int part, int rank, int row) { return p.parts + ((int64_t)(slot * p.cut.cut + part) * 2 + rank) * (64 * 128) + row; }

template <int OUT>
__global__ void __launch_bounds__(RP_THREADS, 1) rows8_pair_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sx,
                                                                   const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ Pair8Params pp) {
  const ProductParams& p = pp.o;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  __shared__ uint64_t full[RP_STAGES], empty[RP_STAGES], tmem_full[2], tmem_empty[2], overlap;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int gave_up;
  __shared__ uint32_t meet[2][2][128];  // largest magnitudes of half a block of units
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, rank = (int)cluster_ctarank(), cluster = (int)blockIdx.x >> 1, clusters = (int)gridDim.x >> 1;
  const int num_m = (p.T + RP_ROWS - 1) / RP_ROWS, num_n = (p.N + RP_COLS - 1) / RP_COLS, num_k = (p.K + R8_BLOCK - 1) / R8_BLOCK, items = pp.whole + pp.cut.rest * pp.cut.cut;
  if (threadIdx.x == 0) {
    for (int i = 0; i < RP_STAGES; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; ++i) mbar_init(&tmem_full[i], 1), mbar_init(&tmem_empty[i], 2 * RP_EPI_WARPS);
    mbar_init(&overlap, RP_EPI_WARPS);  // the warps of one half of the columns, in both CTAs
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc<2>(&tmem_slot, 512);
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_trigger();
  pdl_wait();
  TileWalk walk;
  walk.start(num_m, num_n);
  int at = 0;
  auto go_to = [&](int tile) {
    walk.advance(tile - at, num_m, num_n);
    at = tile;
  };
  auto waited = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, bounded_wait(bar, parity, &gave_up)) != 0; };

  if (warp == 0) {
    const uint32_t full_first = cluster_first(full);
    uint32_t s = 0, par = 0, issued = 0;
    bool fine = true;
    for (int i = cluster; i < items && fine; i += clusters) {
      const PairItem it = pair_item(pp, i, num_k);
      go_to(it.tile);
      const int t0 = walk.m() * RP_ROWS + rank * 128, n0 = walk.n() * RP_COLS;
      for (int kb = it.kb0; kb < it.kb1; ++kb) {
        fine = waited(&empty[s], par ^ 1);
        if (!fine) break;
        if (elect_one()) {
          const bool scales = kb == it.kb0 || (kb & 3) == 0;
          uint8_t* const st = smem + s * RP_STAGE;
          const uint32_t bar = full_first + s * 8u;
          // both CTAs' copies count on the first one's barrier (the other's may land before it is armed: the count goes negative)
          if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * (2 * RP_HALF + (scales ? 3 * R8_TILE : 0)));
          tma_load_2d_pair(st, &map_x, bar, kb * R8_BLOCK, t0);
          tma_load_2d_pair(st + RP_HALF, &map_w, bar, kb * R8_BLOCK, n0 + rank * 128);
          if (scales) {
            tma_load_3d_pair(st + 2 * RP_HALF, &map_sx, bar, 0, kb >> 2, t0 >> 7);
            tma_load_3d_pair(st + 2 * RP_HALF + R8_TILE, &map_sw, bar, 0, kb >> 2, n0 >> 7);
          }
        }
        __syncwarp();
        ++issued;
        if (++s == RP_STAGES) s = 0, par ^= 1;
      }
    }
    if (gave_up && rank == 0)  // the copies land before the CTAs leave
      for (uint32_t i = issued > RP_STAGES ? issued - RP_STAGES : 0; i < issued; ++i) {
        int zero = 0;
        bounded_wait(&full[i % RP_STAGES], (i / RP_STAGES) & 1, &zero);
      }
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t ring = umma_desc_lo(smem_u32(smem)), sx = tmem + RP_SCALES_X, sw = tmem + RP_SCALES_W;
      uint32_t s = 0, par = 0, nth = 0;
      bool fine = true;
      for (int i = cluster; i < items && fine; i += clusters, ++nth) {
        const PairItem it = pair_item(pp, i, num_k);
        const uint32_t acc = nth & 1, d = tmem + acc * RP_SECOND;
        fine = waited(&tmem_empty[acc], ((nth >> 1) & 1) ^ 1) && (nth == 0 || waited(&overlap, (nth - 1) & 1));
        if (!fine) break;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          fine = waited(&full[s], par);
          if (!fine) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t a = ring + s * (RP_STAGE >> 4), b = a + (RP_HALF >> 4);
            if (kb == it.kb0 || (kb & 3) == 0) {
              const uint32_t src = smem_u32(smem) + s * RP_STAGE + 2 * RP_HALF;
              copy_scales_pair(sx, src);
              copy_scales_pair(sw, src + R8_TILE);
              copy_scales_pair(sw + 4, src + 2 * R8_TILE);
            }
            const uint32_t idesc = r8_idesc(RP_ROWS, RP_COLS, kb & 3);
            umma_mx8_pair(d, a, b, idesc, sx, sw, kb > it.kb0 ? 1u : 0u);
#pragma unroll
            for (int k = 1; k < 4; ++k) umma_mx8_pair(d, a + 2 * k, b + 2 * k, idesc, sx, sw, 1u);
            umma_commit_pair(&empty[s]);
            if (kb == it.kb1 - 1) umma_commit_pair(&tmem_full[acc]);
          }
          __syncwarp();
          if (++s == RP_STAGES) s = 0, par ^= 1;
        }
      }
    }
  } else {
    const int quarter = warp & 3, half = (warp - 2) >> 2, row = quarter * 32 + lane;
    uint8_t* const turn = smem + RP_STAGES * RP_STAGE + (warp - 2) * RP_TURN;
    uint32_t nth = 0;
    bool fine = true;
    for (int i = cluster; i < items; i += clusters, ++nth) {
      const PairItem it = pair_item(pp, i, num_k);
      go_to(it.tile);
      const int64_t t = (int64_t)walk.m() * RP_ROWS + rank * 128 + row;
      const int n0 = walk.n() * RP_COLS;
      const uint32_t acc = nth & 1, from = tmem + ((uint32_t)(quarter * 32) << 16) + acc * RP_SECOND;
      fine = fine && waited(&tmem_full[acc], (nth >> 1) & 1);
      tc_fence_after();
      // blocks of 32 columns 0, 1, 2, 3 or 7, 6, 5, 4: the columns that both accumulators have come first
      auto column = [&](int c) { return half ? 7 - c : c; };
      auto read = [&](int c, uint32_t(&v)[32]) {
        if (fine) {
          tmem_ld_32x32b_x32(from + 32 * column(c), v);
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0x7fffffffu;
        }
        const bool shared = c == 0 && half == (acc ? 0 : 1);
        if (shared || c == 3) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (shared) mbar_arrive_cluster(cluster_first(&overlap));
            if (c == 3) mbar_arrive_cluster(cluster_first(&tmem_empty[acc]));
          }
        }
      };
      if (it.part >= 0) {
        float4* const to = pair_part(pp, it.slot, it.part, rank, row);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          read(c, v);
#pragma unroll
          for (int q = 0; q < 8; ++q)
            to[(column(c) * 8 + q) * 128] = make_float4(__uint_as_float(v[4 * q]), __uint_as_float(v[4 * q + 1]), __uint_as_float(v[4 * q + 2]), __uint_as_float(v[4 * q + 3]));
        }
        continue;
      }
      if constexpr (OUT != R8_OUT_GATE) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          read(c, v);
          const int n = n0 + 32 * column(c);
          r8_store32<OUT>(p, turn, t - lane, n, v);
        }
      } else {
        float g[4][16];
        uint32_t amax = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t v[32];
          read(c, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            g[c][i] = silu_times(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
            amax = max(amax, r8_bits(g[c][i]));
          }
        }
        meet[acc][half][row] = amax;
        asm volatile("bar.sync %0, 64;" ::"r"(4 + quarter) : "memory");
        amax = max(amax, meet[acc][half ^ 1][row]);
        const int block = n0 / RP_COLS;
        uint4 own[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) own[half ? 3 - c : c] = r8_codes16(g[c], amax);
        r8_store_turned(turn, own, p.codes + (t - lane) * p.width + (int64_t)block * R8_BLOCK + half * 64, p.width, (int)min((int64_t)32, p.T - (t - lane)));
        if (half == 0) r8_store_unit_scale(p, t, block, num_n, amax);
      }
    }
  }
  tc_fence_before();
  cluster_sync_all();  // nobody leaves while the other's copies, commits or arrivals may reach it
  if (warp == 1) tmem_dealloc<2>(tmem, 512);
}

// The parts of cut tiles, added in the order of k, and finished: a CTA takes 32 tokens and all columns of a tile, a warp 16 columns of them, a lane a token.  All parts are requested at
// once, and results turned in shared memory: a warp writes whole rows.
constexpr int RP_JOIN_THREADS = 512;
template <int OUT>
__global__ void __launch_bounds__(RP_JOIN_THREADS) rows8_pair_join_kernel(const __grid_constant__ Pair8Params pp) {
  pdl_trigger();
  const ProductParams& p = pp.o;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, slot = (int)blockIdx.x >> 3, rank = ((int)blockIdx.x >> 2) & 1, row0 = ((int)blockIdx.x & 3) * 32;
  using O = std::conditional_t<OUT == R8_OUT_F32, float, bf16>;
  constexpr int PITCH = OUT == R8_OUT_GATE ? R8_BLOCK + 16 : RP_COLS * (int)sizeof(O) + 16;  // bytes of a token's row
  __shared__ __align__(16) uint8_t turn[32 * PITCH];
  __shared__ uint32_t meet[16][32];
  TileWalk walk;
  const int num_m = (p.T + RP_ROWS - 1) / RP_ROWS, num_n = (p.N + RP_COLS - 1) / RP_COLS;
  walk.start(num_m, num_n);
  walk.advance(pp.whole + slot, num_m, num_n);
  const int64_t t0 = (int64_t)walk.m() * RP_ROWS + rank * 128 + row0;
  const int n0 = walk.n() * RP_COLS;
  pdl_wait();
  if (t0 >= ((p.T + 127) & ~127)) return;
  float4 x[RP_MAX_CUT][4];
#pragma unroll
  for (int j = 0; j < RP_MAX_CUT; ++j) {
    const float4* from = pair_part(pp, slot, j, rank, row0 + lane) + warp * 4 * 128;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (j < pp.cut.cut) x[j][q] = from[q * 128];
  }
#pragma unroll
  for (int j = 1; j < RP_MAX_CUT; ++j)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      if (j < pp.cut.cut) x[0][q].x += x[j][q].x, x[0][q].y += x[j][q].y, x[0][q].z += x[j][q].z, x[0][q].w += x[j][q].w;
  if constexpr (OUT != R8_OUT_GATE) {
    uint4* const at = reinterpret_cast<uint4*>(turn + lane * PITCH + warp * 16 * (int)sizeof(O));
    if constexpr (OUT == R8_OUT_F32) {
#pragma unroll
      for (int q = 0; q < 4; ++q) at[q] = make_uint4(__float_as_uint(x[0][q].x), __float_as_uint(x[0][q].y), __float_as_uint(x[0][q].z), __float_as_uint(x[0][q].w));
    } else {
#pragma unroll
      for (int q = 0; q < 4; q += 2)
        at[q / 2] = make_uint4(pack2_rn(x[0][q].x, x[0][q].y), pack2_rn(x[0][q].z, x[0][q].w), pack2_rn(x[0][q + 1].x, x[0][q + 1].y), pack2_rn(x[0][q + 1].z, x[0][q + 1].w));
    }
    __syncthreads();
    const int columns = min(RP_COLS, p.N - n0);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int64_t t = t0 + 2 * warp + h;
      if (t >= p.T) return;
      const O* const from = reinterpret_cast<const O*>(turn + (2 * warp + h) * PITCH);
      O* const to = reinterpret_cast<O*>(p.out) + t * p.ld + n0;
      if (columns == RP_COLS && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
#pragma unroll
        for (int i = 0; i < (int)sizeof(O) / 2; ++i) reinterpret_cast<uint4*>(to)[i * 32 + lane] = reinterpret_cast<const uint4*>(from)[i * 32 + lane];
      } else {
        for (int i = lane; i < columns; i += 32) to[i] = from[i];
      }
    }
  } else {
    float g[8];
    uint32_t amax = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      g[2 * q] = silu_times(x[0][q].x, x[0][q].y);
      g[2 * q + 1] = silu_times(x[0][q].z, x[0][q].w);
      amax = max(amax, max(r8_bits(g[2 * q]), r8_bits(g[2 * q + 1])));
    }
    meet[warp][lane] = amax;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 16; ++j) amax = max(amax, meet[j][lane]);
    const float inverse = r8_inverse(r8_byte(amax));
    uint2 c;
    c.x = to_e4m3x2(g[0] * inverse, g[1] * inverse) | to_e4m3x2(g[2] * inverse, g[3] * inverse) << 16;
    c.y = to_e4m3x2(g[4] * inverse, g[5] * inverse) | to_e4m3x2(g[6] * inverse, g[7] * inverse) << 16;
    *reinterpret_cast<uint2*>(turn + lane * PITCH + warp * 8) = amax < 0x7f800000u ? c : make_uint2(R8_ONES, R8_ONES);
    __syncthreads();
    const int block = n0 / RP_COLS;
    if (warp == 0) r8_store_unit_scale(p, t0 + lane, block, num_n, amax);
    const int r = 2 * warp + (lane >> 4);
    if (t0 + r < p.T)
      reinterpret_cast<uint2*>(p.codes + (t0 + r) * p.width + (int64_t)block * R8_BLOCK)[lane & 15] = *reinterpret_cast<const uint2*>(turn + r * PITCH + (lane & 15) * 8);
  }
}

// ---- host ----
inline PairCut rows8_pair_cut(int64_t T, int64_t N, int64_t K, int sms) {
  return pair_cut((N + RP_COLS - 1) / RP_COLS * ((T + RP_ROWS - 1) / RP_ROWS), (int)((K + R8_BLOCK - 1) / R8_BLOCK), sms / 2);
}
// bytes of scratch
inline int64_t rows8_pair_scratch(int64_t T, int64_t N, int64_t K, int sms) {
  const PairCut c = rows8_pair_cut(T, N, K, sms);
  return c.cut > 1 ? c.rest * c.cut * RP_PART : 0;
}
template <int OUT>
int launch_rows8_pair(const ProductParams& o, const void* xc, const void* xs, const void* wc, const void* ws, void* scratch, int64_t scratch_bytes, int sms, cudaStream_t st) {
  CUtensorMap mx, mw, msx, msw;
  const int64_t width = r8_width(o.K), quads = r8_quads(o.K);
  int rc = r8_code_map(&mx, xc, o.T, width, 128);
  if (!rc) rc = r8_code_map(&mw, wc, o.N, width, 128);
  if (!rc) rc = r8_scale_map(&msx, xs, o.T, quads, 1);
  if (!rc) rc = r8_scale_map(&msw, ws, o.N, quads, 2);
  if (rc) return rc;
  const int64_t tiles = (int64_t)((o.N + RP_COLS - 1) / RP_COLS) * ((o.T + RP_ROWS - 1) / RP_ROWS), pairs = sms / 2, need = rows8_pair_scratch(o.T, o.N, o.K, sms);
  MB_CHECK_ARG(tiles < (1 << 30), "product: %lld tiles", (long long)tiles);
  MB_CHECK_ARG(need == 0 || (scratch && (uintptr_t)scratch % 16 == 0 && scratch_bytes >= need), "product: %lld bytes of scratch, %lld are needed", (long long)scratch_bytes, (long long)need);
  Pair8Params p;
  p.o = o;
  p.cut = rows8_pair_cut(o.T, o.N, o.K, sms);
  p.whole = (int)tiles - p.cut.rest;
  p.parts = reinterpret_cast<float4*>(scratch);
  MB_CHECK_CUDA(device_info::allow_shared<rows8_pair_kernel<OUT>>(RP_SMEM));
  const int64_t items = p.whole + p.cut.rest * p.cut.cut;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * (unsigned)(items < pairs ? items : pairs));
  cfg.blockDim = dim3(RP_THREADS);
  cfg.dynamicSmemBytes = RP_SMEM;
  cfg.stream = st;
  cudaLaunchAttribute a[2];
  a[0].id = cudaLaunchAttributeClusterDimension;
  a[0].val.clusterDim.x = 2;
  a[0].val.clusterDim.y = a[0].val.clusterDim.z = 1;
  a[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = a;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  MB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, rows8_pair_kernel<OUT>, mx, mw, msx, msw, p));
  if (need) MB_CHECK_CUDA(launch_pdl(rows8_pair_join_kernel<OUT>, dim3((unsigned)p.cut.rest * 8), dim3(RP_JOIN_THREADS), 0, st, p));
  return MB200_OK;
}

}  // namespace mb200
