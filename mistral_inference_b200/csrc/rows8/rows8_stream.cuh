// Products of 8-bit rows for a few tokens (up to 128): every weight byte is read once, so HBM bounds it, and for small matrices the latency of a launch.
//
// The weights are the MMA's 128 rows, the tokens its columns (16, 32, 64 or 128).  A cluster of `split` CTAs computes 128 features, each CTA a range of k-blocks.  Each sends its fp32 sums to the
// CTA that finishes them (the r-th takes the r-th part of the features), which adds them in the order of k: the same bits in every run.  What is sent lies over the ring,
// behind a meeting of the cluster at the end of its MMAs, or for up to 32 tokens beside the ring, without that meeting (0.8 us).
// Why not fewer features a CTA and all of K: an MMA takes 52 clocks however narrow it is, and a CTA of 40 features gets 1.3 KB of weights into one, no more than its share of what memory delivers
// (32 tokens 5120 x 14336: 23 us between the first block and the last, now 9); and the scales of rows that do not begin with a tile had to be gathered (4 to 8 us).
// Weights that are fixed (the caller says that nobody writes them any more) are requested before the wait for the predecessor, tokens after it; others are asked into L2 before it,
// where whatever is still written to them arrives as well (us, 1 token: 6144 x 4096 8.5 without, 8.1 with, 4096 x 14336 13.8, 13.0; fixed 7.4, 12.6).
//
// Gated units: their power is that of 128 units, 256 features, so a cluster holds two such groups; its CTAs exchange their tokens' largest magnitudes.  Units are laid out by tokens in
// shared memory, so that a thread has 16 of a token's next to one another.
#pragma once
#include "rows8_product.cuh"

namespace mb200 {

constexpr int RS_MAX_T = 128, RS_THREADS = 192, RS_MAX_STAGES = 12, RS_MAX_SPLIT = 8;
constexpr int RS_W = 128 * R8_BLOCK;  // a k-block of the weights
// columns c .. c + 15 of this warp's lanes
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                 "=r"(v[14]), "=r"(v[15])
               : "r"(taddr));
  tmem_wait_ld();
}
// *p = max(*p, v) in the shared memory of the cluster's CTA `rank`
__device__ __forceinline__ void max_in_cluster(uint32_t* p, int rank, uint32_t v) {
  asm volatile(
      "{\n"
      ".reg .b32 a;\n"
      "mapa.shared::cluster.u32 a, %0, %1;\n"
      "red.relaxed.cluster.shared::cluster.max.u32 [a], %2;\n"
      "}\n" ::"r"(smem_u32(p)),
      "r"(rank), "r"(v)
      : "memory");
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

MB_HD constexpr int R8_UNITS_PITCH(int units) { return units + 4; }  // floats of a token's units
struct StreamParams {
  ProductParams o;
  int split;    // CTAs of 128 features
  int stages, stage_bytes, x_bytes;  // of the ring: weights, tokens, the scales of both
  int share;    // features that a CTA finishes
  int pitch;    // floats of a feature: T rounded up to 16, and 4 so that lanes' 16 bytes meet no bank twice
  int sums_at;  // what the cluster's CTAs send, in shared memory: 0, over the ring, or behind it
  int units_at; // gated units there, behind what was sent
  int ahead;    // the weights are fixed
};

template <int OUT, int COLS>
__global__ void __launch_bounds__(RS_THREADS) rows8_stream_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_sx,
                                                                  const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ StreamParams p) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  float* sums = reinterpret_cast<float*>(smem + p.sums_at);  // [split][share][pitch]: what the cluster's CTAs send this one, a feature's tokens side by side
  __shared__ uint64_t full[RS_MAX_STAGES], empty[RS_MAX_STAGES], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int gave_up;
  __shared__ uint32_t most[RS_MAX_T];  // largest magnitudes of the tokens' units in the cluster
  constexpr uint32_t TMEM = COLS * 2, SW = COLS, SX = COLS + 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tile = (int)blockIdx.x / p.split, part = (int)blockIdx.x % p.split;
  const int num_k = (p.o.K + R8_BLOCK - 1) / R8_BLOCK, kb0 = num_k * part / p.split, kb1 = num_k * (part + 1) / p.split;
  constexpr bool GATE = OUT == R8_OUT_GATE;
  const bool sends = p.split > 1, over = p.sums_at == 0;
  const int meetings = sends ? (GATE ? 3 : 2) : (GATE ? 2 : 0);  // of the cluster's threads: all may write, sums are there, magnitudes are there
  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    mbar_init(&done, 1);
    gave_up = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (GATE && threadIdx.x >= 64) most[threadIdx.x - 64] = 0;
  if (warp == 1) tmem_alloc(&tmem_slot, TMEM);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  if (meetings > 0 && !(sends && over)) cluster_arrive();  // this CTA has begun: others may write to it
  pdl_trigger();
  if (!p.ahead) {
    if (warp == 0 && elect_one())
      for (int kb = kb0; kb < min(kb1, kb0 + p.stages); ++kb)
        asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global [%0, {%1, %2}];" ::"l"(&map_w), "r"(kb * R8_BLOCK), "r"(tile * 128) : "memory");
    __syncwarp();
    pdl_wait();
  }

  if (warp == 0) {
    // ================= copies =================
    const uint32_t x_at = RS_W, sw_at = x_at + (uint32_t)p.x_bytes, sx_at = sw_at + R8_TILE;
    const int steps = kb1 - kb0, head = min(steps, p.stages);
    auto scaled = [&](int it) { return it == 0 || ((kb0 + it) & 3) == 0; };
    auto weights = [&](int it, int s) {
      const int kb = kb0 + it;
      uint8_t* st = smem + s * p.stage_bytes;
      mbar_arrive_expect_tx(&full[s], RS_W + (uint32_t)p.x_bytes + (scaled(it) ? 2 * R8_TILE : 0));
      tma_load_2d(st, &map_w, &full[s], kb * R8_BLOCK, tile * 128);
      if (scaled(it)) tma_load_3d(st + sw_at, &map_sw, &full[s], 0, kb >> 2, tile);
    };
    auto tokens = [&](int it, int s) {
      const int kb = kb0 + it;
      uint8_t* st = smem + s * p.stage_bytes;
      tma_load_2d(st + x_at, &map_x, &full[s], kb * R8_BLOCK, 0);
      if (scaled(it)) tma_load_3d(st + sx_at, &map_sx, &full[s], 0, kb >> 2, 0);
    };
    if (elect_one())
      for (int it = 0; it < head; ++it) weights(it, it);
    pdl_wait();
    if (elect_one())
      for (int it = 0; it < head; ++it) tokens(it, it);
    int s = 0, par = 0, issued = head;
    for (int it = head; it < steps; ++it) {
      if (!__all_sync(0xffffffffu, bounded_wait(&empty[s], par, &gave_up))) break;
      if (elect_one()) {
        weights(it, s);
        tokens(it, s);
      }
      __syncwarp();
      issued = it + 1;
      if (++s == p.stages) s = 0, par ^= 1;
    }
    if (gave_up)  // the copies land before the CTA leaves
      for (int i = issued > p.stages ? issued - p.stages : 0; i < issued; ++i) {
        int zero = 0;
        bounded_wait(&full[i % p.stages], (i / p.stages) & 1, &zero);
      }
  } else if (warp == 1) {
    // ================= MMAs =================
    pdl_wait();  // (the tokens come behind it: the waits' limits count from there)
    const uint32_t base = smem_u32(smem);
    int s = 0, par = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!__all_sync(0xffffffffu, bounded_wait(&full[s], par, &gave_up))) break;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t at = base + s * p.stage_bytes, w = umma_desc_lo(at), x = w + (RS_W >> 4);
        if (kb == kb0 || (kb & 3) == 0) {
          copy_scales(tmem + SW, at + RS_W + p.x_bytes);
          copy_scales(tmem + SX, at + RS_W + p.x_bytes + R8_TILE);
        }
        const uint32_t idesc = r8_idesc(128, COLS, kb & 3);
#pragma unroll
        for (int k = 0; k < 4; ++k) umma_mx8(tmem, w + 2 * k, x + 2 * k, idesc, tmem + SW, tmem + SX, (kb > kb0 || k > 0) ? 1u : 0u);
        umma_commit(&empty[s]);
        if (kb == kb1 - 1) umma_commit(&done);
      }
      __syncwarp();
      if (++s == p.stages) s = 0, par ^= 1;
    }
  } else {
    // ================= epilogue: TMEM lanes (features) 32 * (warp % 4) .. + 31 =================
    pdl_wait();  // (what is written here may still be read by the predecessor)
    const bool fine = __all_sync(0xffffffffu, bounded_wait(&done, 0, &gave_up)) != 0;
    tc_fence_after();
    const int f = (warp & 3) * 32 + lane, T = p.o.T, id = threadIdx.x - 64;
    const int owner = f / p.share, mine = min(p.share, 128 - part * p.share);  // features that this CTA finishes
    const uint32_t from = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    using O = std::conditional_t<OUT == R8_OUT_F32, float, bf16>;
    uint32_t to = smem_u32(sums + (size_t)(part * p.share + f % p.share) * p.pitch);
    if (sends) {
      if (over) cluster_arrive();  // this CTA's ring is free: its MMAs have read it
      cluster_wait();
      const int rank = GATE ? (tile & 1) * p.split + owner : owner;
      asm volatile("mapa.shared::cluster.u32 %0, %0, %1;" : "+r"(to) : "r"(rank));
    } else if (GATE) {
      cluster_wait();
    }
    O* const out = reinterpret_cast<O*>(p.o.out) + (int64_t)tile * 128 + f;
    const bool there = tile * 128 + f < p.o.N;
#pragma unroll 1
    for (int c = 0; c < T; c += 16) {
      uint32_t v[16];
      if (fine) {
        tmem_ld16(from + c, v);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0x7fffffffu;
      }
      if (sends) {
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          if (c + i < T)
            asm volatile("st.shared::cluster.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(to + (c + i) * 4), "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3]) : "memory");
      } else if (GATE) {  // lanes 2 i and 2 i + 1 have a unit's gate and up: the even one takes the first eight tokens, the odd one the others
        const bool odd = lane & 1;
        float* const at = reinterpret_cast<float*>(smem + p.units_at) + (c + (odd ? 8 : 0)) * R8_UNITS_PITCH(64) + (f >> 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float own = __uint_as_float(odd ? v[i + 8] : v[i]), other = __uint_as_float(__shfl_xor_sync(0xffffffffu, odd ? v[i] : v[i + 8], 1));
          const float g = silu_times(odd ? other : own, odd ? own : other);
          if (c + i + (odd ? 8 : 0) < T) at[i * R8_UNITS_PITCH(64)] = g;
        }
      } else if (there) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (c + i < T) out[(int64_t)(c + i) * p.o.ld] = (O)__uint_as_float(v[i]);
      }
    }
    if (sends) {
      __syncwarp();
      cluster_arrive();
      cluster_wait();
    }
    if (sends || GATE) {
      const int n0 = tile * 128 + part * p.share;  // the first feature that this CTA finishes
      auto total = [&](int i, int q) {             // of the CTA's feature i and tokens 4 q .. 4 q + 3
        const float4* at = reinterpret_cast<const float4*>(sums + (size_t)i * p.pitch) + q;
        const int step = p.share * p.pitch / 4;
        float4 x[RS_MAX_SPLIT];
        constexpr int MOST = GATE ? RS_MAX_SPLIT / 2 : RS_MAX_SPLIT;
#pragma unroll
        for (int j = 0; j < MOST; ++j) x[j] = j < p.split ? at[j * step] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 1; j < MOST; ++j)
          if (j < p.split) x[0].x += x[j].x, x[0].y += x[j].y, x[0].z += x[j].z, x[0].w += x[j].w;
        return x[0];
      };
      // a feature (or unit) a lane, so that a token's results are side by side
      const int per = GATE ? mine / 2 : mine, lanes = per <= 16 ? 16 : 32, groups = 128 / lanes, quads = (T + 3) / 4;
      if constexpr (!GATE) {
        for (int q = id / lanes; q < quads; q += groups)
          for (int i = id % lanes; i < per; i += lanes) {
            if (n0 + i >= p.o.N) break;
            const float4 v = total(i, q);
            O* const at = reinterpret_cast<O*>(p.o.out) + (int64_t)(4 * q) * p.o.ld + n0 + i;
            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (4 * q + j < T) at[j * p.o.ld] = (O)x[j];
          }
      } else {
        const int block = tile >> 1, pitch = R8_UNITS_PITCH(per);  // (64, 32 or 16 units)
        float* const units = reinterpret_cast<float*>(smem + p.units_at);
        for (int q = sends ? id / lanes : quads; q < quads; q += groups)
          for (int u = id % lanes; u < per; u += lanes) {
            const float4 x = total(2 * u, q), y = total(2 * u + 1, q);
            float* const at = units + 4 * q * pitch + u;
            at[0] = silu_times(x.x, y.x), at[pitch] = silu_times(x.y, y.y), at[2 * pitch] = silu_times(x.z, y.z), at[3 * pitch] = silu_times(x.w, y.w);
          }
        __syncwarp();
        asm volatile("bar.sync 2, 128;" ::: "memory");
        const int threads = per / 16, step = 128 / threads, k = id % threads;  // threads of a token, tokens at a time
        auto sixteen = [&](int t, float(&g)[16]) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 v = reinterpret_cast<const float4*>(units + t * pitch + 16 * k)[i];
            g[4 * i] = v.x, g[4 * i + 1] = v.y, g[4 * i + 2] = v.z, g[4 * i + 3] = v.w;
          }
        };
        for (int t = id / threads; t < T; t += step) {
          float g[16];
          sixteen(t, g);
          uint32_t a = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) a = max(a, r8_bits(g[i]));
          for (int r = 0; r < 2 * p.split; ++r) max_in_cluster(&most[t], r, a);
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        for (int t = id / threads; t < T; t += step) {
          float g[16];
          sixteen(t, g);
          const uint32_t a = most[t];
          *reinterpret_cast<uint4*>(p.o.codes + (int64_t)t * p.o.width + n0 / 2 + 16 * k) = r8_codes16(g, a);
        }
        if (part == 0 && !(tile & 1)) r8_store_unit_scale(p.o, id, block, (p.o.N + 255) / 256, id < T ? most[id] : 0);  // a row of the scales' tile a thread
      }
    }
  }
  if (warp < 2) {  // the meetings above are all the cluster's threads'
    __syncwarp();
    for (int i = 0; i < meetings; ++i) {
      if (i > 0 || (sends && over)) cluster_arrive();
      cluster_wait();
    }
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) tmem_dealloc(tmem, TMEM);
}

// ---- host ----
constexpr int RS_SMEM = 225 * 1024;  // (beside what the kernel names)
constexpr int RS_SMEM_TWO = 110 * 1024;  // two CTAs an SM
// The least a CTA asks for, by columns of tensor memory: 228 KB an SM end before its 512 columns do.  An SM takes CTAs by shared memory alone, and one that found no columns would wait for those of other
// clusters, whose own CTAs may wait for its cluster's on another SM (gated units of 128 tokens with few k-blocks, or products on several streams).
constexpr int RS_SMEM_COLUMN = 430;
static_assert(RS_SMEM_COLUMN * (512 + 32) > 228 * 1024 && RS_SMEM_COLUMN * 2 * RS_MAX_T <= RS_SMEM_TWO, "columns come in multiples of 32");
inline int rs_larger(int a, int b) { return a > b ? a : b; }
inline int rs_up(int n, int step) { return (n + step - 1) / step * step; }
// CTAs that run at once.  A cluster lies within one GPC, so they are fewer than the SMs hold; of 148 SMs, by the CTAs of a cluster: two an SM 6 270, 7 259, 8 264 (of 288 in clusters of six some
// began when others had ended); one an SM 2 148, 4 132, 5 130, 7 105, 8 120 (gated units of 4000 x 4096, 1 token, 128 CTAs in clusters of eight: 15.1 us one an SM, two an SM 8.4)
inline int rs_two(int sms) { return 7 * sms / 4; }
inline int rs_one(int cluster, int sms) { return cluster > 6 ? 7 * sms / 10 : cluster > 2 ? 7 * sms / 8 : sms; }
// CTAs of 128 features: as many as let all CTAs run at once, two an SM.  us of a call with cold weights by CTAs of 128 features, 1 token 6144 x 4096: 1 11.5, 2 9.1, 4 7.1, 5 7.4, 6 10.8;
// 4096 x 14336: 1 35, 2 20, 4 14.4, 6 13.1, 8 12.6; 32 tokens 5120 x 14336: 4 17.9, 5 16.9, 6 16.5, 8 22.5; 8 tokens 32000 x 4096: 1 23.2, 2 28.3.  With more tokens what the CTAs send counts for
// more, and one CTA an SM is better: always from 65 on (128 tokens 4096 x 2048: 8 21.3, 4 11.3; 5120 x 5120: 6 18.6, 3 17.1; 5120 x 14336: 6 25.9, 3 25.7; 1024 x 4096: 8 9.8, 4 11.5), from 33 on if
// one an SM uses nearly all SMs (64 tokens 4096 x 4096: 8 12.8, 4 10.5; but 5120 x 14336: 6 19.5, 3 21.1).  For gated units a power of two, so that a CTA finishes a multiple of 16 of them.
inline int rows8_stream_split(int64_t T, int64_t tiles, int64_t K, bool gate, int sms) {
  const int64_t blocks = (K + 127) / 128, most = blocks < RS_MAX_SPLIT ? blocks : RS_MAX_SPLIT;
  int two = 1, one = 1;
  for (int s = 2; s <= (gate && most > 4 ? 4 : most); s += gate ? s : 1) {
    if (tiles * s <= rs_two(sms)) two = s;
    if (tiles * s <= rs_one(gate ? 2 * s : s, sms)) one = s;
  }
  return T > 64 || (T > 32 && tiles * one >= 17 * sms / 20) ? one : two;
}
inline int64_t rows8_stream_tiles(int64_t N, bool gate) { return gate ? (N + 255) / 256 * 2 : (N + 127) / 128; }
// Sizes of a launch, and its dynamic shared memory
inline size_t rows8_stream_layout(StreamParams& s, int64_t T, int64_t N, int64_t K, bool gate, int sms) {
  const int64_t tiles = rows8_stream_tiles(N, gate);
  s.split = rows8_stream_split(T, tiles, K, gate, sms);
  s.share = (128 + s.split - 1) / s.split;
  s.pitch = (int)((T + 15) / 16 * 16 + 4);
  const int cols = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
  s.x_bytes = cols * R8_BLOCK;
  s.stage_bytes = RS_W + s.x_bytes + 2 * R8_TILE;
  const int64_t ctas = tiles * s.split, blocks = ((K + 127) / 128 + s.split - 1) / s.split;
  const int sums = s.split > 1 ? s.split * s.share * s.pitch * 4 : 0, units = gate ? rs_up((int)T, 4) * R8_UNITS_PITCH(s.share / 2) * 4 : 0;
  const int beside = T <= 32 ? sums + units : 0, room = (ctas <= rs_one(gate ? 2 * s.split : s.split, sms) ? RS_SMEM : RS_SMEM_TWO) - 1024 - beside;
  s.stages = room / s.stage_bytes;
  if (s.stages > RS_MAX_STAGES) s.stages = RS_MAX_STAGES;
  if (s.stages > blocks) s.stages = (int)blocks;
  const int ring = s.stages * s.stage_bytes;
  s.sums_at = beside > 0 ? ring : 0;
  s.units_at = s.sums_at + sums;
  const int end = s.units_at + units, least = 2 * cols * RS_SMEM_COLUMN;
  return (size_t)rs_up(rs_larger(rs_larger(ring, end) + 1024, least), 16);
}

template <int OUT, int COLS>
int launch_rows8_stream(const ProductParams& o, const void* xc, const void* xs, const void* wc, const void* ws, bool fixed, int sms, cudaStream_t st) {
  constexpr bool GATE = OUT == R8_OUT_GATE;
  StreamParams p;
  p.o = o;
  p.ahead = fixed;
  const size_t smem = rows8_stream_layout(p, o.T, o.N, o.K, GATE, sms);
  CUtensorMap mx, mw, msx, msw;
  const int64_t width = r8_width(o.K), quads = r8_quads(o.K);
  int rc = r8_code_map(&mx, xc, o.T, width, COLS);
  if (!rc) rc = r8_code_map(&mw, wc, o.N, width, 128);
  if (!rc) rc = r8_scale_map(&msx, xs, o.T, quads, 1);
  if (!rc) rc = r8_scale_map(&msw, ws, o.N, quads, 1);
  if (rc) return rc;
  MB_CHECK_CUDA((device_info::allow_shared<rows8_stream_kernel<OUT, COLS>>(RS_SMEM)));
  const int64_t tiles = rows8_stream_tiles(o.N, GATE);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(tiles * p.split));
  cfg.blockDim = dim3(RS_THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute a[2];
  int n = 0;
  if (pdl_enabled()) {
    a[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    a[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (GATE || p.split > 1) {
    a[n].id = cudaLaunchAttributeClusterDimension;
    a[n].val.clusterDim.x = (unsigned)(GATE ? 2 * p.split : p.split);
    a[n].val.clusterDim.y = a[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = a;
  cfg.numAttrs = n;
  MB_CHECK_CUDA(cudaLaunchKernelEx(&cfg, rows8_stream_kernel<OUT, COLS>, mx, mw, msx, msw, p));
  return MB200_OK;
}
template <int OUT>
int launch_rows8_stream(const ProductParams& o, const void* xc, const void* xs, const void* wc, const void* ws, bool fixed, int sms, cudaStream_t st) {
  return o.T <= 16   ? launch_rows8_stream<OUT, 16>(o, xc, xs, wc, ws, fixed, sms, st)
         : o.T <= 32 ? launch_rows8_stream<OUT, 32>(o, xc, xs, wc, ws, fixed, sms, st)
         : o.T <= 64 ? launch_rows8_stream<OUT, 64>(o, xc, xs, wc, ws, fixed, sms, st)
                     : launch_rows8_stream<OUT, 128>(o, xc, xs, wc, ws, fixed, sms, st);
}

}  // namespace mb200
