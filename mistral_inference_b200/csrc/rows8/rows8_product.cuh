// y[t, n] = sum over blocks b of 2^(ex[t, b] + ew[n, b]) sum over the block of cx[t, k] cw[n, k]: products of 8-bit rows on tcgen05.mma.kind::mxf8f6f4, which multiplies
// by both powers as it adds to the fp32 accumulator in tensor memory.
// Here: the instructions and what both kernels store.  rows8_stream.cuh: up to 128 tokens, bound by the weights' bytes; rows8_pair.cuh: prompts, bound by the tensor pipe.
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

// The instruction's descriptor: e4m3 by e4m3, scales e8m0, of which byte `block` of every four is taken (a block of 128 is four instructions with one byte)
constexpr uint32_t R8_IDESC = 1u << 23;
__device__ __forceinline__ uint32_t r8_idesc(int rows, int columns, uint32_t block) { return R8_IDESC | (uint32_t)(columns >> 3) << 17 | (uint32_t)(rows >> 4) << 24 | block << 29 | block << 4; }
// D[tmem] (+)= A[smem] * B[smem], 32 entries of K; a, b: lower words of the tiles' descriptors, sa, sb: tensor memory of their scales
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
// silu(gate) * up, at most (3 + |gate| / 3) 2^-22 of it off: 2^-22 by the exponential, 2^-23 by the reciprocal, 2^-24 by the sum and each product, and |gate| 2^-23.7 by the exponent, whose constant
// and product are rounded (it grows to 2^-17 at -87).  Below -87 silu is less than 2^-119, and 0 from where the exponential is infinite.  e4m3 keeps 2^-4.
__device__ __forceinline__ float silu_times(float gate, float up) {
  float e, r;
  asm("ex2.approx.f32 %0, %1;" : "=f"(e) : "f"(gate * -1.4426950408889634f));
  asm("rcp.approx.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return gate * r * up;
}

// A warp's 32 rows of 64 bytes to memory, lane's row in `own`: turned in `turn` (2 KB of the warp's), so that an instruction writes 8 rows of 64 bytes and not 32 of 16, which took an
// epilogue of 256 x 256 8000 clocks.  row0: the first lane's row, `rows` of them exist, ld bytes apart.
__device__ __forceinline__ void r8_store_turned(uint8_t* turn, const uint4 (&own)[4], uint8_t* row0, int64_t ld, int rows) {
  const int lane = threadIdx.x & 31;
  uint4* const t = reinterpret_cast<uint4*>(turn);
#pragma unroll
  for (int i = 0; i < 4; ++i) t[lane * 4 + (i ^ ((lane >> 1) & 3))] = own[i];  // (eight lanes' units meet no bank twice)
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 8 * i + (lane >> 2), u = lane & 3;
    const uint4 v = t[r * 4 + (u ^ ((r >> 1) & 3))];
    if (r < rows) *reinterpret_cast<uint4*>(row0 + r * ld + u * 16) = v;
  }
  __syncwarp();
}
// 32 features n .. of a warp's 32 tokens, lane's token t0 + lane.  Rows that do not begin on 16 bytes go number by number, each lane in its own row (300 tokens, 1555 features of 1003 entries: 42 us).
template <int OUT>
__device__ __forceinline__ void r8_store32(const ProductParams& p, uint8_t* turn, int64_t t0, int n, const uint32_t (&v)[32]) {
  using O = std::conditional_t<OUT == R8_OUT_F32, float, bf16>;
  const int lane = threadIdx.x & 31, rows = (int)min((int64_t)32, p.T - t0);
  O* const to = reinterpret_cast<O*>(p.out) + t0 * p.ld + n;
  if (rows <= 0 || n >= p.N) return;
  if (n + 32 <= p.N && (reinterpret_cast<uintptr_t>(to) & 15) == 0 && (rows == 1 || p.ld * sizeof(O) % 16 == 0)) {
    if constexpr (OUT == R8_OUT_F32) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        uint4 own[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) own[i] = make_uint4(v[16 * h + 4 * i], v[16 * h + 4 * i + 1], v[16 * h + 4 * i + 2], v[16 * h + 4 * i + 3]);
        r8_store_turned(turn, own, reinterpret_cast<uint8_t*>(to + 16 * h), p.ld * sizeof(O), rows);
      }
    } else {
      uint4 own[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = pack2_rn(__uint_as_float(v[8 * i + 2 * j]), __uint_as_float(v[8 * i + 2 * j + 1]));
        own[i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      r8_store_turned(turn, own, reinterpret_cast<uint8_t*>(to), p.ld * sizeof(O), rows);
    }
    return;
  }
  if (lane < rows) {
#pragma unroll
    for (int i = 0; i < 32; ++i)
      if (n + i < p.N) to[lane * p.ld + i] = (O)__uint_as_float(v[i]);
  }
}

// The power of token t's block of gated units, `blocks` of them in all; places of no token or block of the scales' tile get 1
__device__ __forceinline__ void r8_store_unit_scale(const ProductParams& p, int64_t t, int block, int blocks, uint32_t amax_bits) {
  if (t >= ((p.T + 127) & ~127)) return;
  uint8_t* sc = p.scales + r8_scale_at(t, block >> 2, p.quads);
  sc[block & 3] = (uint8_t)(t < p.T ? r8_byte(amax_bits) : 127u);
  if (block == blocks - 1)
    for (int b = (block & 3) + 1; b < 4; ++b) sc[b] = 127;
}

}  // namespace mb200
