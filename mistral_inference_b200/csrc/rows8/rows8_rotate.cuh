// Rotary positions and the cache phase behind a query, key and value product that another kernel has written: queries and keys are rotated pair by pair, as the reference does it
// (rope.py:18-23: a complex product in 32 bits of numbers rounded to 16, rounded again), and go to their own matrices, or keys and values to rows of the cache.
//
// A thread has 8 numbers, four pairs.  Latency for decode steps, memory for prompts: every number is read and written once, and a position's 512 bytes of the table once a head, out of L1 or L2.
#pragma once
#include "rows8_common.cuh"

namespace mb200 {

constexpr int RR_THREADS = 128;
struct RotateParams {
  const uint4* qkv;  // [T, (H + 2 KV) * 128]
  const float4* rope;  // [positions, 64, 2]
  const int32_t *positions, *rows;  // rows: of keys and values, -1 none; null: token t's are row t
  uint4 *q, *k, *v;
  int T, H, KV;
};
__global__ void __launch_bounds__(RR_THREADS) rows8_rotate_kernel(const RotateParams p) {
  pdl_trigger();
  pdl_wait();
  const int heads = p.H + 2 * p.KV, t = (int)blockIdx.x, i = (int)blockIdx.y * RR_THREADS + threadIdx.x;  // 16 threads a head
  if (i >= heads * 16) return;
  const int h = i >> 4, at = i & 15;
  const int64_t row = h < p.H || p.rows == nullptr ? t : p.rows[t];
  if (row < 0) return;
  uint4 x = p.qkv[(int64_t)t * heads * 16 + i];
  if (h < p.H + p.KV) {
    const float4* cs = p.rope + ((int64_t)p.positions[t] * 32 + at * 2);
    const float4 a = cs[0], b = cs[1];
    auto turned = [](uint32_t u, float c, float s) {
      float re, im;
      ref_cmul(bf16lo(u), bf16hi(u), c, s, re, im);
      return pack_bf16x2(re, im);
    };
    x = make_uint4(turned(x.x, a.x, a.y), turned(x.y, a.z, a.w), turned(x.z, b.x, b.y), turned(x.w, b.z, b.w));
  }
  uint4* const to = h < p.H ? p.q + (row * p.H + h) * 16 : h < p.H + p.KV ? p.k + (row * p.KV + h - p.H) * 16 : p.v + (row * p.KV + h - p.H - p.KV) * 16;
  to[at] = x;
}

}  // namespace mb200
