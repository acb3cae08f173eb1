// Attention of few query rows per key/value head over a 4-bit paged cache: the decode step.
//
// A warp a row, a key after the other, in 32 bits: the running maximum m and sum l of the softmax, and O relative
// to m. Splits of a long sequence are joined by the launch that follows.
#include <type_traits>

#include "attn_dev.cuh"

namespace vq2 {
namespace {

template <typename T>
__global__ void __launch_bounds__(512) attn_decode4_kernel(const AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = blockIdx.y, h = blockIdx.z;
  const int b = blockIdx.x / a.row_blocks, rb = blockIdx.x - b * a.row_blocks;
  const AttnRows w = attn_rows(a, b, rb);
  blank_strays(a, w, b, ((int64_t)rb * a.kv.heads + h) * a.splits + split, (int64_t)a.row_blocks * a.kv.heads * a.splits);
  if (warp >= w.rows) return;
  int lo, hi;
  block_keys(a, w, lo, hi);
  if (split > 0 && (int64_t)split * a.chunk >= hi - lo) return;
  const int s0 = lo + split * a.chunk, s1 = s0 + min(a.chunk, hi - s0);
  const int r = w.r0 + warp, tok = r / a.G, head = h * a.G + r % a.G;
  const int k0 = max(s0, row_lo(a, w, tok)), k1 = min(s1, row_hi(a, w, tok));
  const int d0 = 8 * lane;   // this lane's 8 values
  const bool mine = d0 < a.D;
  const Scale4 places(a.D);
  const uint8_t *ks = reinterpret_cast<const uint8_t*>(a.kv.k_scale), *vs = reinterpret_cast<const uint8_t*>(a.kv.v_scale);
  float q[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    o[j] = 0.f;
    q[j] = mine ? to_f32<T>(static_cast<const T*>(a.q)[(int64_t)(w.first + tok) * a.q_ts + head * a.q_hs + d0 + j]) : 0.f;
  }
  for (int k = k0; k < k1; ++k) {
    const int64_t slot = slot_of(a.kv, b, k);
    if (slot < 0) continue;
    const int64_t row = pool_row(a.kv, slot, h), at = row * (a.D >> 1) + (d0 >> 1);
    float s = 0.f, v_step = 0.f;
    uint32_t kw = 0, vw = 0;
    if (mine) {
      kw = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.kv.k) + at);
      vw = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.kv.v) + at);
#pragma unroll
      for (int j = 0; j < 8; ++j) s += q[j] * (float)((int)(kw >> (4 * j) & 15) - 8);
      s *= e4m3_value(ks[places.factor(row, d0 >> 6)]);
      v_step = e4m3_value(vs[places.factor(row, d0 >> 6)]) * *reinterpret_cast<const float*>(vs + places.row(row));
    }
#pragma unroll
    for (int i = 16; i; i >>= 1) s += __shfl_xor_sync(0xffffffffu, s, i);
    s *= *reinterpret_cast<const float*>(ks + places.row(row)) * a.scale_log2;
    const float mn = fmaxf(m, s), by = m == -INFINITY ? 0.f : ex2(m - mn), p = ex2(s - mn);
    m = mn;
    l = l * by + p;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = o[j] * by + p * v_step * (float)((int)(vw >> (4 * j) & 15) - 8);
  }
  const int64_t at = (int64_t)(w.first + tok) * a.hq + head;
  if (hi - lo <= a.chunk) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
    if (mine) {
#pragma unroll
      for (int j = 0; j < 8; ++j) static_cast<T*>(a.out)[at * a.D + d0 + j] = from_f32<T>(o[j] * inv);
    }
    if (a.lse && lane == 0) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
  } else {
    if (mine) {
#pragma unroll
      for (int j = 0; j < 8; ++j) a.part_o[(at * a.splits + split) * a.D + d0 + j] = o[j];
    }
    if (lane == 0) a.part_ml[at * a.splits + split] = make_float2(m, l);
  }
}

}  // namespace

void plan_attn_decode4(AttnArgs& a, int64_t max_new, int64_t max_len) { plan_attn_decode(a, max_new, max_len); }

int launch_attn_decode4(const AttnArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)(a.kv.seqs * a.row_blocks), (unsigned)a.splits, (unsigned)a.kv.heads), block(a.rows_per_block * 32);
  return a.q_bf16 ? launch_kernel(attn_decode4_kernel<__nv_bfloat16>, grid, block, 0, st, a)
                  : launch_kernel(attn_decode4_kernel<__half>, grid, block, 0, st, a);
}

}  // namespace vq2
