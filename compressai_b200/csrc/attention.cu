// Attention of new tokens over a paged key/value cache.
//
//   o[t, h] = sum_l softmax_l(scale * q[t, h] . k[l, h / G]) v[l, h / G]
//
// over the keys l of t's sequence that t sees: l < len, l <= position(t) when causal, l >
// position(t) - window when there is a window. A row that sees no key is zero (lse -inf).
//
// One warp per (token, query head), one pass over the keys with the running maximum and sum of the
// softmax, all sums in 32 bits.
#include "kv_dev.cuh"

namespace vq2 {
namespace {

struct AttnArgs {
  PagedKV kv;
  const void* q;
  int64_t q_ts, q_hs;
  int T, hq, D;
  float scale;
  int causal, window;
  void* out;
  float* lse;
};

template <typename T, bool I8>
__global__ void __launch_bounds__(128) attn_simple_kernel(const AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x, lane = threadIdx.x & 31;
  const int b = sequence_of(a.kv, t);
  const int h = blockIdx.y * 4 + (threadIdx.x >> 5);
  if (h >= a.hq) return;
  const int hk = h / (a.hq / a.kv.heads);
  float q[8], o[8], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = lane + 32 * i;
    q[i] = e < a.D ? to_f32<T>(static_cast<const T*>(a.q)[t * a.q_ts + h * a.q_hs + e]) : 0.f;
    o[i] = 0.f;
  }
  if (b >= 0) {
    int first, count;
    sequence_rows(a.kv, b, first, count);
    const int len = length_of(a.kv, b), pos = len - count + (t - first);
    const int hi = a.causal ? min(len, pos + 1) : len;
    const int lo = a.window ? max(0, pos - a.window + 1) : 0;
    for (int p = lo; p < hi; ++p) {
      const int64_t slot = slot_of(a.kv, b, p);
      if (slot < 0) continue;
      const int64_t row = pool_row(a.kv, slot, hk);
      float s = 0.f, v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int e = lane + 32 * i;
        v[i] = 0.f;
        if (e < a.D) {
          if (I8) {
            s += q[i] * (float)static_cast<const int8_t*>(a.kv.k)[row * a.D + e];
            v[i] = (float)static_cast<const int8_t*>(a.kv.v)[row * a.D + e] * a.kv.v_scale[row];
          } else {
            s += q[i] * to_f32<T>(static_cast<const T*>(a.kv.k)[row * a.D + e]);
            v[i] = to_f32<T>(static_cast<const T*>(a.kv.v)[row * a.D + e]);
          }
        }
      }
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
      s *= a.scale * (I8 ? a.kv.k_scale[row] : 1.f);
      const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
      const float f = expf(m - base), w = expf(s - base);
      l = l * f + w;
#pragma unroll
      for (int i = 0; i < 8; ++i) o[i] = o[i] * f + w * v[i];
      m = mn;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = lane + 32 * i;
    if (e < a.D)
      static_cast<T*>(a.out)[((int64_t)t * a.hq + h) * a.D + e] = from_f32<T>(l == 0.f ? 0.f : o[i] / l);
  }
  if (a.lse && lane == 0) a.lse[(int64_t)t * a.hq + h] = l == 0.f ? -INFINITY : m + logf(l);
}

template <typename T>
int run(const AttnArgs& a, bool i8, cudaStream_t st) {
  const dim3 grid((unsigned)a.T, (unsigned)((a.hq + 3) / 4)), block(128);
  return i8 ? launch_kernel(attn_simple_kernel<T, true>, grid, block, 0, st, a)
            : launch_kernel(attn_simple_kernel<T, false>, grid, block, 0, st, a);
}

}  // namespace
}  // namespace vq2

using namespace vq2;

extern "C" int64_t vq2_paged_attention_workspace(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_size,
                                                 int64_t seqs, int64_t max_new, int64_t max_len, int causal,
                                                 int64_t window) {
  return 0;
}

extern "C" int vq2_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype,
                                   int64_t tokens, int64_t q_heads, const void* k_pages, const void* v_pages,
                                   int kv_dtype, const float* k_scale, const float* v_scale, int64_t pages,
                                   int64_t kv_heads, int64_t page_size, int64_t head_size, const int32_t* table,
                                   int64_t table_stride, int64_t table_cols, const int32_t* lens, const int32_t* starts,
                                   int64_t seqs, int64_t max_new, int64_t max_len, float scale, int causal,
                                   int64_t window, void* out, float* lse, void* ws, int64_t ws_bytes, void* stream) {
  AttnArgs a = {};
  int s = paged_kv(a.kv, k_pages, v_pages, kv_dtype, k_scale, v_scale, pages, kv_heads, page_size, head_size, table,
                   table_stride, table_cols, lens, starts, seqs);
  if (s != VQ2_OK) return s;
  if (!q || !out || !lens) return VQ2_ERR_ARG;
  if ((dtype != VQ2_F16 && dtype != VQ2_BF16) || (kv_dtype != dtype && kv_dtype != VQ2_I8)) return VQ2_ERR_DTYPE;
  if (tokens < 0 || tokens > 0x7fffffff || q_heads < 1 || q_heads > 4096 || q_heads % kv_heads || max_new < 0 ||
      max_len < 0 || window < 0 || window > 0x7fffffff || (!starts && tokens != seqs))
    return VQ2_ERR_SHAPE;
  if (!aligned(q, 16) || q_token_stride % 8 || q_head_stride % 8 || !aligned(out, 16)) return VQ2_ERR_ALIGN;
  if (tokens == 0) return VQ2_OK;
  a.q = q;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.T = (int)tokens;
  a.hq = (int)q_heads;
  a.D = (int)head_size;
  a.scale = scale;
  a.causal = causal;
  a.window = (int)window;
  a.out = out;
  a.lse = lse;
  (void)ws;
  (void)ws_bytes;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool i8 = kv_dtype == VQ2_I8;
  return dtype == VQ2_F16 ? run<__half>(a, i8, st) : run<__nv_bfloat16>(a, i8, st);
}
