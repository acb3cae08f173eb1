// Attention of new tokens over a paged key/value cache: checks, plan and launches.
//
//   o[t, h] = sum_l softmax_l(scale * q[t, h] . k[l, h / G]) v[l, h / G]
//
// over the keys l of t's sequence that t sees: l < len, l <= position(t) when causal, l >
// position(t) - window when there is a window. A row that sees no key, and one of no sequence, is zero (lse -inf).
#include "attn_dev.cuh"

namespace vq2 {
namespace {

// Which kernel, the splits of the keys and the workspace they and a widened 8-bit cache take: a function
// of shapes and bounds alone. Points into `ws` where it is given; returns its bytes.
int64_t plan(AttnArgs& a, int bits, int64_t max_new, int64_t max_len, bool& chunked, char* ws) {
  // Rows that share a key: the decode kernel holds 16 and would read the keys again for more; from there
  // on the tensor-core kernel takes over (16 sequences of 4000 tokens, 32/8 heads of 128: 16 rows 60 us
  // here, 20 to 40 rows 63 us there; 32 rows here took 100). Over an 8-bit cache, which it has to widen
  // first, from 49 rows on (the same, 32 rows: 96 us here, 156 there; 16/2 heads of 256: 63 and 88); over a 4-bit
  // one, half as many bytes to read again, from 97 on (64 rows: 100 us here, 133 there; 16/2 heads of 256 55 and 77; 96 rows 143
  // and 134, 71 and 76; 128 rows, of an earlier version here, 180 and 135, 93 and 77). Its
  // fp16 copy of such a cache is kept to 4 GB; past that (a batch of very long sequences) the decode
  // kernel reads the 8 bits again after all.
  // A bound of 0 leaves it one tile: a launch of no blocks is an error.
  const int64_t wide_len = max_len ? (max_len + 127) & ~int64_t(127) : 128, wide_rows = a.kv.seqs * (int64_t)a.kv.heads * wide_len;
  chunked = max_new * a.G > (bits == 4 ? 96 : bits == 8 ? 48 : 16) && (bits == 16 || wide_rows * a.D <= int64_t(1) << 30);
  if (chunked) plan_attn_chunk(a, max_new, max_len);
  else if (bits == 4) plan_attn_decode4(a, max_new, max_len);
  else plan_attn_decode(a, max_new, max_len);
  a.keys_end = 0x7fffffff;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    char* p = ws ? ws + at : nullptr;
    at += (bytes + 255) & ~int64_t(255);
    return p;
  };
  if (a.splits > 1) {
    a.part_o = reinterpret_cast<float*>(take((int64_t)a.T * a.hq * a.splits * a.D * 4));
    a.part_ml = reinterpret_cast<float2*>(take((int64_t)a.T * a.hq * a.splits * 8));
  }
  if (!chunked && bits == 4) {
    a.segments = reinterpret_cast<int2*>(take((int64_t)a.kv.seqs * a.row_blocks * a.kv.heads * 8));
    if (a.whole != 0x7fffffff) {
      a.part_o = reinterpret_cast<float*>(take((int64_t)a.blocks * 2 * a.rows_per_block * a.D * 4));
      a.part_ml = reinterpret_cast<float2*>(take((int64_t)a.blocks * 2 * a.rows_per_block * 8));
    }
  }
  if (chunked && bits < 16) {
    a.wide_len = a.keys_end = (int)wide_len;
    a.wide_k = take(wide_rows * a.D * 2);
    a.wide_v = take(wide_rows * a.D * 2);
    a.wide_ks = reinterpret_cast<float*>(take(wide_rows * 4));
    a.wide_vs = reinterpret_cast<float*>(take(wide_rows * 4));
  }
  return at;
}

// No sequence at all: every token is one of none.
__global__ void __launch_bounds__(256) attn_blank_kernel(const AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  blank_tokens(a, 0, a.T, blockIdx.x, gridDim.x);
}

int bits_of(int kv_dtype) { return kv_dtype == VQ2_I4 ? 4 : kv_dtype == VQ2_I8 ? 8 : 16; }

bool bad_attn(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t seqs, int64_t max_new, int64_t max_len,
              int64_t window) {
  return tokens < 0 || tokens > 0x7fffffff || q_heads < 1 || q_heads > 4096 || kv_heads < 1 || q_heads % kv_heads ||
         seqs < 0 || max_new < 0 || max_new > 0x7fffffff || max_len < 0 || max_len > 0x7fffff00 || window < 0 ||
         window > 0x7fffffff || max_new * (q_heads / kv_heads) > 0x7fffff00;
}

}  // namespace
}  // namespace vq2

using namespace vq2;

extern "C" int64_t vq2_paged_attention_workspace(int64_t tokens, int64_t q_heads, int64_t kv_heads, int64_t head_size,
                                                 int kv_dtype, int64_t seqs, int64_t max_new, int64_t max_len,
                                                 int64_t window) {
  if (bad_attn(tokens, q_heads, kv_heads, seqs, max_new, max_len, window) || bad_head_size(head_size)) return 0;
  AttnArgs a = {};
  a.T = (int)tokens;
  a.hq = (int)q_heads;
  a.kv.heads = (int)kv_heads;
  a.kv.seqs = (int)seqs;
  a.D = (int)head_size;
  a.G = a.hq / a.kv.heads;
  a.window = (int)window;
  bool chunked;
  return tokens && seqs ? plan(a, bits_of(kv_dtype), max_new, max_len, chunked, nullptr) : 0;
}

extern "C" int vq2_paged_attention(const void* q, int64_t q_token_stride, int64_t q_head_stride, int dtype,
                                   int64_t tokens, int64_t q_heads, const void* k_pages, const void* v_pages,
                                   int kv_dtype, const float* k_scale, const float* v_scale, int64_t pages,
                                   int64_t kv_heads, int64_t page_size, int64_t head_size, const int32_t* table,
                                   int64_t table_stride, int64_t table_cols, const int32_t* lens, const int32_t* starts,
                                   int64_t seqs, int64_t max_new, int64_t max_len, float scale, int causal,
                                   int64_t window, void* out, float* lse, void* workspace, int64_t workspace_bytes,
                                   void* stream) {
  AttnArgs a = {};
  int s = paged_kv(a.kv, k_pages, v_pages, kv_dtype, k_scale, v_scale, pages, kv_heads, page_size, head_size, table,
                   table_stride, table_cols, lens, starts, seqs);
  if (s != VQ2_OK) return s;
  if (!q || !out || (!lens && seqs > 0)) return VQ2_ERR_ARG;
  if ((dtype != VQ2_F16 && dtype != VQ2_BF16) || (kv_dtype != dtype && kv_dtype != VQ2_I8 && kv_dtype != VQ2_I4))
    return VQ2_ERR_DTYPE;
  if (bad_attn(tokens, q_heads, kv_heads, seqs, max_new, max_len, window) || (!starts && tokens != seqs)) return VQ2_ERR_SHAPE;
  if (!aligned(q, 16) || q_token_stride % 8 || q_head_stride % 8 || !aligned(out, 16) || !aligned(workspace, 16))
    return VQ2_ERR_ALIGN;
  if (tokens == 0) return VQ2_OK;
  a.q = q;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.T = (int)tokens;
  a.hq = (int)q_heads;
  a.D = (int)head_size;
  a.G = a.hq / a.kv.heads;
  a.q_bf16 = dtype == VQ2_BF16;
  a.scale_log2 = scale * 1.44269504088896340736f;
  a.causal = causal;
  a.window = (int)window;
  a.out = out;
  a.lse = lse;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (seqs == 0) return launch_kernel(attn_blank_kernel, dim3(2 * sm_count()), dim3(256), 0, st, a);
  bool chunked;
  const int bits = bits_of(kv_dtype);
  const int64_t bytes = plan(a, bits, starts ? max_new : 1, max_len, chunked, static_cast<char*>(workspace));
  if (bytes && (!workspace || workspace_bytes < bytes)) return VQ2_ERR_ARG;
  if ((int64_t)a.kv.seqs * a.row_blocks > 0x3fffffff) return VQ2_ERR_SHAPE;
  s = chunked ? launch_attn_chunk(a, bits, st) : bits == 4 ? launch_attn_decode4(a, st) : launch_attn_decode(a, bits == 8, st);
  if (s != VQ2_OK || a.splits == 1) return s;
  return launch_attn_join(a, st);
}
