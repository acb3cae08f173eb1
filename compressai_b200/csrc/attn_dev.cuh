// What the attention kernels share: arguments, the keys that query rows see, and how rows are split
// along the keys and joined.
#pragma once
#include <type_traits>

#include "kv_dev.cuh"

namespace vq2 {

struct AttnArgs {
  PagedKV kv;
  const void* q;
  int64_t q_ts, q_hs;   // strides of q, elements
  int T, hq, D, G;      // G: query heads per key/value head
  int q_bf16;           // type of q and out
  float scale_log2;     // scale * log2(e): scores in powers of two
  int causal, window;
  void* out;            // [T, hq, D]
  float* lse;           // [T, hq] or null
  // Split s of a block of rows takes the keys lo + s * chunk .. lo + (s + 1) * chunk - 1 of the keys
  // [lo, hi) that the block sees, lo rounded down by lo_mask. rows_per_block: query rows a block takes.
  int chunk, splits, rows_per_block, row_blocks, lo_mask;
  float* part_o;        // [T * hq, splits, D]: weighted sums of V relative to the maximum
  float2* part_ml;      // [T * hq, splits]: (maximum score in powers of two, sum of weights)
  // 8-bit cache, many rows: the visible keys and values as fp16 [seqs, heads, wide_len, D], their scales
  void *wide_k, *wide_v;
  float *wide_ks, *wide_vs;
  int wide_len;
  int keys_end;         // no key from here on is looked at: wide_len there, else past every position
};

constexpr float kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The power of two above a positive V scale, which the weights of an 8-bit cache are relative to. 2^126 at most,
// so that its inverse is a normal number too (a scale above overflows with any value beyond 2 anyway).
__device__ __forceinline__ float above(float scale) {
  return __uint_as_float(min((__float_as_uint(scale) & 0x7f800000u) + 0x00800000u, 0x7e800000u));
}

// The exponent that brings a bf16 row whose largest magnitude is `top` into fp16, to 2^13 .. 2^14, and back: its
// power of two and the inverse are normal numbers. 0 where there is nothing to bring, or no finite number.
__device__ __forceinline__ int fp16_lift(float top) {
  return top > 0.f && top < INFINITY ? min(13 - ilogbf(top), 126) : 0;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if (std::is_same<T, __half>::value) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Two bytes of w (offset binary, v + 128), chosen by sel's nibbles 0 and 2, as two exact fp16 values.
__device__ __forceinline__ uint32_t bytes_f16(uint32_t w, uint32_t sel) {
  const uint32_t p = __byte_perm(w, 0x64646464u, sel);  // 0x6400 | u = 1024 + u
  const uint32_t bias = 0x64806480u;                    // 1152
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&p), *reinterpret_cast<const __half2*>(&bias));
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A sequence's new tokens, and the block of query rows [r0, r0 + rows) among its count * G: row r is
// new token r / G, head r % G of the key/value head.
struct AttnRows {
  int first, count, len;  // first new token, new tokens, length of the sequence
  int r0, rows;
};

__device__ __forceinline__ AttnRows attn_rows(const AttnArgs& a, int b, int rb) {
  AttnRows w;
  sequence_rows(a.kv, b, w.first, w.count);
  w.first = max(0, min(w.first, a.T));
  w.count = max(0, min(w.count, a.T - w.first));
  w.len = length_of(a.kv, b);
  w.r0 = rb * a.rows_per_block;
  w.rows = (int)max((int64_t)0, min((int64_t)a.rows_per_block, (int64_t)w.count * a.G - w.r0));
  return w;
}

// Keys that new token i sees: [row_lo, row_hi).
__device__ __forceinline__ int row_lo(const AttnArgs& a, const AttnRows& w, int i) {
  return a.window ? max(0, w.len - w.count + i - a.window + 1) : 0;
}
__device__ __forceinline__ int row_hi(const AttnArgs& a, const AttnRows& w, int i) {
  return a.causal ? max(0, min(w.len, w.len - w.count + i + 1)) : w.len;
}

// Keys that any row of the block sees, the start rounded down; no more than the splits cover, and of a
// widened cache no more than its copy holds, whatever lens says when the kernel runs.
__device__ __forceinline__ void block_keys(const AttnArgs& a, const AttnRows& w, int& lo, int& hi) {
  lo = row_lo(a, w, w.r0 / a.G) & a.lo_mask;
  hi = w.rows > 0 ? row_hi(a, w, (w.r0 + w.rows - 1) / a.G) : 0;
  hi = (int)min((int64_t)min(hi, a.keys_end), lo + (int64_t)a.splits * a.chunk);
}

// Zeros, lse -inf, for `rows` rows (token, head) of `vecs` 16-byte pieces: part `part` of `parts` blocks. Not
// inlined: a launch that has no such rows then does not fetch these instructions.
static __device__ __noinline__ void blank(uint4* out, float* lse, int64_t rows, int vecs, int64_t part, int64_t parts) {
  const int64_t i0 = part * blockDim.x + threadIdx.x, step = parts * blockDim.x;
  for (int64_t i = i0; i < rows * vecs; i += step) out[i] = make_uint4(0, 0, 0, 0);
  if (lse)
    for (int64_t i = i0; i < rows; i += step) lse[i] = -INFINITY;
}

// The tokens [from, to).
__device__ __forceinline__ void blank_tokens(const AttnArgs& a, int from, int to, int64_t part, int64_t parts) {
  const int64_t row = (int64_t)from * a.hq;
  blank(reinterpret_cast<uint4*>(static_cast<uint16_t*>(a.out) + row * a.D), a.lse ? a.lse + row : nullptr,
        (int64_t)(to - from) * a.hq, a.D >> 3, part, parts);
}

// Tokens of no sequence (a step padded to a fixed size): the first sequence's blocks blank those before its
// tokens, the last one's those after, each its share.
__device__ __forceinline__ void blank_strays(const AttnArgs& a, const AttnRows& w, int b, int64_t part, int64_t parts) {
  const bool before = b == 0 && w.first > 0, after = b == a.kv.seqs - 1 && w.first + w.count < a.T;
  if (!before && !after) return;
  if (before) blank_tokens(a, 0, w.first, part, parts);
  if (after) blank_tokens(a, w.first + w.count, a.T, part, parts);
}

// Joins the splits of every row (launched after a kernel that left more than one).
int launch_attn_join(const AttnArgs& a, cudaStream_t st);
// Few rows per key/value head (attn_decode.cu), and many (attn_chunk.cu). The plans set
// chunk, splits, rows_per_block, row_blocks and lo_mask.
int launch_attn_decode(const AttnArgs& a, bool i8, cudaStream_t st);
void plan_attn_decode(AttnArgs& a, int64_t max_new, int64_t max_len);
int launch_attn_chunk(const AttnArgs& a, bool i8, cudaStream_t st);
void plan_attn_chunk(AttnArgs& a, int64_t max_new, int64_t max_len);
int attn_chunk_status(int reset);   // its part of vq2_attention_status

}  // namespace vq2
