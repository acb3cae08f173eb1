// Rotary positions, and the paged key/value cache: written (rotary of q and k fused, 8-bit
// quantisation optional) and read back.
//
// Pools are [pages, kv_heads, page_size, head] so that a (page, head) pair is one contiguous piece
// for the attention that reads it. Position p of sequence b lives in page table[b][p / page_size],
// row p % page_size.
//
// All three are moved bytes: each thread owns 8 consecutive values of a head (one 16-byte load),
// LPR = 2..32 lanes a row. In the half layout a value's partner sits half a rotary width away; it
// is read a second time rather than shuffled (it hits L1, and needs no rule about where the halves
// fall among the lanes). cos and sin belong to (token, pair) and serve every head, so a block takes
// one token and computes them once into shared memory, behind the value loads already in flight.
#include "kv_dev.cuh"

namespace vq2 {
namespace {

constexpr int kRopeThreads = 256;

struct RopeRows {           // rows of one kind: [T, heads, D], last dimension contiguous
  const void* x;
  int64_t ts, hs;           // token and head strides, elements
  int heads, vec;           // vec: base and strides allow 16-byte loads
};

struct RopeArgs {
  RopeRows in[3];           // q, k, v (v: cache write only)
  void* q_out;              // [T, heads, D] contiguous
  void* k_out;              // rotary only
  const void* positions;    // rotary only: int32 or int64 [T]
  int pos64;
  const float* inv_freq;    // [rot / 2]; null: no rotation
  int rot, interleaved;
  float factor, sign;
  int D, lanes_log2;        // lanes_log2: log2 of the lanes a row takes
  PagedKV kv;               // cache write only
};

// 8 values at p (16-byte load when the tensor allows it, else one by one).
template <typename T>
__device__ __forceinline__ uint4 load8(const T* p, bool vec) {
  if (vec) return *reinterpret_cast<const uint4*>(p);
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = p[i];
  uint4 r;
  memcpy(&r, t, 16);
  return r;
}

// The values that pair with the 8 at `i0` in the half layout (unspecified past the rotary width).
template <typename T>
__device__ __forceinline__ uint4 load_partner(const T* row, int i0, int rot, bool vec) {
  const int h = rot >> 1;
  if ((h & 7) == 0) return load8(row + (i0 < h ? i0 + h : i0 - h), vec);
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int e = i0 + i;
    t[i] = row[e < h ? e + h : e < rot ? e - h : e];
  }
  uint4 r;
  memcpy(&r, t, 16);
  return r;
}

template <typename T>
__device__ __forceinline__ void widen8(uint4 u, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 p = unpack2<T>((&u.x)[j]);
    f[2 * j] = p.x;
    f[2 * j + 1] = p.y;
  }
}

template <typename T>
__device__ __forceinline__ uint4 narrow8(const float (&f)[8]) {
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = from_f32<T>(f[i]);
  uint4 r;
  memcpy(&r, t, 16);
  return r;
}

// Maximum that a NaN passes through.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// (cos, sin) of the 8 values at i0 -- of their 4 pairs where neighbours are paired, else of each, the
// sine's sign the value's side -- and the turn in 32 bits. Values past the rotary width: (1, 0).
template <bool INTER>
struct Turn {
  float2 c[INTER ? 4 : 8];
  __device__ __forceinline__ void load(int i0, int rot, const float2* cs) {
    const int h = rot >> 1;
#pragma unroll
    for (int j = 0; j < (INTER ? 4 : 8); ++j) {
      const int e = INTER ? i0 + 2 * j : i0 + j;
      c[j] = make_float2(1.f, 0.f);
      if (e < rot) {
        c[j] = cs[INTER ? e >> 1 : e < h ? e : e - h];
        if (!INTER && e < h) c[j].y = -c[j].y;
      }
    }
  }
  __device__ __forceinline__ void apply(float (&x)[8], const float (&w)[8]) const {
    if (INTER) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = x[2 * j], b = x[2 * j + 1];
        x[2 * j] = a * c[j].x - b * c[j].y;
        x[2 * j + 1] = b * c[j].x + a * c[j].y;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) x[j] = x[j] * c[j].x + w[j] * c[j].y;
    }
  }
};

// MODE 0: rotary of q and k into contiguous outputs. MODE 1: rotary of q, k (rotated) and v into a
// 16-bit cache. MODE 2: the same into an 8-bit cache. NIT rows per lane group. INTER: neighbours are
// paired, and no partners are loaded (also where nothing is turned).
template <typename T, int MODE, int NIT, bool INTER>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a) {
  __shared__ float2 cs[128];
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x;
  const int groups = blockDim.x >> a.lanes_log2;
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1), g = threadIdx.x >> a.lanes_log2;
  const int rows_q = a.in[0].heads, rows_k = a.in[1].heads, rows = rows_q + rows_k * (MODE ? 2 : 1);
  const int i0 = lane * 8;
  const bool turning = a.inv_freq != nullptr;

  uint4 x[NIT], w[INTER ? 1 : NIT];
#pragma unroll
  for (int n = 0; n < NIT; ++n) {
    const int r = (blockIdx.y * NIT + n) * groups + g;
    x[n] = make_uint4(0, 0, 0, 0);
    if (!INTER) w[n] = make_uint4(0, 0, 0, 0);
    if (r < rows && i0 < a.D) {
      const int kind = r < rows_q ? 0 : r < rows_q + rows_k ? 1 : 2;
      const RopeRows& in = a.in[kind];
      const int h = kind == 0 ? r : kind == 1 ? r - rows_q : r - rows_q - rows_k;
      const T* row = static_cast<const T*>(in.x) + t * in.ts + h * in.hs;
      x[n] = load8(row + i0, in.vec);
      if (!INTER && turning && kind < 2 && i0 < a.rot) w[n] = load_partner(row, i0, a.rot, in.vec);
    }
  }

  int64_t pos = 0, slot = -1;  // slot: page * page_size + row, or -1 (token stored nowhere)
  if (MODE == 0) {
    pos = a.pos64 ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int32_t*>(a.positions)[t];
  } else {
    const int b = sequence_of(a.kv, t);
    if (b >= 0) {
      int first, count;
      sequence_rows(a.kv, b, first, count);
      pos = (int64_t)a.kv.lens[b] - count + (t - first);
      slot = slot_of(a.kv, b, pos);
    }
  }
  if (turning) {
    for (int i = threadIdx.x; i < (a.rot >> 1); i += blockDim.x) {
      // The angle in turns in 64 bits, whole turns dropped before it is rounded: at position 10^5 the
      // product rounded to 32 bits is off by up to 0.004 rad.
      const double turns = (double)pos * (double)a.inv_freq[i] * 0.15915494309189533577;
      float s, c;
      sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
      cs[i] = make_float2(c * a.factor, s * a.factor * a.sign);
    }
    __syncthreads();
  }
  // a lane has the same values of every row: one set of (cos, sin) in registers
  Turn<INTER> turn;
  if (turning) turn.load(i0, a.rot, cs);

#pragma unroll
  for (int n = 0; n < NIT; ++n) {
    const int r = (blockIdx.y * NIT + n) * groups + g;
    const int kind = r < rows_q ? 0 : r < rows_q + rows_k ? 1 : 2;
    const int h = kind == 0 ? r : kind == 1 ? r - rows_q : r - rows_q - rows_k;
    const bool mine = r < rows && i0 < a.D;
    float f[8], p[8];
    widen8<T>(x[n], f);
    const bool turned = turning && kind < 2 && i0 < a.rot;
    if (turned) {
      if (!INTER) widen8<T>(w[n], p);
      turn.apply(f, p);
    }
    if (MODE != 2 || kind == 0) {
      if (mine && (MODE != 1 || kind == 0 || slot >= 0)) {
        T* dst;
        if (kind == 0) dst = static_cast<T*>(a.q_out) + ((int64_t)t * rows_q + h) * a.D;
        else if (MODE == 0) dst = static_cast<T*>(a.k_out) + ((int64_t)t * rows_k + h) * a.D;
        else dst = static_cast<T*>(const_cast<void*>(kind == 1 ? a.kv.k : a.kv.v)) + pool_row(a.kv, slot, h) * a.D;
        *reinterpret_cast<uint4*>(dst + i0) = turned ? narrow8<T>(f) : x[n];
      }
    }
    if (MODE == 2 && __any_sync(0xffffffffu, kind != 0)) {
      // amax over the row's lanes, a NaN above all numbers. Rows of different kinds can share a warp, so
      // every lane takes part.
      float amax = 0.f;
      if (mine) {
#pragma unroll
        for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(f[j]));
      }
      for (int o = 1; o < (1 << a.lanes_log2); o <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      if (kind == 0 || !mine || slot < 0) continue;
      float scale = 0.f;
      uint32_t o[2] = {0, 0};
      if (!(amax < INFINITY)) scale = __uint_as_float(0x7fc00000u);
      else if (amax >= 1e-30f) {
        scale = __fdiv_rn(amax, 127.f);
        const float inv = __fdiv_rn(127.f, amax);
        // |x * inv| <= 127 (1 + 2^-23): no clamp. Adding 1.5 * 2^23 rounds to the nearest even integer
        // and leaves it in the low byte.
        uint32_t u[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = __float_as_uint(__fadd_rn(__fmul_rn(f[j], inv), 12582912.f));
#pragma unroll
        for (int j = 0; j < 2; ++j)
          o[j] = __byte_perm(__byte_perm(u[4 * j], u[4 * j + 1], 0x0040), __byte_perm(u[4 * j + 2], u[4 * j + 3], 0x0040), 0x5410);
      }
      const int64_t row = pool_row(a.kv, slot, h);
      int8_t* dst = static_cast<int8_t*>(const_cast<void*>(kind == 1 ? a.kv.k : a.kv.v)) + row * a.D;
      *reinterpret_cast<uint2*>(dst + i0) = make_uint2(o[0], o[1]);
      if (lane == 0) const_cast<float*>(kind == 1 ? a.kv.k_scale : a.kv.v_scale)[row] = scale;
    }
  }
}

struct ReadArgs {
  PagedKV kv;
  void *k_out, *v_out;      // [total, kv_heads, D] contiguous
  int64_t total;
  int D, lanes_log2;
};

// Row (token, head) per lane group, K and V together; NIT rows per group, their loads in flight at once.
template <typename T, bool I8, int NIT>
__global__ void __launch_bounds__(kRopeThreads) cache_read_kernel(const ReadArgs a) {
  pdl_wait();
  pdl_trigger();
  const int groups = blockDim.x >> a.lanes_log2;
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1), g = threadIdx.x >> a.lanes_log2;
  const int H = a.kv.heads, i0 = lane * 8;
  const int64_t r0 = (int64_t)blockIdx.x * groups * NIT, rows = a.total * H;
  const int b0 = sequences_before(a.kv, (int)(r0 / H));   // the block's first row's; later rows step on from it
  uint4 x[NIT][2];
  float s[NIT][2];
#pragma unroll
  for (int n = 0; n < NIT; ++n) {
    const int64_t r = r0 + n * groups + g;
    x[n][0] = x[n][1] = make_uint4(0, 0, 0, 0);
    s[n][0] = s[n][1] = 0.f;
    if (r >= rows || i0 >= a.D) continue;
    const int t = (int)(r / H), h = (int)(r - (int64_t)t * H);
    int b = b0;
    while (b < a.kv.seqs && a.kv.starts[b + 1] <= t) ++b;
    if (b >= a.kv.seqs || a.kv.starts[b] > t) continue;
    const int64_t slot = slot_of(a.kv, b, t - a.kv.starts[b]);
    if (slot < 0) continue;
    const int64_t row = pool_row(a.kv, slot, h), e = row * a.D + i0;
    if (I8) {
      const uint2 k = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.kv.k) + e);
      const uint2 v = *reinterpret_cast<const uint2*>(static_cast<const int8_t*>(a.kv.v) + e);
      x[n][0] = make_uint4(k.x, k.y, 0, 0);
      x[n][1] = make_uint4(v.x, v.y, 0, 0);
      s[n][0] = a.kv.k_scale[row];
      s[n][1] = a.kv.v_scale[row];
    } else {
      x[n][0] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.kv.k) + e);
      x[n][1] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.kv.v) + e);
    }
  }
#pragma unroll
  for (int n = 0; n < NIT; ++n) {
    const int64_t r = r0 + n * groups + g;
    if (r >= rows || i0 >= a.D) continue;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      uint4 y = x[n][c];
      if (I8) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (float)(int8_t)((&x[n][c].x)[j >> 2] >> (8 * (j & 3))) * s[n][c];
        y = narrow8<T>(f);
      }
      *reinterpret_cast<uint4*>(static_cast<T*>(c ? a.v_out : a.k_out) + r * a.D + i0) = y;
    }
  }
}

int lanes_log2(int D) {
  int l = 1;
  while ((8 << l) < D) ++l;
  return l;
}

template <typename T, int MODE>
int launch_rope(const RopeArgs& a, int64_t T_, cudaStream_t st) {
  const int rows = a.in[0].heads + a.in[1].heads * (MODE ? 2 : 1);
  const int per = kRopeThreads >> a.lanes_log2;
  // One row per lane group while the blocks are fewer than the card holds at once (2048 threads an
  // SM): a lone token is spread over blocks. Then four, so that a block's
  // table of cos and sin and its sequence lookup serve more rows; six in the 8-bit write, which
  // instructions bound (11,731 tokens of 32 + 16 heads of 128: four rows 78 us, six 70, eight 75).
  const int64_t blocks1 = T_ * ((rows + per - 1) / per);
  const bool wide = blocks1 > (int64_t)sm_count() * 8;
  const bool inter = a.interleaved || !a.inv_freq;
  constexpr int kRows = MODE == 2 ? 6 : 4;
  const int nit = !wide ? 1 : inter ? kRows : 4;
  const int y = (rows + per * nit - 1) / (per * nit);
  const int groups = (rows + y * nit - 1) / (y * nit);        // groups a block needs
  const int threads = (((groups << a.lanes_log2) + 31) / 32) * 32;
  const dim3 grid((unsigned)T_, (unsigned)y);
  if (inter)
    return wide ? launch_kernel(rope_kernel<T, MODE, kRows, true>, grid, dim3(threads), 0, st, a)
                : launch_kernel(rope_kernel<T, MODE, 1, true>, grid, dim3(threads), 0, st, a);
  return wide ? launch_kernel(rope_kernel<T, MODE, 4, false>, grid, dim3(threads), 0, st, a)
              : launch_kernel(rope_kernel<T, MODE, 1, false>, grid, dim3(threads), 0, st, a);
}

RopeRows rows_of(const void* x, int64_t ts, int64_t hs, int64_t heads) {
  return {x, ts, hs, (int)heads, aligned(x, 16) && ts % 8 == 0 && hs % 8 == 0};
}

bool bad_rotary(const float* inv_freq, int64_t rot, int64_t D) {
  return inv_freq ? rot < 2 || rot > D || rot % 2 : rot != 0;
}

}  // namespace
}  // namespace vq2

using namespace vq2;

extern "C" int vq2_rotary(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads, const void* k,
                          int64_t k_token_stride, int64_t k_head_stride, int64_t k_heads, int dtype, int64_t tokens,
                          int64_t head_size, const void* positions, int positions64, const float* inv_freq, int64_t rot,
                          int interleaved, float factor, int inverse, void* q_out, void* k_out, void* stream) {
  if (!positions || !inv_freq || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return VQ2_ERR_ARG;
  if (dtype != VQ2_F16 && dtype != VQ2_BF16) return VQ2_ERR_DTYPE;
  if (tokens < 0 || tokens > 0x7fffffff || q_heads < 0 || k_heads < 0 || q_heads > 4096 || k_heads > 4096 ||
      bad_head_size(head_size) || bad_rotary(inv_freq, rot, head_size))
    return VQ2_ERR_SHAPE;
  if (!aligned(q_out, 16) || !aligned(k_out, 16)) return VQ2_ERR_ALIGN;
  if (tokens == 0 || q_heads + k_heads == 0) return VQ2_OK;
  RopeArgs a = {};
  a.in[0] = rows_of(q, q_token_stride, q_head_stride, q_heads);
  a.in[1] = rows_of(k, k_token_stride, k_head_stride, k_heads);
  a.q_out = q_out;
  a.k_out = k_out;
  a.positions = positions;
  a.pos64 = positions64;
  a.inv_freq = inv_freq;
  a.rot = (int)rot;
  a.interleaved = interleaved;
  a.factor = factor;
  a.sign = inverse ? -1.f : 1.f;
  a.D = (int)head_size;
  a.lanes_log2 = lanes_log2(a.D);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == VQ2_F16 ? launch_rope<__half, 0>(a, tokens, st) : launch_rope<__nv_bfloat16, 0>(a, tokens, st);
}

extern "C" int vq2_cache_write(const void* q, int64_t q_token_stride, int64_t q_head_stride, int64_t q_heads, void* q_out,
                               const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                               int64_t v_token_stride, int64_t v_head_stride, int dtype, int64_t tokens,
                               const float* inv_freq, int64_t rot, int interleaved, float factor, void* k_pages,
                               void* v_pages, int kv_dtype, float* k_scale, float* v_scale, int64_t pages,
                               int64_t kv_heads, int64_t page_size, int64_t head_size, const int32_t* table,
                               int64_t table_stride, int64_t table_cols, const int32_t* lens, const int32_t* starts,
                               int64_t seqs, void* stream) {
  RopeArgs a = {};
  int s = paged_kv(a.kv, k_pages, v_pages, kv_dtype, k_scale, v_scale, pages, kv_heads, page_size, head_size, table,
                   table_stride, table_cols, lens, starts, seqs);
  if (s != VQ2_OK) return s;
  if (!k || !v || !lens || (q_heads && (!q || !q_out))) return VQ2_ERR_ARG;
  if ((dtype != VQ2_F16 && dtype != VQ2_BF16) || (kv_dtype != dtype && kv_dtype != VQ2_I8)) return VQ2_ERR_DTYPE;
  if (tokens < 0 || tokens > 0x7fffffff || q_heads < 0 || q_heads > 4096 || bad_rotary(inv_freq, rot, head_size) ||
      (!starts && tokens != seqs))
    return VQ2_ERR_SHAPE;
  if (!aligned(q_out, 16)) return VQ2_ERR_ALIGN;
  if (tokens == 0) return VQ2_OK;
  a.in[0] = rows_of(q, q_token_stride, q_head_stride, q_heads);
  a.in[1] = rows_of(k, k_token_stride, k_head_stride, kv_heads);
  a.in[2] = rows_of(v, v_token_stride, v_head_stride, kv_heads);
  a.q_out = q_out;
  a.inv_freq = inv_freq;
  a.rot = (int)rot;
  a.interleaved = interleaved;
  a.factor = factor;
  a.sign = 1.f;
  a.D = (int)head_size;
  a.lanes_log2 = lanes_log2(a.D);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (kv_dtype == VQ2_I8)
    return dtype == VQ2_F16 ? launch_rope<__half, 2>(a, tokens, st) : launch_rope<__nv_bfloat16, 2>(a, tokens, st);
  return dtype == VQ2_F16 ? launch_rope<__half, 1>(a, tokens, st) : launch_rope<__nv_bfloat16, 1>(a, tokens, st);
}

extern "C" int vq2_cache_read(const void* k_pages, const void* v_pages, int kv_dtype, const float* k_scale,
                              const float* v_scale, int64_t pages, int64_t kv_heads, int64_t page_size,
                              int64_t head_size, const int32_t* table, int64_t table_stride, int64_t table_cols,
                              const int32_t* starts, int64_t seqs, void* k_out, void* v_out, int out_dtype,
                              int64_t total, void* stream) {
  ReadArgs a = {};
  int s = paged_kv(a.kv, k_pages, v_pages, kv_dtype, k_scale, v_scale, pages, kv_heads, page_size, head_size, table,
                   table_stride, table_cols, nullptr, starts, seqs);
  if (s != VQ2_OK) return s;
  if (!starts || !k_out || !v_out) return VQ2_ERR_ARG;
  if ((out_dtype != VQ2_F16 && out_dtype != VQ2_BF16) || (kv_dtype != out_dtype && kv_dtype != VQ2_I8)) return VQ2_ERR_DTYPE;
  if (total < 0 || total > 0x7fffffff) return VQ2_ERR_SHAPE;
  if (!aligned(k_out, 16) || !aligned(v_out, 16)) return VQ2_ERR_ALIGN;
  if (total == 0) return VQ2_OK;
  a.k_out = k_out;
  a.v_out = v_out;
  a.total = total;
  a.D = (int)head_size;
  a.lanes_log2 = lanes_log2(a.D);
  constexpr int NIT = 2;
  const int64_t per = (int64_t)(kRopeThreads >> a.lanes_log2) * NIT;
  const int64_t blocks = (total * kv_heads + per - 1) / per;
  if (blocks > 0x7fffffff) return VQ2_ERR_SHAPE;
  const dim3 grid((unsigned)blocks), block(kRopeThreads);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (kv_dtype == VQ2_I8)
    return out_dtype == VQ2_F16 ? launch_kernel(cache_read_kernel<__half, true, NIT>, grid, block, 0, st, a)
                                : launch_kernel(cache_read_kernel<__nv_bfloat16, true, NIT>, grid, block, 0, st, a);
  return out_dtype == VQ2_F16 ? launch_kernel(cache_read_kernel<__half, false, NIT>, grid, block, 0, st, a)
                              : launch_kernel(cache_read_kernel<__nv_bfloat16, false, NIT>, grid, block, 0, st, a);
}
