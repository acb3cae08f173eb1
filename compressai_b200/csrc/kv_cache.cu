// Rotary positions, and the paged key/value cache: written (rotary of q and k fused, 8-bit
// quantisation optional) and read back.
//
// Pools are [pages, kv_heads, page_size, head] so that a (page, head) pair is one contiguous piece
// for the attention that reads it. Position p of sequence b lives in page table[b][p / page_size],
// row p % page_size.
//
// All three are moved bytes: each thread owns 8 consecutive values of a head (one 16-byte load),
// LPR = 2..32 lanes a row. In the half layout a value's partner sits half a rotary width away: a
// lane holds 4 values and their 4 partners (two 8-byte loads), or, for few tokens and for widths that
// are no multiple of 8, 8 values in a row and reads their partners beside them. cos and sin belong to
// (token, pair) and serve every head, so a block takes one token and computes them once into shared
// memory, behind the value loads already in flight.
#include <type_traits>

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

// The four values at p and the four `apart` values on.
template <typename T>
__device__ __forceinline__ uint4 load_fours(const T* p, int apart, bool vec) {
  if (vec) {
    const uint2 a = *reinterpret_cast<const uint2*>(p), b = *reinterpret_cast<const uint2*>(p + apart);
    return make_uint4(a.x, a.y, b.x, b.y);
  }
  T t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = p[i < 4 ? i : apart + i - 4];
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

// Which 8 values of a row a lane holds, and where their partners are.
enum class Hold {
  kNeighbours,   // 8 in a row, paired with each other (also where nothing is turned)
  kPartners,     // 8 in a row of the half layout, the partners loaded beside them: any rotary width
  kSplit,        // half layout: 4 in a row and the 4 that pair with them, half a rotary width on
};

// (cos, sin) of a lane's 8 values -- of their 4 pairs, or with partners of each, the sine's sign the
// value's side -- and the turn in 32 bits. Values past the rotary width: (1, 0).
template <Hold HOLD>
struct Turn {
  static constexpr int N = HOLD == Hold::kPartners ? 8 : 4;
  float2 c[N];
  __device__ __forceinline__ void load(int lane, int rot, const float2* cs) {
    const int h = rot >> 1;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int e = lane * 8 + j;   // with partners
      const int pair = HOLD == Hold::kPartners ? (e < h ? e : e < rot ? e - h : h) : lane * 4 + j;
      c[j] = pair < h ? cs[pair] : make_float2(1.f, 0.f);
      if (HOLD == Hold::kPartners && e < h) c[j].y = -c[j].y;
    }
  }
  __device__ __forceinline__ void apply(float (&x)[8], const float (&w)[8]) const {
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (HOLD == Hold::kPartners) {
        x[j] = x[j] * c[j].x + w[j] * c[j].y;
      } else {
        float &a = x[HOLD == Hold::kSplit ? j : 2 * j], &b = x[HOLD == Hold::kSplit ? j + 4 : 2 * j + 1];
        const float a0 = a;
        a = a0 * c[j].x - b * c[j].y;
        b = b * c[j].x + a0 * c[j].y;
      }
    }
  }
};

// (cos, sin) * factor of each pair of token position pos (block-wide).
__device__ __forceinline__ void fill_turns(const RopeArgs& a, int64_t pos, float2* cs) {
  for (int i = threadIdx.x; i < (a.rot >> 1); i += blockDim.x) {
    // The angle in turns in 64 bits, whole turns dropped before it is rounded: at position 10^5 the
    // product rounded to 32 bits is off by up to 0.004 rad.
    const double turns = (double)pos * (double)a.inv_freq[i] * 0.15915494309189533577;
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    cs[i] = make_float2(c * a.factor, s * a.factor * a.sign);
  }
}

// Token t's position and its place in the cache (block-wide): page * page_size + row, or -1.
template <int MODE>
__device__ __forceinline__ void place_of(const RopeArgs& a, int t, int64_t& pos, int64_t& slot) {
  pos = 0;
  slot = -1;
  if (MODE == 0) {
    pos = a.pos64 ? static_cast<const int64_t*>(a.positions)[t] : static_cast<const int32_t*>(a.positions)[t];
    return;
  }
  const int b = sequence_of(a.kv, t);
  if (b < 0) return;
  int first, count;
  sequence_rows(a.kv, b, first, count);
  pos = (int64_t)a.kv.lens[b] - count + (t - first);
  slot = slot_of(a.kv, b, pos);
}

// 8 values of a row held by 2^lanes_log2 lanes as int8, and the row's scale: amax / 127, 0 below 1e-30, NaN
// where a value is not finite. Warp-wide; a lane that is not `mine` adds nothing.
__device__ __forceinline__ uint2 quantise8(const float (&f)[8], bool mine, int lanes_log2, float& scale) {
  float amax = 0.f;   // a NaN passes through
  if (mine) {
#pragma unroll
    for (int j = 0; j < 8; ++j) amax = max_nan(amax, fabsf(f[j]));
  }
  for (int o = 1; o < (1 << lanes_log2); o <<= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  uint32_t o[2] = {0, 0};
  scale = 0.f;
  if (!(amax < INFINITY)) {
    scale = __uint_as_float(0x7fc00000u);
  } else if (amax >= 1e-30f) {
    scale = __fdiv_rn(amax, 127.f);
    const float inv = __fdiv_rn(127.f, amax);
    // |x * inv| <= 127 (1 + 2^-23): no clamp. Adding 1.5 * 2^23 rounds to the nearest even integer and
    // leaves it in the low byte.
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) u[j] = __float_as_uint(__fadd_rn(__fmul_rn(f[j], inv), 12582912.f));
#pragma unroll
    for (int j = 0; j < 2; ++j)
      o[j] = __byte_perm(__byte_perm(u[4 * j], u[4 * j + 1], 0x0040), __byte_perm(u[4 * j + 2], u[4 * j + 3], 0x0040), 0x5410);
  }
  return make_uint2(o[0], o[1]);
}

// MODE 0: rotary of q and k into contiguous outputs. MODE 1: rotary of q, k (rotated) and v into a
// 16-bit cache. MODE 2: the same into an 8-bit cache. For few tokens: a row per lane group, its kind by its
// number.
template <typename T, int MODE, Hold HOLD>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a) {
  __shared__ float2 cs[128];
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x;
  const int groups = blockDim.x >> a.lanes_log2;
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1), g = threadIdx.x >> a.lanes_log2;
  const int rows_q = a.in[0].heads, rows_k = a.in[1].heads, rows = rows_q + rows_k * (MODE ? 2 : 1);
  const int i0 = lane * 8, r = blockIdx.y * groups + g;
  const int kind = r < rows_q ? 0 : r < rows_q + rows_k ? 1 : 2;
  const int h = kind == 0 ? r : kind == 1 ? r - rows_q : r - rows_q - rows_k;
  const bool mine = r < rows && i0 < a.D, turning = a.inv_freq != nullptr, turned = turning && kind < 2 && i0 < a.rot;

  uint4 x = make_uint4(0, 0, 0, 0), w = x;
  if (mine) {   // ahead of the chain that finds the position
    const RopeRows& in = a.in[kind];
    const T* row = static_cast<const T*>(in.x) + t * in.ts + h * in.hs;
    x = load8(row + i0, in.vec);
    if (HOLD == Hold::kPartners && turned) w = load_partner(row, i0, a.rot, in.vec);
  }
  int64_t pos, slot;
  place_of<MODE>(a, t, pos, slot);
  Turn<HOLD> turn;
  if (turning) {
    fill_turns(a, pos, cs);
    __syncthreads();
    turn.load(lane, a.rot, cs);
  }
  float f[8], p[8];
  widen8<T>(x, f);
  if (turned) {
    if (HOLD == Hold::kPartners) widen8<T>(w, p);
    turn.apply(f, p);
  }
  if (MODE != 2 || kind == 0) {
    if (mine && (MODE != 1 || kind == 0 || slot >= 0)) {
      T* dst;
      if (kind == 0) dst = static_cast<T*>(a.q_out) + ((int64_t)t * rows_q + h) * a.D;
      else if (MODE == 0) dst = static_cast<T*>(a.k_out) + ((int64_t)t * rows_k + h) * a.D;
      else dst = static_cast<T*>(const_cast<void*>(kind == 1 ? a.kv.k : a.kv.v)) + pool_row(a.kv, slot, h) * a.D;
      *reinterpret_cast<uint4*>(dst + i0) = turned ? narrow8<T>(f) : x;
    }
  }
  if (MODE == 2) {   // rows of different kinds can share a warp, so every lane takes part
    float scale;
    const uint2 o = quantise8(f, mine, a.lanes_log2, scale);
    if (kind == 0 || !mine || slot < 0) return;
    const int64_t row = pool_row(a.kv, slot, h);
    int8_t* dst = static_cast<int8_t*>(const_cast<void*>(kind == 1 ? a.kv.k : a.kv.v)) + row * a.D;
    *reinterpret_cast<uint2*>(dst + i0) = o;
    if (lane == 0) const_cast<float*>(kind == 1 ? a.kv.k_scale : a.kv.v_scale)[row] = scale;
  }
}

// The same for many tokens, q, k and v one after the other: what a row is (turned or not, quantised or
// not, where it goes) is then the same for a whole loop; choosing it per row took a third of the
// instructions. In the half layout a lane holds both sides of its pairs (SPLIT), so that each value is
// loaded and turned once. 40 registers, for the loads in flight that 6 blocks an SM hold; U rows at a
// time, as many as fit them. B200, device time: rotary of 8191 tokens of 40 heads of 128 29.5 us (5.7
// TB/s), half layout 32.3 (50.9 with the partners loaded beside the values, 42.8 so in these loops);
// 11,731 tokens of 32 + 16 heads of 128 written in int8 and read back 70.8 us, half layout 75.1 (79.3 and
// 114 with a row per lane group).
template <typename T, int MODE, bool SPLIT>
__global__ void __launch_bounds__(kRopeThreads, 6) rope_wide_kernel(const RopeArgs a) {
  __shared__ float2 cs[128];
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x;
  const int groups = blockDim.x >> a.lanes_log2;
  const int lane = threadIdx.x & ((1 << a.lanes_log2) - 1), g = threadIdx.x >> a.lanes_log2;
  const bool turning = a.inv_freq != nullptr, in_row = lane * 8 < a.D, in_rot = turning && lane * 8 < a.rot;
  const int i0 = SPLIT && in_rot ? lane * 4 : lane * 8, apart = SPLIT && in_rot ? a.rot >> 1 : 4;

  int64_t pos, slot;
  place_of<MODE>(a, t, pos, slot);
  if (turning) {
    fill_turns(a, pos, cs);
    __syncthreads();
  }
  Turn<SPLIT ? Hold::kSplit : Hold::kNeighbours> turn;
  if (turning) turn.load(lane, a.rot, cs);

  // rows of kind KIND: 0 q, 1 k, 2 v; U at a time
  auto rows_of_kind = [&](auto kind_c, auto u_c) {
    constexpr int KIND = decltype(kind_c)::value, U = decltype(u_c)::value;
    const RopeRows& in = a.in[KIND];
    const bool turned = KIND < 2 && in_rot;
    const T* src = static_cast<const T*>(in.x) + t * in.ts + i0;
    constexpr bool kPool = MODE != 0 && KIND > 0;
    T* dst = kPool ? static_cast<T*>(const_cast<void*>(KIND == 1 ? a.kv.k : a.kv.v))
                   : static_cast<T*>(KIND == 0 ? a.q_out : a.k_out) + (int64_t)t * in.heads * a.D;
    const int64_t pool0 = kPool && slot >= 0 ? pool_row(a.kv, slot, 0) : 0;   // of head 0; the next head is a page of rows on
    for (int h0 = g; h0 - g < in.heads; h0 += U * groups) {
      uint4 x[U];
#pragma unroll
      for (int n = 0; n < U; ++n) {
        const int h = h0 + n * groups;
        x[n] = make_uint4(0, 0, 0, 0);
        if (h < in.heads && in_row) {
          if constexpr (SPLIT) x[n] = load_fours(src + h * in.hs, apart, in.vec);
          else x[n] = load8(src + h * in.hs, in.vec);
        }
      }
#pragma unroll
      for (int n = 0; n < U; ++n) {
        const int h = h0 + n * groups;
        const bool mine = h < in.heads && in_row;
        float f[8];
        if (turned || (kPool && MODE == 2)) widen8<T>(x[n], f);
        if (turned) turn.apply(f, f);
        const int64_t row = kPool ? pool0 + ((int64_t)h << a.kv.page_log2) : h;
        if (!kPool || MODE == 1) {
          if (mine && (!kPool || slot >= 0)) {
            if constexpr (SPLIT) {
              T* to = dst + row * a.D + i0;
              if (turned) x[n] = narrow8<T>(f);
              *reinterpret_cast<uint2*>(to) = make_uint2(x[n].x, x[n].y);
              *reinterpret_cast<uint2*>(to + apart) = make_uint2(x[n].z, x[n].w);
            } else {
              *reinterpret_cast<uint4*>(dst + row * a.D + i0) = turned ? narrow8<T>(f) : x[n];
            }
          }
        } else {
          float scale;
          const uint2 o = quantise8(f, mine, a.lanes_log2, scale);
          if (mine && slot >= 0) {
            int8_t* to = reinterpret_cast<int8_t*>(dst) + row * a.D + i0;
            if constexpr (SPLIT) {
              *reinterpret_cast<uint32_t*>(to) = o.x;
              *reinterpret_cast<uint32_t*>(to + apart) = o.y;
            } else {
              *reinterpret_cast<uint2*>(to) = o;
            }
            if (lane == 0) const_cast<float*>(KIND == 1 ? a.kv.k_scale : a.kv.v_scale)[row] = scale;
          }
        }
      }
    }
  };
  using std::integral_constant;
  rows_of_kind(integral_constant<int, 0>(), integral_constant<int, SPLIT ? 2 : 4>());
  rows_of_kind(integral_constant<int, 1>(), integral_constant<int, 1>());
  if (MODE != 0) rows_of_kind(integral_constant<int, 2>(), integral_constant<int, 1>());
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
  const bool neighbours = a.interleaved || !a.inv_freq;
  // One row per lane group while the blocks are fewer than the card holds at once (2048 threads an
  // SM): a lone token is spread over blocks. Then a block a token, the rows of a kind in a loop; not
  // where a half of the rotary width is no whole number of fours.
  if (T_ * ((rows + per - 1) / per) <= (int64_t)sm_count() * 8 || (!neighbours && a.rot % 8)) {
    const int y = (rows + per - 1) / per, groups = (rows + y - 1) / y;
    const dim3 grid((unsigned)T_, (unsigned)y), block((((groups << a.lanes_log2) + 31) / 32) * 32);
    return neighbours ? launch_kernel(rope_kernel<T, MODE, Hold::kNeighbours>, grid, block, 0, st, a)
                      : launch_kernel(rope_kernel<T, MODE, Hold::kPartners>, grid, block, 0, st, a);
  }
  // four rows of the most numerous kind a lane group
  const int most = a.in[0].heads > a.in[1].heads ? a.in[0].heads : a.in[1].heads;
  int groups = (most + 3) / 4;
  if (groups > per) groups = per;
  const dim3 grid((unsigned)T_), block((((groups << a.lanes_log2) + 31) / 32) * 32);
  return neighbours ? launch_kernel(rope_wide_kernel<T, MODE, false>, grid, block, 0, st, a)
                    : launch_kernel(rope_wide_kernel<T, MODE, true>, grid, block, 0, st, a);
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
  if (!k || !v || (!lens && seqs > 0) || (q_heads && (!q || !q_out))) return VQ2_ERR_ARG;
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
