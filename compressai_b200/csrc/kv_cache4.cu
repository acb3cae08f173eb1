// A 4-bit cache written from keys that are turned already (or are not turned at all), and read back.
//
// Both are moved bytes: 2 a value on one side, about 0.55 on the other; instructions come close behind. A lane has 16 values
// of a row (two 16-byte loads or stores, one of 8): a row's largest magnitude is 4 shuffles away at most, a group's 2, and
// what a row costs whatever its length is shared by 16 values. A lane group has a token's rows, K's and V's of U heads at a time, so
// that a token's sequence and page are looked up once and the heads' addresses follow by addition (a row per lane group, each
// looking its token up: 40.7 us for 53,000 tokens of 2 heads of 256, 607 instructions a warp and row pair).
#include "kv4_dev.cuh"

namespace vq2 {
namespace {

constexpr int kThreads = 256;

struct Args4 {
  PagedKV kv;
  const void *k, *v;                     // write: [tokens, heads, D], strides in elements
  int64_t k_ts, k_hs, v_ts, v_hs;
  int by;                                // their (read: the outputs') base and strides are multiples of: 32 or 16 bytes, or less
  void *k_out, *v_out;                   // read: [tokens, heads, D] contiguous
  int64_t tokens;
  int D;
  int heads_per;                         // of a block
};

// The sequence of new token t (block-wide; b0: of the block's first token), or -1.
__device__ __forceinline__ int sequence_from(const PagedKV& kv, int b0, int t) {
  if (!kv.starts) return t < kv.seqs ? t : -1;
  while (b0 < kv.seqs && kv.starts[b0 + 1] <= t) ++b0;
  return b0 < kv.seqs && kv.starts[b0] <= t ? b0 : -1;
}

// 16 values, as they lie; `by`: what address and strides are multiples of, in bytes (32: one access, 16: two). Two accesses of
// 16 bytes each touch half of every 32-byte sector (read-back of 53,000 tokens of 2 heads of 256: 35.8 us).
template <typename T>
__device__ __forceinline__ void load16(const T* p, int by, uint32_t (&x)[8]) {
  if (by == 32) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]), "=r"(x[4]), "=r"(x[5]), "=r"(x[6]), "=r"(x[7]) : "l"(p) : "memory");
    return;
  }
  if (by == 16) {
    const uint4 a = reinterpret_cast<const uint4*>(p)[0], b = reinterpret_cast<const uint4*>(p)[1];
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint16_t lo = reinterpret_cast<const uint16_t*>(p)[2 * i], hi = reinterpret_cast<const uint16_t*>(p)[2 * i + 1];
    x[i] = lo | (uint32_t)hi << 16;
  }
}
__device__ __forceinline__ void put16(void* p, int by, const uint32_t (&x)[8]) {
  if (by == 32) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 ::"l"(p), "r"(x[0]), "r"(x[1]), "r"(x[2]), "r"(x[3]), "r"(x[4]), "r"(x[5]), "r"(x[6]), "r"(x[7]) : "memory");
    return;
  }
  static_cast<uint4*>(p)[0] = make_uint4(x[0], x[1], x[2], x[3]);
  static_cast<uint4*>(p)[1] = make_uint4(x[4], x[5], x[6], x[7]);
}

// The largest magnitude of 16 values, as 16 bits: a NaN's are above an infinity's.
__device__ __forceinline__ uint32_t top16(const uint32_t (&x)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; i += 2) m = __vimax3_u16x2(m, x[i] & 0x7fff7fffu, x[i + 1] & 0x7fff7fffu);
  return max(m & 0xffffu, m >> 16);
}

// L: log2 of a row's lanes. (Blocks an SM: 64 registers, of 79; 3 blocks 64.0 us at the 53,000 tokens, 4 and 5 60.5, 5 and 6 69.3.)
template <typename T, int L, int U>
__global__ void __launch_bounds__(kThreads, 4) store4_kernel(const __grid_constant__ Args4 a) {
  pdl_wait();
  pdl_trigger();
  constexpr int lanes = 1 << L, groups = kThreads >> L;
  const int lane = threadIdx.x & (lanes - 1), i0 = 16 * lane;
  const int64_t t0 = (int64_t)blockIdx.x * groups, t = t0 + (threadIdx.x >> L);
  const int h_end = min(a.kv.heads, ((int)blockIdx.y + 1) * a.heads_per);
  int h = blockIdx.y * a.heads_per;
  const bool mine = t < a.tokens && i0 < a.D;
  const T* from[2] = {static_cast<const T*>(a.k) + t * a.k_ts + h * a.k_hs + i0, static_cast<const T*>(a.v) + t * a.v_ts + h * a.v_hs + i0};
  const int64_t hs[2] = {a.k_hs, a.v_hs};
  uint32_t x[U][2][8];
  auto load = [&](int n, bool there) {   // heads h + n; ahead of the chain that finds the place
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int i = 0; i < 8; ++i) x[n][c][i] = 0;
      if (there) load16(from[c] + n * hs[c], a.by, x[n][c]);
    }
  };
#pragma unroll
  for (int n = 0; n < U; ++n) load(n, mine && h + n < h_end);
  const int b0 = a.kv.starts ? sequences_before(a.kv, (int)t0) : 0;
  int64_t row = -1;
  if (mine) {
    const int b = sequence_from(a.kv, b0, (int)t);
    if (b >= 0) {
      int first, count;
      sequence_rows(a.kv, b, first, count);
      const int64_t slot = slot_of(a.kv, b, (int64_t)a.kv.lens[b] - count + ((int)t - first));
      if (slot >= 0) row = pool_row(a.kv, slot, h);
    }
  }
  const Scale4 places(a.D);
  const int64_t to0 = max(row, (int64_t)0) * (a.D >> 1) + (i0 >> 1), scale0 = places.row(max(row, (int64_t)0)), factor0 = places.factor(max(row, (int64_t)0), lane >> 2);
  const int64_t to_step = (int64_t)(a.D >> 1) << a.kv.page_log2, scale_step = (int64_t)places.record() << (a.kv.page_log2 - 4);
#pragma unroll 1
  for (int done = 0;; ) {
#pragma unroll
    for (int n = 0; n < U; ++n) {
      const bool stored = row >= 0 && h + n < h_end;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t top = top16(x[n][c]);
#pragma unroll
        for (int o = 1; o < lanes && o < 4; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
        uint32_t most = top;
#pragma unroll
        for (int o = 4; o < lanes; o <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        const float group = unpack2<T>(top).x, all = unpack2<T>(most).x;
        uint32_t byte, codes[2] = {0x88888888u, 0x88888888u};   // zeros
        float scale;
        const float per = quantiser4(group, all, byte, scale);
        if (per != 0.f) {
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 y = unpack2<T>(x[n][c][4 * j + i]);
              f[2 * i] = y.x;
              f[2 * i + 1] = y.y;
            }
            codes[j] = codes8(f, per);
          }
        }
        if (!stored) continue;
        uint8_t* scales = reinterpret_cast<uint8_t*>(const_cast<float*>(c ? a.kv.v_scale : a.kv.k_scale)) + (done + n) * scale_step;
        uint8_t* to = static_cast<uint8_t*>(const_cast<void*>(c ? a.kv.v : a.kv.k)) + (done + n) * to_step + to0;
        *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
        if (!(lane & 3)) scales[factor0] = (uint8_t)byte;
        if (lane == 0) *reinterpret_cast<float*>(scales + scale0) = scale;
      }
    }
    h += U;
    done += U;
    if (h >= h_end) break;
    from[0] += U * hs[0];
    from[1] += U * hs[1];
#pragma unroll
    for (int n = 0; n < U; ++n) load(n, mine && h + n < h_end);
  }
}

template <typename T, int L, int U>
__global__ void __launch_bounds__(kThreads, 5) load4_kernel(const __grid_constant__ Args4 a) {
  pdl_wait();
  pdl_trigger();
  constexpr int groups = kThreads >> L;
  const int lane = threadIdx.x & ((1 << L) - 1), i0 = 16 * lane;
  const int64_t t0 = (int64_t)blockIdx.x * groups, t = t0 + (threadIdx.x >> L);
  const int h0 = blockIdx.y * a.heads_per, h_end = min(a.kv.heads, h0 + a.heads_per);
  const int b0 = sequences_before(a.kv, (int)t0);
  if (t >= a.tokens || i0 >= a.D) return;
  const int b = sequence_from(a.kv, b0, (int)t);
  int64_t row = -1;
  if (b >= 0) {
    const int64_t slot = slot_of(a.kv, b, t - a.kv.starts[b]);
    if (slot >= 0) row = pool_row(a.kv, slot, h0);
  }
  const Scale4 places(a.D);
  const int64_t from = max(row, (int64_t)0) * (a.D >> 1) + (i0 >> 1), factor = places.factor(max(row, (int64_t)0), lane >> 2),
                scale = places.row(max(row, (int64_t)0));
  const int64_t from_step = (int64_t)(a.D >> 1) << a.kv.page_log2, scale_step = (int64_t)places.record() << (a.kv.page_log2 - 4);
  const int64_t to = (t * a.kv.heads + h0) * a.D + i0;
#pragma unroll 1
  for (int done = 0; h0 + done < h_end; done += U) {
    uint2 x[U][2];
    float step[U][2];
    uint32_t byte[U][2];
#pragma unroll
    for (int n = 0; n < U; ++n)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        x[n][c] = make_uint2(0x88888888u, 0x88888888u);   // codes of 0: rows that are not there are +0, as in other caches
        step[n][c] = 0.f;
        byte[n][c] = 0;
        if (row < 0 || h0 + done + n >= h_end) continue;
        const uint8_t* scales = reinterpret_cast<const uint8_t*>(c ? a.kv.v_scale : a.kv.k_scale) + (done + n) * scale_step;
        x[n][c] = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(c ? a.kv.v : a.kv.k) + (done + n) * from_step + from);
        byte[n][c] = scales[factor];
        step[n][c] = *reinterpret_cast<const float*>(scales + scale);
      }
#pragma unroll
    for (int n = 0; n < U; ++n) {
      if (h0 + done + n >= h_end) continue;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float by = e4m3_value(byte[n][c]) * step[n][c];
        uint32_t y[8];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t w = j ? x[n][c].y : x[n][c].x;
          float f[8];
#pragma unroll
          for (int i = 0; i < 4; ++i) {   // values i and i + 4
            const uint32_t q = (w >> (4 * i) & 0x000f000fu) | 0x64006400u, bias = 0x64086408u;   // 1024 + code + 8, 1032
            const float2 z = __half22float2(__hsub2(*reinterpret_cast<const __half2*>(&q), *reinterpret_cast<const __half2*>(&bias)));
            f[i] = z.x * by;
            f[i + 4] = z.y * by;
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) y[4 * j + i] = pack2<T>(f[2 * i], f[2 * i + 1]);
        }
        put16(static_cast<T*>(c ? a.v_out : a.k_out) + to + (int64_t)(done + n) * a.D, a.by, y);
      }
    }
  }
}

// Blocks: a token per lane group; few tokens' heads are spread over blocks, two a block at least.
// f(type, log2 of the lanes) -> kernel
template <typename F>
int launch4(F f, bool half, Args4& a, cudaStream_t st) {
  using std::integral_constant;
  int l = 1;
  while ((16 << l) < a.D) ++l;
  const int64_t per = kThreads >> l, blocks = (a.tokens + per - 1) / per;
  if (blocks > 0x7fffffff) return VQ2_ERR_SHAPE;
  const int64_t want = (16 * sm_count() + blocks - 1) / blocks, most = (a.kv.heads + 1) / 2, parts = want < most ? want : most;
  a.heads_per = (int)((a.kv.heads + parts - 1) / parts);
  if (a.heads_per % 2 && a.heads_per < a.kv.heads) ++a.heads_per;
  auto typed = [&](auto type) {
    return l == 1 ? f(type, integral_constant<int, 1>()) : l == 2 ? f(type, integral_constant<int, 2>())
                                                          : l == 3 ? f(type, integral_constant<int, 3>()) : f(type, integral_constant<int, 4>());
  };
  const auto kern = half ? typed(__half()) : typed(__nv_bfloat16());
  return launch_kernel(kern, dim3((unsigned)blocks, (unsigned)((a.kv.heads + a.heads_per - 1) / a.heads_per)), dim3(kThreads), 0, st, a);
}

constexpr int kStoreHeads = 2, kLoadHeads = 2;   // of a lane group at a time

}  // namespace

int launch_store4(const PagedKV& kv, const void* k, int64_t k_ts, int64_t k_hs, const void* v, int64_t v_ts, int64_t v_hs,
                  bool half, int64_t tokens, int64_t D, cudaStream_t st) {
  Args4 a = {};
  a.kv = kv;
  a.k = k;
  a.v = v;
  a.k_ts = k_ts;
  a.k_hs = k_hs;
  a.v_ts = v_ts;
  a.v_hs = v_hs;
  const uintptr_t all = reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) | 2 * (k_ts | k_hs | v_ts | v_hs);
  a.by = all % 32 == 0 ? 32 : all % 16 == 0 ? 16 : 2;
  a.tokens = tokens;
  a.D = (int)D;
  return launch4([](auto t, auto l) { return store4_kernel<decltype(t), decltype(l)::value, kStoreHeads>; }, half, a, st);
}

int launch_load4(const PagedKV& kv, void* k, void* v, bool half, int64_t tokens, int64_t D, cudaStream_t st) {
  Args4 a = {};
  a.kv = kv;
  a.k_out = k;
  a.v_out = v;
  a.by = aligned(k, 32) && aligned(v, 32) ? 32 : 16;
  a.tokens = tokens;
  a.D = (int)D;
  return launch4([](auto t, auto l) { return load4_kernel<decltype(t), decltype(l)::value, kLoadHeads>; }, half, a, st);
}

}  // namespace vq2
