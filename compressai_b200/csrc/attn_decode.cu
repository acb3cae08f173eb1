// Attention of few query rows per key/value head over a paged cache: the decode step.
//
// A cached key and value are read once for all rows that share them (G query heads times the new
// tokens, 8 * NT rows a block), so at one new token a byte of cache buys about G flops: HBM bounds
// it, and the kernel's work is to keep loads in flight. A warp takes 16 keys a step, computes
//
//   S^T [16 keys x 8 rows] = K Q^T,   P = 2^(S - m),   O^T [D x 8 rows] += V^T P^T
//
// with mma.m16n8k16 and its own running maximum m and sum; warps, and blocks that split a long
// sequence, are joined at the end. The keys stand on the MMA's 16 side, so 8 rows waste nothing,
// and the maximum and sum of a row live in the lanes that hold its column of O^T.
//
// Every MMA fragment is 16 consecutive bytes of one cached row per lane: the order of the summed
// index (D for S, keys for O) and of O's rows is free, so each lane takes the values it has. A lane
// therefore copies (cp.async) exactly the bytes that it will itself read, into a ring of its own in
// shared memory (slot [piece][lane], conflict-free): no barriers, no transposed loads, and the data
// in flight cost no registers.
//   K piece: rows g, g + 8 (g = lane / 4), 16 bytes at column 16 bytes * (4 k + t), t = lane % 4.
//   V piece: rows 2t, 2t + 1, 2t + 8, 2t + 9, 16 bytes at 16 bytes * (8 c + g); two rows' values are
//     interleaved into (key, key + 1) pairs by byte permutes.
//
// 8-bit caches: an int8 is exact in fp16 (1024 + u - 1152 with u = v + 128 placed in the mantissa),
// so both products run in fp16 without loss, the scales outside: the key's into the score, the
// value's into P, relative to a power of two at least the largest seen (vref) so that P stays in
// fp16's range. bf16 queries become fp16 by a power of two per row, exact down to 2^-28 of the
// row's largest value.
//
// Rescaling is lazy: m moves only when a score passes it by 8 powers of two, so P is at most 256 --
// in range for fp16 -- and the usual step has no shuffles beyond one vote. P is rounded to the
// cache's 16 bits (fp16 for int8) for the second product; maxima, sums and O are 32 bits.
#include <atomic>
#include <type_traits>

#include "attn_dev.cuh"

namespace vq2 {
namespace {

__device__ __forceinline__ uint32_t smem32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// 16 bytes to shared memory, zeros when !ok (src is then any valid address).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(ok ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t dst, const void* src, bool ok) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(ok ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  if (std::is_same<T, __half>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
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

// Shapes of one variant. DP: head size rounded up (values past D are zeros); NT: 8-row tiles.
template <int DP, int NT, bool I8>
struct DecodeShape {
  static constexpr int kKP = I8 ? DP / 64 : DP / 32;    // 16-byte K pieces a row and lane
  static constexpr int kVC = I8 ? DP / 128 : DP / 64;   // 16-byte V pieces a row and lane
  static constexpr int kPieces = 2 * kKP + 4 * kVC + (I8 ? 1 : 0);
  static constexpr int kStage = kPieces * 512;          // a warp's bytes per 16 keys
  // About 100 KB a block, two blocks an SM: one block's start and end hide behind the other's stream.
  static constexpr int kWarps = DP == 256 && !I8 ? 2 : 4;
  static constexpr int kBudget = 106496 / (kWarps * kStage);
  static constexpr int kStages = kBudget > 6 ? 6 : kBudget;
  static_assert(kStages >= 3, "two tiles in flight a warp");
  static constexpr int kQ = NT * (DP / 32) * 512;       // query fragments
  static constexpr int kJoin = kWarps * NT * 8 * (DP + 4) * 4;   // the warps' O, over the ring
  static constexpr int kRing = kWarps * kStages * kStage;
  static constexpr int kSmem = kQ + (kRing > kJoin ? kRing : kJoin);
};

template <int DP, int NT, bool I8, typename T>
__global__ void __launch_bounds__(DecodeShape<DP, NT, I8>::kWarps * 32)
    attn_decode_kernel(const AttnArgs a) {
  using S = DecodeShape<DP, NT, I8>;
  using M = typename std::conditional<I8, __half, T>::type;  // type of the products
  extern __shared__ __align__(16) unsigned char sm[];
  __shared__ float2 ml_s[S::kWarps][NT * 8];
  __shared__ float qexp_s[NT * 8];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.y, h = blockIdx.z;
  const int b = blockIdx.x / a.row_blocks, rb = blockIdx.x - b * a.row_blocks;
  const AttnRows w = attn_rows(a, b, rb);
  if (w.rows <= 0) return;
  int lo, hi;
  block_keys(a, w, lo, hi);
  const int s0 = lo + split * a.chunk, s1 = min(hi, s0 + a.chunk);
  if (split > 0 && s0 >= hi) return;   // split 0 stays: it writes the rows that see nothing
  const bool alone = hi - lo <= a.chunk;
  const int tiles = s1 > s0 ? (s1 - s0 + 15) >> 4 : 0;

  // ---- the ring: copies of the 16 keys of tile n of this block
  const uint32_t q_sm = smem32(sm), ring = q_sm + S::kQ + warp * S::kStages * S::kStage + lane * 16;
  const int32_t* table = a.kv.table + b * a.kv.table_stride;
  const int page_mask = (1 << a.kv.page_log2) - 1;
  auto page_of = [&](int n) { return n < tiles ? table[(s0 + 16 * n) >> a.kv.page_log2] : -1; };
  uint32_t gone = 0;   // stages whose page id is outside the pool: their keys do not exist
  auto fetch = [&](int n, int stage, int page) {
    const int k0 = s0 + 16 * n;
    const bool there = page >= 0 && page < a.kv.pages;
    gone = (gone & ~(1u << stage)) | ((there ? 0u : 1u) << stage);
    const int64_t row0 = there ? (((int64_t)page * a.kv.heads + h) << a.kv.page_log2) + (k0 & page_mask) : 0;
    const uint32_t dst = ring + stage * S::kStage;
    constexpr int E = I8 ? 1 : 2;
    const int left = there ? s1 - k0 : 0;   // rows of the tile that are in the sequence
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const bool ok = g + 8 * r < left;
      const char* src = static_cast<const char*>(a.kv.k) + ((row0 + (ok ? g + 8 * r : 0)) * a.D) * E + 16 * t;
#pragma unroll
      for (int k = 0; k < S::kKP; ++k) {
        const bool in = ok && (64 / E) * k + (16 / E) * t < a.D;
        copy16(dst + (r * S::kKP + k) * 512, in ? src + 64 * k : a.kv.k, in);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int key = 2 * t + (r & 1) + 8 * (r >> 1);
      const bool ok = key < left;
      const char* src = static_cast<const char*>(a.kv.v) + ((row0 + (ok ? key : 0)) * a.D) * E + 16 * g;
#pragma unroll
      for (int c = 0; c < S::kVC; ++c) {
        const bool in = ok && (128 / E) * c + (16 / E) * g < a.D;
        copy16(dst + (2 * S::kKP + r * S::kVC + c) * 512, in ? src + 128 * c : a.kv.v, in);
      }
    }
    if (I8) {  // scales of keys g, g + 8: K, V
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const bool ok = g + 8 * r < left;
        const int64_t row = row0 + (ok ? g + 8 * r : 0);
        copy4(dst + (S::kPieces - 1) * 512 + 4 * r, a.kv.k_scale + row, ok);
        copy4(dst + (S::kPieces - 1) * 512 + 8 + 4 * r, a.kv.v_scale + row, ok);
      }
    }
  };
  int next = warp, page = page_of(next);
#pragma unroll
  for (int j = 0; j < S::kStages - 1; ++j) {
    const int following = page_of(next + S::kWarps);
    if (next < tiles) fetch(next, j, page);
    copy_commit();
    next += S::kWarps;
    page = following;
  }

  // ---- queries as B fragments, in the order of K's pieces: [NT][DP / 32] x 16 bytes a lane
  for (int i = warp; i < NT; i += S::kWarps) {
    const int r = w.r0 + 8 * i + g;
    const bool ok = 8 * i + g < w.rows;
    const char* src = static_cast<const char*>(a.q);
    if (ok) src += ((w.first + r / a.G) * a.q_ts + (h * a.G + r % a.G) * a.q_hs) * 2;
    uint4 v[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) {
      // 16-bit cache: piece k holds d = 32 k + 8 t ..; int8: pieces 2k, 2k + 1 hold d = 64 k + 16 t ..
      const int d = I8 ? 64 * (k >> 1) + 16 * t + 8 * (k & 1) : 32 * k + 8 * t;
      v[k] = make_uint4(0, 0, 0, 0);
      if (ok && d < a.D) v[k] = *reinterpret_cast<const uint4*>(src + 2 * d);
    }
    if (I8) {
      float back = 1.f;
      if (a.q_bf16) {
        float top = 0.f;
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2<__nv_bfloat16>((&v[k].x)[j]);
            top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // largest value into [2^13, 2^14); exponents of the row's largest outside +-100 stay as they are
        int e = 0;
        if (top > 1e-30f && top < 1e30f) e = 13 - ilogbf(top);
        const float by = __int_as_float((127 + e) << 23);
        back = __int_as_float((127 - e) << 23);
#pragma unroll
        for (int k = 0; k < DP / 32; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 f = unpack2<__nv_bfloat16>((&v[k].x)[j]);
            (&v[k].x)[j] = pack2<__half>(f.x * by, f.y * by);
          }
      }
      if (t == 0) qexp_s[8 * i + g] = back;
    }
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) *reinterpret_cast<uint4*>(sm + (i * (DP / 32) + k) * 512 + lane * 16) = v[k];
  }
  __syncthreads();

  // ---- this lane's two rows of each tile (columns 2t, 2t + 1 of S^T): what they see
  int klo[NT][2], khi[NT][2];
  float sc[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = 8 * i + 2 * t + c;
      const bool ok = r < w.rows;
      const int tok = (w.r0 + (ok ? r : 0)) / a.G;
      klo[i][c] = row_lo(a, w, tok);
      khi[i][c] = ok ? row_hi(a, w, tok) : 0;
      sc[i][c] = a.scale_log2 * (I8 ? qexp_s[r] : 1.f);
    }
  // keys that every row sees need no mask
  const int all_lo = row_lo(a, w, (w.r0 + w.rows - 1) / a.G), all_hi = row_hi(a, w, w.r0 / a.G);

  float o[NT][DP / 16][4], m[NT][2], l[NT][2], vref = 0.f, vinv = 0.f;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
#pragma unroll
    for (int j = 0; j < DP / 16; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][j][c] = 0.f;
    m[i][0] = m[i][1] = -INFINITY;
    l[i][0] = l[i][1] = 0.f;
  }

  int stage = 0;
  for (int n = warp; n < tiles; n += S::kWarps) {
    copy_wait<S::kStages - 2>();
    const uint32_t src = ring + stage * S::kStage;
    // ---- S^T = K Q^T; two sums per tile, so that no MMA waits for the one before it
    float s[NT][2][4];
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[i][0][c] = s[i][1][c] = 0.f;
#pragma unroll
    for (int k = 0; k < S::kKP; ++k) {
      uint4 k0 = lds16(src + k * 512), k1 = lds16(src + (S::kKP + k) * 512);
      if (I8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t x = (&k0.x)[j] ^ 0x80808080u, y = (&k1.x)[j] ^ 0x80808080u;
          const uint32_t a0 = bytes_f16(x, 0x4140), a2 = bytes_f16(x, 0x4342);
          const uint32_t a1 = bytes_f16(y, 0x4140), a3 = bytes_f16(y, 0x4342);
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint32_t qa = q_sm + (i * (DP / 32) + 2 * k + (j >> 1)) * 512 + lane * 16 + 8 * (j & 1);
            uint32_t b0, b1;
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(b0), "=r"(b1) : "r"(qa));
            mma16816<M>(s[i][j & 1], a0, a1, a2, a3, b0, b1);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          const uint4 q = lds16(q_sm + (i * (DP / 32) + k) * 512 + lane * 16);
          mma16816<M>(s[i][0], k0.x, k1.x, k0.y, k1.y, q.x, q.y);
          mma16816<M>(s[i][1], k0.z, k1.z, k0.w, k1.w, q.z, q.w);
        }
      }
    }
    float ks[2] = {1.f, 1.f}, vs[2] = {1.f, 1.f};
    if (I8) {
      const uint4 f = lds16(src + (S::kPieces - 1) * 512);
      ks[0] = __uint_as_float(f.x);
      ks[1] = __uint_as_float(f.y);
      vs[0] = __uint_as_float(f.z);
      vs[1] = __uint_as_float(f.w);
    }
    // ---- scores, masks
    const int k0 = s0 + 16 * n;
    const bool none = (gone >> stage) & 1;
    const bool whole = k0 >= all_lo && k0 + 16 <= all_hi && k0 + 16 <= s1 && !none;
    bool high = false;
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        float v = (s[i][0][c] + s[i][1][c]) * (sc[i][c & 1] * ks[c >> 1]);
        if (!whole) {
          const int key = k0 + g + 8 * (c >> 1);
          if (none || key >= s1 || key < klo[i][c & 1] || key >= khi[i][c & 1]) v = -INFINITY;
        }
        s[i][0][c] = v;
        high |= v > m[i][c & 1] + 8.f;
      }
    if (__any_sync(0xffffffffu, high)) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = fmaxf(s[i][0][c], s[i][0][c + 2]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          const float mn = fmaxf(m[i][c], x);
          const float by = mn == -INFINITY ? 1.f : ex2(m[i][c] - mn);
          m[i][c] = mn;
          l[i][c] *= by;
#pragma unroll
          for (int j = 0; j < DP / 16; ++j) {
            o[i][j][c] *= by;
            o[i][j][c + 2] *= by;
          }
        }
    }
    if (I8 && __any_sync(0xffffffffu, fmaxf(vs[0], vs[1]) > vref)) {
      float x = fmaxf(vs[0], vs[1]);
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
      x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
      // the power of two above it; at most 2^120, so that its inverse is a normal number too
      const float ref = fminf(fmaxf(__uint_as_float((__float_as_uint(x) & 0x7f800000u) + 0x00800000u), vref), 1.3e36f);
      const float by = vref * (1.f / ref);
      vref = ref;
      vinv = 1.f / ref;
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int j = 0; j < DP / 16; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[i][j][c] *= by;
    }
    // ---- P^T: columns summed, then turned into B fragments
    uint32_t p0[NT], p1[NT];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      float p[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float base = m[i][c & 1] == -INFINITY ? 0.f : m[i][c & 1];
        p[c] = ex2(s[i][0][c] - base);
        l[i][c & 1] += p[c];
        if (I8) p[c] = p[c] > 0.f ? p[c] * (vs[c >> 1] * vinv) : 0.f;  // a masked key's scale may be anything
      }
      p0[i] = transpose8x8(pack2<M>(p[0], p[1]));
      p1[i] = transpose8x8(pack2<M>(p[2], p[3]));
    }
    // ---- O^T += V^T P^T
#pragma unroll
    for (int c = 0; c < S::kVC; ++c) {
      uint4 v[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) v[r] = lds16(src + (2 * S::kKP + r * S::kVC + c) * 512);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (I8) {
          const uint32_t x0 = (&v[0].x)[j] ^ 0x80808080u, x1 = (&v[1].x)[j] ^ 0x80808080u;
          const uint32_t x2 = (&v[2].x)[j] ^ 0x80808080u, x3 = (&v[3].x)[j] ^ 0x80808080u;
#pragma unroll
          for (int e = 0; e < 2; ++e) {  // values 4 j + 2 e, 4 j + 2 e + 1 of the piece
            const uint32_t lo2 = __byte_perm(x0, x1, e ? 0x7362 : 0x5140);
            const uint32_t hi2 = __byte_perm(x2, x3, e ? 0x7362 : 0x5140);
            const uint32_t a0 = bytes_f16(lo2, 0x4140), a1 = bytes_f16(lo2, 0x4342);
            const uint32_t a2 = bytes_f16(hi2, 0x4140), a3 = bytes_f16(hi2, 0x4342);
#pragma unroll
            for (int i = 0; i < NT; ++i) mma16816<M>(o[i][c * 8 + 2 * j + e], a0, a1, a2, a3, p0[i], p1[i]);
          }
        } else {
          const uint32_t a0 = __byte_perm((&v[0].x)[j], (&v[1].x)[j], 0x5410);
          const uint32_t a1 = __byte_perm((&v[0].x)[j], (&v[1].x)[j], 0x7632);
          const uint32_t a2 = __byte_perm((&v[2].x)[j], (&v[3].x)[j], 0x5410);
          const uint32_t a3 = __byte_perm((&v[2].x)[j], (&v[3].x)[j], 0x7632);
#pragma unroll
          for (int i = 0; i < NT; ++i) mma16816<M>(o[i][c * 4 + j], a0, a1, a2, a3, p0[i], p1[i]);
        }
      }
    }
    // ---- refill the stage read one step ago
    int into = stage + S::kStages - 1;
    if (into >= S::kStages) into -= S::kStages;
    const int following = page_of(next + S::kWarps);
    if (next < tiles) fetch(next, into, page);
    copy_commit();
    next += S::kWarps;
    page = following;
    if (++stage == S::kStages) stage = 0;
  }
  copy_wait<0>();
  __syncthreads();   // every warp is done with its ring: O takes its place

  // ---- join the warps: maximum, then sums relative to it
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float x = l[i][c];
      x += __shfl_xor_sync(0xffffffffu, x, 4);
      x += __shfl_xor_sync(0xffffffffu, x, 8);
      x += __shfl_xor_sync(0xffffffffu, x, 16);
      if (g == 0) ml_s[warp][8 * i + 2 * t + c] = make_float2(m[i][c], x);
    }
  float* acc = reinterpret_cast<float*>(sm + S::kQ);   // [warp][row][DP + 4]
  constexpr int LD = DP + 4;
  const float undo = I8 ? vref : 1.f;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      // rows g, g + 8 of the MMA tile are the values d, d + 1
      const int d = I8 ? 128 * (j >> 3) + 16 * g + 2 * (j & 7) : 64 * (j >> 2) + 8 * g + 2 * (j & 3);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float2* dst = reinterpret_cast<float2*>(acc + (warp * NT * 8 + 8 * i + 2 * t + c) * LD + d);
        *dst = make_float2(o[i][j][c] * undo, o[i][j][c + 2] * undo);
      }
    }
  __syncthreads();
  const int vecs = a.D >> 2;
  for (int e = threadIdx.x; e < w.rows * vecs; e += blockDim.x) {
    const int r = e / vecs, d = (e - r * vecs) * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int k = 0; k < S::kWarps; ++k) top = fmaxf(top, ml_s[k][r].x);
    const float base = top == -INFINITY ? 0.f : top;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < S::kWarps; ++k) {
      const float by = ex2(ml_s[k][r].x - base);
      const float4 y = *reinterpret_cast<const float4*>(acc + (k * NT * 8 + r) * LD + d);
      sum += ml_s[k][r].y * by;
      x.x += y.x * by;
      x.y += y.y * by;
      x.z += y.z * by;
      x.w += y.w * by;
    }
    const int row = w.r0 + r;
    const int64_t at = (int64_t)(w.first + row / a.G) * a.hq + h * a.G + row % a.G;
    if (alone) {
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      const uint2 y = make_uint2(pack2<T>(x.x * inv, x.y * inv), pack2<T>(x.z * inv, x.w * inv));
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.D + d) = y;
      if (a.lse && d == 0) a.lse[at] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * kLn2;
    } else {
      *reinterpret_cast<float4*>(a.part_o + (at * a.splits + split) * a.D + d) = x;
      if (d == 0) a.part_ml[at * a.splits + split] = make_float2(top, sum);
    }
  }
}

// Joins the splits of one row (token, head) a block: the warps' share of splits, then theirs.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
  __shared__ float4 acc[256];
  __shared__ float by_s[64];
  __shared__ float lse_s;
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x, hq = blockIdx.y;
  const int b = sequence_of(a.kv, t);
  const int64_t at = (int64_t)t * a.hq + hq;
  if (b < 0) return;
  int first, count, lo, hi;
  sequence_rows(a.kv, b, first, count);
  block_keys(a, attn_rows(a, b, ((t - first) * a.G + hq % a.G) / a.rows_per_block), lo, hi);
  if (hi - lo <= a.chunk) return;   // written already
  const int n = (hi - lo + a.chunk - 1) / a.chunk;
  const int vecs = a.D >> 2;
  if (threadIdx.x < 32) {
    const int i = threadIdx.x;
    const float2 x = i < n ? a.part_ml[at * a.splits + i] : make_float2(-INFINITY, 0.f);
    const float2 y = i + 32 < n ? a.part_ml[at * a.splits + i + 32] : make_float2(-INFINITY, 0.f);
    float top = fmaxf(x.x, y.x);
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    const float base = top == -INFINITY ? 0.f : top;
    float sum = x.y * ex2(x.x - base) + y.y * ex2(y.x - base);
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    by_s[i] = ex2(x.x - base) * inv;
    by_s[i + 32] = ex2(y.x - base) * inv;
    if (i == 0) lse_s = sum == 0.f ? -INFINITY : (base + log2f(sum)) * kLn2;
  }
  __syncthreads();
  const int parts = blockDim.x / vecs, part = threadIdx.x / vecs, e = threadIdx.x - part * vecs;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
  if (part < parts) {
#pragma unroll 4
    for (int i = part; i < n; i += parts) {
      const float by = by_s[i];
      const float4 y = *reinterpret_cast<const float4*>(a.part_o + (at * a.splits + i) * a.D + 4 * e);
      x.x += y.x * by;
      x.y += y.y * by;
      x.z += y.z * by;
      x.w += y.w * by;
    }
    acc[threadIdx.x] = x;
  }
  __syncthreads();
  if (part == 0) {
    for (int k = 1; k < parts; ++k) {
      const float4 y = acc[k * vecs + e];
      x.x += y.x;
      x.y += y.y;
      x.z += y.z;
      x.w += y.w;
    }
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.D + 4 * e) = make_uint2(pack2<T>(x.x, x.y), pack2<T>(x.z, x.w));
    if (a.lse && threadIdx.x == 0) a.lse[at] = lse_s;
  }
}

template <int DP, int NT, bool I8, typename T>
int launch(const AttnArgs& a, cudaStream_t st) {
  using S = DecodeShape<DP, NT, I8>;
  auto kern = attn_decode_kernel<DP, NT, I8, T>;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(done.load() & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem);
    if (e != cudaSuccess) {
      set_last_cuda_error(e);
      return VQ2_ERR_LAUNCH;
    }
    done.fetch_or(bit);
  }
  const dim3 grid((unsigned)(a.kv.seqs * a.row_blocks), (unsigned)a.splits, (unsigned)a.kv.heads);
  return launch_kernel(kern, grid, dim3(S::kWarps * 32), S::kSmem, st, a);
}

template <bool I8, typename T>
int launch_shape(const AttnArgs& a, cudaStream_t st) {
  const int nt = a.rows_per_block / 8;
  if (a.D > 128) return nt == 1 ? launch<256, 1, I8, T>(a, st) : launch<256, 2, I8, T>(a, st);
  if (I8 || a.D > 64)
    return nt == 1 ? launch<128, 1, I8, T>(a, st) : nt == 2 ? launch<128, 2, I8, T>(a, st) : launch<128, 4, I8, T>(a, st);
  return nt == 1 ? launch<64, 1, false, T>(a, st) : nt == 2 ? launch<64, 2, false, T>(a, st) : launch<64, 4, false, T>(a, st);
}

}  // namespace

void plan_attn_decode(AttnArgs& a, int64_t max_new, int64_t max_len) {
  // Rows of a block: all that share a key, up to the accumulators that registers hold.
  const int64_t rows = max_new * a.G;
  const int cap = a.D > 128 ? 2 : 4;
  int nt = 1;
  while (nt < cap && 8 * nt < rows) nt *= 2;
  a.rows_per_block = 8 * nt;
  a.row_blocks = (int)((rows + 8 * nt - 1) / (8 * nt));
  if (a.row_blocks < 1) a.row_blocks = 1;
  a.lo_mask = ~15;
  // Split the keys until there are four rounds of blocks (two an SM): ragged lengths then even out.
  // A split is at least 64 keys (a warp's latency to start is about what 64 keys take) and there
  // are at most 64 of them.
  int64_t keys = max_len;
  if (a.window && a.window + max_new + 16 < keys) keys = a.window + max_new + 16;
  const int64_t blocks = (int64_t)a.kv.seqs * a.kv.heads * a.row_blocks;
  const int64_t want = (8 * (int64_t)sm_count() + blocks - 1) / blocks;
  int64_t chunk = (keys + want - 1) / want;
  if (chunk < (keys + 15 + 63) / 64) chunk = (keys + 15 + 63) / 64;   // the first key is rounded down by up to 15
  if (chunk < 64) chunk = 64;
  chunk = (chunk + 15) & ~int64_t(15);
  a.chunk = (int)chunk;
  a.splits = (int)((keys + 15 + chunk - 1) / chunk);
  if (a.splits < 1) a.splits = 1;
}

int launch_attn_decode(const AttnArgs& a, bool i8, cudaStream_t st) {
  if (i8) return a.q_bf16 ? launch_shape<true, __nv_bfloat16>(a, st) : launch_shape<true, __half>(a, st);
  return a.q_bf16 ? launch_shape<false, __nv_bfloat16>(a, st) : launch_shape<false, __half>(a, st);
}

int launch_attn_join(const AttnArgs& a, cudaStream_t st) {
  const dim3 grid((unsigned)a.T, (unsigned)a.hq), block(256);
  return a.q_bf16 ? launch_kernel(attn_join_kernel<__nv_bfloat16>, grid, block, 0, st, a)
                  : launch_kernel(attn_join_kernel<__half>, grid, block, 0, st, a);
}

}  // namespace vq2
