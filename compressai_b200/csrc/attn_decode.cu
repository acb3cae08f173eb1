// Attention of few query rows per key/value head over a paged cache: the decode step.
//
// A cached key and value are read once for all rows that share them (G query heads times the new
// tokens, 8 * NT rows a block), so at one new token a byte of cache buys about G flops: HBM bounds
// it, and the kernel's work is to keep loads in flight. A warp takes 16 or 32 keys a step, computes per 16
//
//   S^T [16 keys x 8 rows] = K Q^T,   P = 2^(S - m),   O^T [D x 8 rows] += V^T P^T
//
// with mma.m16n8k16 and its own running maximum m and sum; warps, and blocks that split a long
// sequence, are joined at the end. The keys stand on the MMA's 16 side, so 8 rows waste nothing,
// and the maximum and sum of a row live in the lanes that hold its column of O^T.
//
// Every MMA fragment is 16 consecutive bytes of one cached row per lane: the order of the summed
// index (D for S, keys for O) and of O's rows is free, so each lane takes the values it has and no
// load is transposed. With g = lane / 4, t = lane % 4, in 128-byte pieces of a row:
//   K: rows g, g + 8, 16-byte chunks 2t and 2t + 1;
//   V: rows 2t, 2t + 1, 2t + 8, 2t + 9, chunk g; byte permutes pair the values of two keys.
// The 16 rows of a tile lie together in their page: TMA brings them as boxes of rows x 128 bytes
// into a ring of the warp's own, and with the 128-byte swizzle all of these reads are free of bank
// conflicts. K and V are separate entries of the ring (a slot is refilled as soon as its half is
// used), a warp waits for nobody but its copies, and the loads in flight cost no registers.
// (64 sequences of 800 to 8000 tokens, 16/2 heads of 256: 101 us, 5.7 TB/s; with cp.async by the lanes,
// 32 copies a lane and tile whose addresses alone were half of the instructions, 145.)
//
// 8-bit caches: an int8 is exact in fp16 (1024 + u - 1152 with u = v + 128 placed in the mantissa),
// so both products run in fp16 without loss, the scales outside: the key's into the score, the
// value's into P, relative to a power of two above the largest that the row has seen (vref) so that P
// stays in fp16's range. bf16 queries become fp16 by a power of two per row, exact down to 2^-28 of the
// row's largest value.
//
// Rescaling is lazy: m moves only when a score passes it by 8 powers of two, so P is at most 256 (fp16:
// 2^15, see kLift) and the usual step has no shuffles beyond one vote. P is rounded to the
// cache's 16 bits (fp16 for int8) for the second product; maxima, sums and O are 32 bits.
#include <atomic>
#include <type_traits>

#include "attn_dev.cuh"
#include "tcgen05.cuh"

// Sticky status of the decode kernel: VQ2_ERR_TIMEOUT once a bounded wait for a copy gave up.
__device__ int32_t g_decode_status;

namespace vq2 {
namespace {

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

// Shapes of one variant. DP: head size rounded up (values past D are zeros); NT: 8-row tiles.
template <int DP, int NT, bool I8>
struct DecodeShape {
  static constexpr int kC = I8 ? DP / 128 : DP / 64;    // 128-byte pieces of a row
  static constexpr int kU = DP == 256 ? 1 : 2;          // 16-key tiles a step, as registers allow
  static constexpr int kKeys = 16 * kU;
  static constexpr int kBox = kKeys * 128;              // bytes of one piece of a step's keys
  static constexpr int kHalf = kC * kBox;               // K or V of a step
  static constexpr int kWarps = 4;
  // Blocks an SM: two and more, so that one's start and end hide behind another's stream. 8-bit tiles
  // are half the bytes for more instructions (the conversion), so they need more warps to cover them.
  static constexpr int kPerSm = I8 && NT == 1 && DP == 128 ? 4 : I8 && NT == 1 ? 3 : 2;
  static constexpr int kFit = (224 * 1024 / kPerSm - 8192) / (kWarps * kHalf);
  static constexpr int kSlots = kFit > 8 ? 8 : kFit;
  static constexpr int kRing = kWarps * kSlots * kHalf;
  static constexpr int kJoin = kWarps * NT * 8 * (DP + 4) * 4;   // the warps' O, over the ring
  static constexpr int kQ = NT * (DP / 32) * 512;       // query fragments
  static constexpr int kScaleStep = 2 * kKeys * 4;      // K's and V's scales of a step
  static constexpr int kScaleSlots = kSlots / 2 + 1;    // steps under way
  static constexpr int kScales = I8 ? kWarps * kScaleSlots * kScaleStep : 0;
  static constexpr int kSmem = 1024 + (kRing > kJoin ? kRing : kJoin) + kQ + kScales;
  static_assert(kSlots >= 3, "a half in use, two in flight");
};

constexpr long long kWaitCycles = 4000000000LL;  // ~2 s at 1.965 GHz

__device__ __forceinline__ bool copy_wait(uint32_t bar, uint32_t parity) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity))
    if (clock64() - t0 > kWaitCycles) {
      atomicMax(&g_decode_status, VQ2_ERR_TIMEOUT);
      return false;
    }
  return true;
}

template <int DP, int NT, bool I8, typename T>
__global__ void __launch_bounds__(DecodeShape<DP, NT, I8>::kWarps * 32, DecodeShape<DP, NT, I8>::kPerSm)
    attn_decode_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using S = DecodeShape<DP, NT, I8>;
  using M = typename std::conditional<I8, __half, T>::type;  // type of the products
  // fp16 weights: 2^7 larger than in bf16, so that those down to 2^-32 of the largest are more than 0
  constexpr bool kHalf = std::is_same<M, __half>::value;
  constexpr float kLift = kHalf ? 7.f : 0.f, kDrop = kHalf ? 1.f / 128.f : 1.f;
  extern __shared__ unsigned char decode_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(decode_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* q_s = sm + (S::kRing > S::kJoin ? S::kRing : S::kJoin);
  __shared__ uint64_t bars[S::kWarps][S::kSlots];
  __shared__ float2 ml_s[S::kWarps][NT * 8];
  __shared__ float qexp_s[NT * 8];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.y, h = blockIdx.z;
  const int b = blockIdx.x / a.row_blocks, rb = blockIdx.x - b * a.row_blocks;
  const AttnRows w = attn_rows(a, b, rb);
  // Behind the first copies where registers allow it: ahead of them it takes 0.2 of 8.8 us of a lone sequence's
  // step; over an 8-bit cache (128 registers) it spills there (four long sequences 143 us for 141).
  auto strays = [&] {
    blank_strays(a, w, b, ((int64_t)rb * a.kv.heads + h) * a.splits + split, (int64_t)a.row_blocks * a.kv.heads * a.splits);
  };
  if (I8 || w.rows <= 0) strays();
  if (w.rows <= 0) return;
  int lo, hi;
  block_keys(a, w, lo, hi);
  if (split > 0 && (int64_t)split * a.chunk >= hi - lo) {   // split 0 stays: it writes the rows that see nothing
    if (!I8) strays();
    return;
  }
  const int s0 = lo + split * a.chunk, s1 = s0 + min(a.chunk, hi - s0);   // no sum past 2^31
  const bool alone = hi - lo <= a.chunk;
  const int tiles = s1 > s0 ? (s1 - s0 + S::kKeys - 1) / S::kKeys : 0;

  // ---- the warp's ring: halves K0 V0 K1 V1 .. of its steps warp, warp + kWarps, ..
  const uint32_t q_sm = su32(q_s), ring = su32(sm) + warp * S::kSlots * S::kHalf, bar0 = su32(&bars[warp][0]);
  const uint32_t scales = q_sm + S::kQ + warp * S::kScaleSlots * S::kScaleStep;
  const int32_t* table = a.kv.table + b * a.kv.table_stride;
  const int page_mask = (1 << a.kv.page_log2) - 1, seen = row_lo(a, w, w.r0 / a.G);
  const int halves = tiles > warp ? 2 * ((tiles - warp + S::kWarps - 1) / S::kWarps) : 0;
  auto key_of = [&](int i) { return s0 + S::kKeys * (warp + S::kWarps * i); };   // first key of the warp's step i
  // A copy is one 128-byte piece of min(page, step) keys: this lane's, and the key it starts at.
  const int box_keys = min(1 << a.kv.page_log2, S::kKeys), piece = lane % S::kC, sub = lane / S::kC * box_keys;
  const bool copies = sub < S::kKeys;
  auto page_of = [&](int i) {   // of this lane's copy; -1 where there is none or its keys are past
    const int k = key_of(i) + (copies ? sub : 0);
    return 2 * i < halves && k < s1 && (k | page_mask) >= seen ? table[k >> a.kv.page_log2] : -1;
  };
  if (lane == 0) {
    for (int i = 0; i < S::kSlots; ++i) mbar_init(bar0 + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  __syncwarp();
  // gone: bit 2 i + u of 32 says that the page of tile u of step i is not in the pool: no such keys
  uint32_t gone = 0;
  int ahead = page_of(0), row = 0;   // page of the lane's next copy; pool row of its present one
  int put = 0, put_slot = 0, put_scale = 0;   // next half to fetch, its slot, its step's place for scales
  auto fetch = [&]() {
    if (put >= halves) return;
    const int i = put >> 1;
    const uint32_t bar = bar0 + 8 * put_slot;
    if (!(put & 1)) {
      const bool there = ahead >= 0 && ahead < a.kv.pages;
      const uint32_t out = __ballot_sync(0xffffffffu, !there);
      const int k = key_of(i);
#pragma unroll
      for (int u = 0; u < S::kU; ++u) {   // of the lane whose copy holds tile u
        const uint32_t bit = (out >> (16 * u / box_keys * S::kC)) & 1;
        const int at = (2 * i + u) & 31;
        gone = (gone & ~(1u << at)) | (bit << at);
      }
      // a page that exists stands in for one that does not
      row = (((there ? ahead : 0) * a.kv.heads + h) << a.kv.page_log2) + ((k + sub) & page_mask);
      ahead = page_of(i + 1);
      if (lane == 0) mbar_arrive_tx(bar, S::kHalf + (I8 ? S::kScaleStep : 0));
      __syncwarp();
      if (I8 && copies && piece == 0) {
        const uint32_t dst = scales + put_scale * S::kScaleStep + 4 * sub;
        bulk_load(dst, a.kv.k_scale + row, 4 * box_keys, bar);
        bulk_load(dst + 4 * S::kKeys, a.kv.v_scale + row, 4 * box_keys, bar);
      }
      if (++put_scale == S::kScaleSlots) put_scale = 0;
    } else {
      if (lane == 0) mbar_arrive_tx(bar, S::kHalf);
      __syncwarp();
    }
    if (copies)
      tma_load_2d(ring + put_slot * S::kHalf + piece * S::kBox + sub * 128, put & 1 ? &vmap : &kmap, piece * (I8 ? 128 : 64),
                  row, bar);
    ++put;
    if (++put_slot == S::kSlots) put_slot = 0;
  };
#pragma unroll 1
  for (int j = 0; j < S::kSlots; ++j) fetch();
  if (!I8) strays();

  // ---- queries as B fragments, in the order of K's pieces: [NT][DP / 32] x 16 bytes a lane
  for (int i = warp; i < NT; i += S::kWarps) {
    const int r = w.r0 + 8 * i + g;
    const bool ok = 8 * i + g < w.rows;
    const char* src = static_cast<const char*>(a.q);
    if (ok) src += ((w.first + r / a.G) * a.q_ts + (h * a.G + r % a.G) * a.q_hs) * 2;
    uint4 v[DP / 32];
#pragma unroll
    for (int k = 0; k < DP / 32; ++k) {
      // the values that this lane's K chunks 2t, 2t + 1 hold: 8 a chunk in 16 bits, 16 in 8
      const int d = I8 ? 128 * (k >> 2) + 32 * t + 8 * (k & 3) : 64 * (k >> 1) + 16 * t + 8 * (k & 1);
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
        const int e = fp16_lift(top);
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
    for (int k = 0; k < DP / 32; ++k) *reinterpret_cast<uint4*>(q_s + (i * (DP / 32) + k) * 512 + lane * 16) = v[k];
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

  float o[NT][DP / 16][4], m[NT][2], base[NT][2], l[NT][2], vref[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
#pragma unroll
    for (int j = 0; j < DP / 16; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[i][j][c] = 0.f;
    m[i][0] = m[i][1] = -INFINITY;
    base[i][0] = base[i][1] = 0.f;   // m, or 0 while no key has been seen
    l[i][0] = l[i][1] = vref[i][0] = vref[i][1] = 0.f;
  }

  // this lane's chunks in a piece: K rows g, g + 8 (1024 bytes on), V rows 2t, 2t + 1 (and 8 on)
  const uint32_t kx[2] = {(uint32_t)(g * 128 + ((2 * t ^ g) << 4)), (uint32_t)(g * 128 + (((2 * t + 1) ^ g) << 4))};
  const uint32_t vx[2] = {(uint32_t)(2 * t * 128 + ((g ^ 2 * t) << 4)), (uint32_t)((2 * t + 1) * 128 + ((g ^ (2 * t + 1)) << 4))};
  int slot = 0, phase = 0, scale_slot = 0;
  bool ok = true;
  auto step = [&]() {   // the half in `slot` is used up: refill it, go to the next
    __syncwarp();
    fetch();
    if (++slot == S::kSlots) {
      slot = 0;
      phase ^= 1;
    }
  };
  for (int n = 0; 2 * n < halves; ++n) {
    ok = __all_sync(0xffffffffu, copy_wait(bar0 + 8 * slot, phase));
    if (!ok) break;
    uint32_t src = ring + slot * S::kHalf;
    // ---- S^T = K Q^T; two sums per tile, so that no MMA waits for the one before it
    float s[S::kU][NT][2][4];
#pragma unroll
    for (int u = 0; u < S::kU; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[u][i][0][c] = s[u][i][1][c] = 0.f;
#pragma unroll
    for (int k = 0; k < 2 * S::kC; ++k) {
#pragma unroll
      for (int u = 0; u < S::kU; ++u) {
        const uint32_t at = src + (k >> 1) * S::kBox + u * 2048 + kx[k & 1];
        const uint4 k0 = lds16(at), k1 = lds16(at + 1024);
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
              mma16816<M>(s[u][i][j & 1], a0, a1, a2, a3, b0, b1);
            }
          }
        } else {
#pragma unroll
          for (int i = 0; i < NT; ++i) {
            const uint4 q = lds16(q_sm + (i * (DP / 32) + k) * 512 + lane * 16);
            mma16816<M>(s[u][i][0], k0.x, k1.x, k0.y, k1.y, q.x, q.y);
            mma16816<M>(s[u][i][1], k0.z, k1.z, k0.w, k1.w, q.z, q.w);
          }
        }
      }
    }
    // ---- scores, masks
    const int k0 = key_of(n);
    const uint32_t none = (gone >> (2 * n & 31)) & (S::kU == 2 ? 3 : 1);
    const bool whole = k0 >= all_lo && k0 + S::kKeys <= all_hi && k0 + S::kKeys <= s1 && !none;
    float ks[S::kU][2], vs[S::kU][2];
    bool high = false;
    float vlow = INFINITY;   // what every row's vref covers
    if (I8) {
#pragma unroll
      for (int i = 0; i < NT; ++i) vlow = fminf(vlow, fminf(vref[i][0], vref[i][1]));
    }
#pragma unroll
    for (int u = 0; u < S::kU; ++u) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        ks[u][e] = vs[u][e] = 1.f;
        if (I8) {
          const uint32_t at = scales + scale_slot * S::kScaleStep + 4 * (16 * u + g + 8 * e);
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(ks[u][e]) : "r"(at));
          asm volatile("ld.shared.f32 %0, [%1];" : "=f"(vs[u][e]) : "r"(at + 4 * S::kKeys));
          // what lies past the keys, or on a page that does not exist, is no scale
          if (!whole && (((none >> u) & 1) || k0 + 16 * u + g + 8 * e >= s1)) vs[u][e] = 0.f;
          high |= vs[u][e] > vlow;
        }
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = (s[u][i][0][c] + s[u][i][1][c]) * (I8 ? sc[i][c & 1] * ks[u][c >> 1] : sc[i][c & 1]);
          if (!whole) {
            const int key = k0 + 16 * u + g + 8 * (c >> 1);
            if (((none >> u) & 1) || key >= s1 || key < klo[i][c & 1] || key >= khi[i][c & 1]) v = -INFINITY;
          }
          s[u][i][0][c] = v;
          high |= v > m[i][c & 1] + (8.f + kLift);
        }
    }
    if (++scale_slot == S::kScaleSlots) scale_slot = 0;
    if (__any_sync(0xffffffffu, high)) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = -INFINITY;
#pragma unroll
          for (int u = 0; u < S::kU; ++u) x = fmaxf(x, fmaxf(s[u][i][0][c], s[u][i][0][c + 2]));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          float undo = 1.f;
          if (I8) {   // of the keys that the row sees: a hidden one's scale must not cost it bits
            float y = 0.f;
#pragma unroll
            for (int u = 0; u < S::kU; ++u)
#pragma unroll
              for (int e = 0; e < 2; ++e)
                if (s[u][i][0][c + 2 * e] != -INFINITY) y = fmaxf(y, vs[u][e]);
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 4));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 8));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, 16));
            if (y > vref[i][c]) {
              const float ref = above(y);
              undo = vref[i][c] / ref;
              vref[i][c] = ref;
            }
          }
          const float mn = fmaxf(m[i][c], x - kLift);
          const float by = mn == -INFINITY ? 1.f : ex2(m[i][c] - mn);
          m[i][c] = mn;
          base[i][c] = mn == -INFINITY ? 0.f : mn;
          l[i][c] *= by;
#pragma unroll
          for (int j = 0; j < DP / 16; ++j) {
            o[i][j][c] *= by * undo;
            o[i][j][c + 2] *= by * undo;
          }
        }
    }
    step();
    // ---- P^T: columns summed, then turned into B fragments
    uint32_t p0[S::kU][NT], p1[S::kU][NT];
#pragma unroll
    for (int u = 0; u < S::kU; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float p[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          p[c] = ex2(s[u][i][0][c] - base[i][c & 1]);
          l[i][c & 1] += p[c];
          if (I8) {
            const bool hidden = !whole && p[c] == 0.f;   // a masked key's scale may be anything
            // 1 / vref, a power of two (2^127 where no scale but 0 has been seen)
            const float vinv = __int_as_float(0x7f000000 - __float_as_int(vref[i][c & 1]));
            p[c] = hidden ? 0.f : p[c] * (vs[u][c >> 1] * vinv);
          }
        }
        p0[u][i] = transpose8x8(pack2<M>(p[0], p[1]));
        p1[u][i] = transpose8x8(pack2<M>(p[2], p[3]));
      }
    ok = __all_sync(0xffffffffu, copy_wait(bar0 + 8 * slot, phase));
    if (!ok) break;
    src = ring + slot * S::kHalf;
    // ---- O^T += V^T P^T
#pragma unroll
    for (int c = 0; c < S::kC; ++c)
#pragma unroll
      for (int u = 0; u < S::kU; ++u) {
        uint4 v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = lds16(src + c * S::kBox + u * 2048 + (r >> 1) * 1024 + vx[r & 1]);
        if (!I8 && !whole) {   // values past the keys may be anything, and 0 * NaN is not 0
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (((none >> u) & 1) || k0 + 16 * u + 2 * t + (r & 1) + 8 * (r >> 1) >= s1) v[r] = make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (I8) {
            const uint32_t x0 = (&v[0].x)[j] ^ 0x80808080u, x1 = (&v[1].x)[j] ^ 0x80808080u;
            const uint32_t x2 = (&v[2].x)[j] ^ 0x80808080u, x3 = (&v[3].x)[j] ^ 0x80808080u;
#pragma unroll
            for (int e = 0; e < 2; ++e) {  // values 4 j + 2 e, 4 j + 2 e + 1 of the chunk
              const uint32_t lo2 = __byte_perm(x0, x1, e ? 0x7362 : 0x5140);
              const uint32_t hi2 = __byte_perm(x2, x3, e ? 0x7362 : 0x5140);
              const uint32_t a0 = bytes_f16(lo2, 0x4140), a1 = bytes_f16(lo2, 0x4342);
              const uint32_t a2 = bytes_f16(hi2, 0x4140), a3 = bytes_f16(hi2, 0x4342);
#pragma unroll
              for (int i = 0; i < NT; ++i) mma16816<M>(o[i][c * 8 + 2 * j + e], a0, a1, a2, a3, p0[u][i], p1[u][i]);
            }
          } else {
            const uint32_t a0 = __byte_perm((&v[0].x)[j], (&v[1].x)[j], 0x5410);
            const uint32_t a1 = __byte_perm((&v[0].x)[j], (&v[1].x)[j], 0x7632);
            const uint32_t a2 = __byte_perm((&v[2].x)[j], (&v[3].x)[j], 0x5410);
            const uint32_t a3 = __byte_perm((&v[2].x)[j], (&v[3].x)[j], 0x7632);
#pragma unroll
            for (int i = 0; i < NT; ++i) mma16816<M>(o[i][c * 4 + j], a0, a1, a2, a3, p0[u][i], p1[u][i]);
          }
        }
      }
    step();
  }
  if (!ok) {   // copies under way have landed before the ring's memory is used for anything else
    for (int i = max(0, put - S::kSlots); i < put; ++i) copy_wait(bar0 + 8 * (i % S::kSlots), (i / S::kSlots) & 1);
#pragma unroll
    for (int i = 0; i < NT; ++i) l[i][0] = l[i][1] = __int_as_float(0x7fffffff);   // the rows come out as NaN
  }
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
      if (g == 0) ml_s[warp][8 * i + 2 * t + c] = make_float2(m[i][c] + kLift, x * kDrop);
    }
  float* acc = reinterpret_cast<float*>(sm);   // [warp][row][DP + 4]
  constexpr int LD = DP + 4;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < DP / 16; ++j) {
      // rows g, g + 8 of the MMA tile are the values d, d + 1
      const int d = I8 ? 128 * (j >> 3) + 16 * g + 2 * (j & 7) : 64 * (j >> 2) + 8 * g + 2 * (j & 3);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float2* dst = reinterpret_cast<float2*>(acc + (warp * NT * 8 + 8 * i + 2 * t + c) * LD + d);
        const float by = kDrop * (I8 ? vref[i][c] : 1.f);
        *dst = make_float2(o[i][j][c] * by, o[i][j][c + 2] * by);
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

// Joins the splits of one row (token, head): a block takes 4 * LANES of its values, LANES threads of
// them for each of 256 / LANES shares of the splits; the shares are then added in order.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) attn_join_kernel(const AttnArgs a) {
  __shared__ float4 acc[256];
  __shared__ float by_s[256], red[8];
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x, hq = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = sequence_of(a.kv, t);
  if (b < 0) return;
  int first, count, lo, hi;
  sequence_rows(a.kv, b, first, count);
  block_keys(a, attn_rows(a, b, ((t - first) * a.G + hq % a.G) / a.rows_per_block), lo, hi);
  if (hi - lo <= a.chunk) return;   // written already
  const int n = min(256, (hi - lo - 1) / a.chunk + 1);
  const int64_t at = (int64_t)t * a.hq + hq;
  // the weight of each split: one a thread
  const int i = threadIdx.x;
  const float2 x = i < n ? a.part_ml[at * a.splits + i] : make_float2(-INFINITY, 0.f);
  constexpr int kParts = 256 / LANES;
  const int part = threadIdx.x / LANES, d = 4 * (blockIdx.z * LANES + threadIdx.x % LANES);
  const float* src = a.part_o + at * a.splits * a.D + d;
  float top = x.x;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) top = fmaxf(top, red[k]);
  const float base = top == -INFINITY ? 0.f : top, mine = ex2(x.x - base);
  by_s[i] = mine;
  float sum = x.y * mine;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  __syncthreads();
  if (lane == 0) red[warp] = sum;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  if (d < a.D) {
#pragma unroll 4
    for (int k = part; k < n; k += kParts) {
      const float w = by_s[k];
      const float4 z = *reinterpret_cast<const float4*>(src + (int64_t)k * a.D);
      y.x += z.x * w;
      y.y += z.y * w;
      y.z += z.z * w;
      y.w += z.w * w;
    }
  }
  acc[threadIdx.x] = y;
  __syncthreads();
  if (part == 0) {
    sum = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += red[k];
#pragma unroll
    for (int k = 1; k < kParts; ++k) {
      const float4 z = acc[LANES * k + threadIdx.x];
      y.x += z.x;
      y.y += z.y;
      y.z += z.z;
      y.w += z.w;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (d < a.D)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.D + d) =
          make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
    if (a.lse && d == 0) a.lse[at] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * kLn2;
  }
}

// The same for many rows and at most 32 splits: a warp a row, 8 heads of a token a block.
template <typename T>
__global__ void __launch_bounds__(256) attn_join_rows_kernel(const AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int t = blockIdx.x, hq = blockIdx.y * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  const int b = sequence_of(a.kv, t);
  if (b < 0 || hq >= a.hq) return;
  int first, count, lo, hi;
  sequence_rows(a.kv, b, first, count);
  block_keys(a, attn_rows(a, b, ((t - first) * a.G + hq % a.G) / a.rows_per_block), lo, hi);
  if (hi - lo <= a.chunk) return;   // written already
  const int n = min(32, (hi - lo - 1) / a.chunk + 1);
  const int64_t at = (int64_t)t * a.hq + hq;
  const float2 x = lane < n ? a.part_ml[at * a.splits + lane] : make_float2(-INFINITY, 0.f);
  float top = x.x;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.f : top, by = ex2(x.x - base);
  float sum = x.y * by;
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  for (int d0 = 0; d0 < a.D; d0 += 128) {
    const int d = d0 + 4 * lane;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < n; ++k) {
      const float w = __shfl_sync(0xffffffffu, by, k);
      if (d < a.D) {
        const float4 z = *reinterpret_cast<const float4*>(a.part_o + (at * a.splits + k) * a.D + d);
        y.x += z.x * w;
        y.y += z.y * w;
        y.z += z.z * w;
        y.w += z.w * w;
      }
    }
    if (d < a.D)
      *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.D + d) =
          make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
  }
  if (a.lse && lane == 0) a.lse[at] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * kLn2;
}

// A pool [rows, D] as boxes of `keys` rows x 128 bytes, 128-byte swizzle; values past D read as zeros.
bool make_pool_map(CUtensorMap* map, const void* base, const AttnArgs& a, bool i8, int keys) {
  const cuuint64_t e = i8 ? 1 : 2;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.D), (static_cast<cuuint64_t>(a.kv.pages) * a.kv.heads) << a.kv.page_log2};
  const cuuint64_t strides[1] = {a.D * e};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(128 / e), static_cast<cuuint32_t>(keys)};
  const cuuint32_t es[2] = {1, 1};
  return encode_fn()(map, i8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(base),
                     dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
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
  CUtensorMap kmap, vmap;
  const int keys = S::kKeys < 1 << a.kv.page_log2 ? S::kKeys : 1 << a.kv.page_log2;
  if (!make_pool_map(&kmap, a.kv.k, a, I8, keys) || !make_pool_map(&vmap, a.kv.v, a, I8, keys)) return VQ2_ERR_LAUNCH;
  return launch_kernel(kern, grid, dim3(S::kWarps * 32), S::kSmem, st, a, kmap, vmap);
}

template <bool I8, typename T>
int launch_shape(const AttnArgs& a, cudaStream_t st) {
  const int nt = a.rows_per_block / 8;
  if (a.D > 128) return nt == 1 ? launch<256, 1, I8, T>(a, st) : launch<256, 2, I8, T>(a, st);
  if (I8 || a.D > 64) return nt == 1 ? launch<128, 1, I8, T>(a, st) : launch<128, 2, I8, T>(a, st);
  return nt == 1 ? launch<64, 1, false, T>(a, st) : launch<64, 2, false, T>(a, st);
}

}  // namespace

void plan_attn_decode(AttnArgs& a, int64_t max_new, int64_t max_len) {
  // Rows of a block: 8, or 16 where more share a key (32 spilled and was slower than the tensor-core
  // kernel: 16 sequences of 4000 tokens, 32 rows, D 128: 100 us).
  const int64_t rows = max_new * a.G;
  const int nt = rows <= 8 ? 1 : 2;
  a.rows_per_block = 8 * nt;
  a.row_blocks = (int)((rows + 8 * nt - 1) / (8 * nt));
  if (a.row_blocks < 1) a.row_blocks = 1;
  a.lo_mask = ~31;
  // Split the keys so that there are about 1.5 blocks an SM, no further than `step` keys (what a
  // block's warps take at once). A split costs about two steps (its start, and the joining launch of
  // 2.5 us): four steps' keys stay whole. Long work is cut finer, at 768 keys, so that ragged lengths
  // even out over several rounds of blocks (64 sequences of 800 to 8000 tokens, D 256: 512 keys
  // 104 us, 768 101.7, 1024 101.4, 2048 104.9), but into 64 splits at most unless there are too few
  // blocks (one sequence of 60000 in int8: 63 splits 32 us, 118 24.4, 209 28.2).
  const int64_t step = a.D > 128 ? 64 : 128;
  int64_t keys = max_len;
  if (a.window && a.window + max_new + 32 < keys) keys = a.window + max_new + 32;
  keys += 31;   // the first key is rounded down by up to 31
  const int64_t blocks = (int64_t)a.kv.seqs * a.kv.heads * a.row_blocks;
  const int64_t fill = (keys * blocks * 2 + 3 * sm_count() - 1) / (3 * sm_count());
  int64_t chunk = fill < 768 ? fill : 768;
  const int64_t least = (keys + 63) / 64 < fill ? (keys + 63) / 64 : fill;
  if (chunk < least) chunk = least;
  if (chunk < step) chunk = step;
  if (chunk < (keys + 255) / 256) chunk = (keys + 255) / 256;   // what the joining kernel takes
  if (keys <= 4 * step + 31) chunk = keys;
  chunk = (chunk + 31) & ~int64_t(31);
  a.chunk = (int)chunk;
  a.splits = (int)((keys + chunk - 1) / chunk);
  if (a.splits < 1) a.splits = 1;
}

int launch_attn_decode(const AttnArgs& a, bool i8, cudaStream_t st) {
  if (!encode_fn()) return VQ2_ERR_LAUNCH;
  if (i8) return a.q_bf16 ? launch_shape<true, __nv_bfloat16>(a, st) : launch_shape<true, __half>(a, st);
  return a.q_bf16 ? launch_shape<false, __nv_bfloat16>(a, st) : launch_shape<false, __half>(a, st);
}

int launch_attn_join(const AttnArgs& a, cudaStream_t st) {
  // Rows enough to fill the card with a warp a row (7000 rows over 2 splits: 25 us with a block a row).
  if (a.splits <= 32 && (int64_t)a.T * a.hq >= 12 * sm_count()) {
    const dim3 grid((unsigned)a.T, (unsigned)((a.hq + 7) / 8));
    return a.q_bf16 ? launch_kernel(attn_join_rows_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, a)
                    : launch_kernel(attn_join_rows_kernel<__half>, grid, dim3(256), 0, st, a);
  }
  // Few splits: a whole row a block. Many: 64 values a block, 16 splits read at once (one sequence of
  // 701 tokens over 12 splits, whole step: 9.1 us with whole rows, 8.2 with 64 values; 64 sequences of
  // up to 8000 over 11: 103.5 and 108.6 us).
  const int lanes = a.splits > 32 || (int64_t)a.T * a.hq < 2 * sm_count() || a.D <= 64 ? 16 : a.D <= 128 ? 32 : 64;
  const dim3 grid((unsigned)a.T, (unsigned)a.hq, (unsigned)((a.D + 4 * lanes - 1) / (4 * lanes))), block(256);
  if (lanes == 16)
    return a.q_bf16 ? launch_kernel(attn_join_kernel<__nv_bfloat16, 16>, grid, block, 0, st, a)
                    : launch_kernel(attn_join_kernel<__half, 16>, grid, block, 0, st, a);
  if (lanes == 32)
    return a.q_bf16 ? launch_kernel(attn_join_kernel<__nv_bfloat16, 32>, grid, block, 0, st, a)
                    : launch_kernel(attn_join_kernel<__half, 32>, grid, block, 0, st, a);
  return a.q_bf16 ? launch_kernel(attn_join_kernel<__nv_bfloat16, 64>, grid, block, 0, st, a)
                  : launch_kernel(attn_join_kernel<__half, 64>, grid, block, 0, st, a);
}

}  // namespace vq2

extern "C" int vq2_attention_status(int reset) {
  int32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_decode_status, sizeof(v));
  if (e == cudaSuccess && reset) {
    const int32_t z = 0;
    e = cudaMemcpyToSymbol(g_decode_status, &z, sizeof(z));
  }
  if (e != cudaSuccess) {
    vq2::set_last_cuda_error(e);
    return VQ2_ERR_LAUNCH;
  }
  const int other = vq2::attn_chunk_status(reset);
  return v > other ? v : other;
}
