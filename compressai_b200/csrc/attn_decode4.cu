// Attention of few query rows per key/value head over a 4-bit paged cache: the decode step.
//
// A cached value is code * factor * scale: a code of -7..7 (stored plus 8, two a byte), a factor of 8 bits for each 64
// values of a row, the row's scale in 32 bits. As over 16 and 8 bits a warp takes its own keys, 16 a tile, computes
//
//   S^T [16 keys x 8 rows] = K Q^T,   P = 2^(S - m),   O^T [D x 8 rows] += V^T P^T
//
// with mma.m16n8k16 and its own running maximum m and sum; warps, and blocks that split a long sequence, are joined at
// the end. HBM bounds it (half of int8's bytes) as long as the codes become operands in few instructions:
//
//   * A code's bits c in the low end of a 16-bit float are the number c 2^-24 (and one place of four further up,
//     16 c 2^-24), exactly: a mask takes two codes out of a word and they are an operand register. Four masks and one
//     shift serve the 8 codes of a word; no conversion, no subtraction.
//   * What the 16 stands for is put right where it is free: in K in the queries' operand (half of it is divided by 16),
//     in V in the rows of O that such codes end in.
//   * The 8 in every code: K's sums start at -8 sum q, and V's gets -8 sum P of each group at the end, summed by one more
//     MMA a group into the row of the group's number, from the same rounded weights.
//   * K's factors multiply a group's sum (4 numbers a lane), V's multiply the weights (2 registers a group): both of
//     them once for 16 keys x 64 values.
//
// Where the codes are: a K operand wants 16 values of a group in the four lanes of a key's row, a V operand 8 in each
// of the eight lanes g: lane (g, t) reads the 8 bytes t of a group from keys of number g and the 4 bytes g from keys of
// number 2t, 2t + 1. With TMA's swizzle (none where a row is 32 bytes) all of these reads are free of bank conflicts if the
// keys are numbered as `key_of_row` does. (4 sequences to 100,003, 32/8 heads of 128, B200.)
//
// Queries become fp16 by a power of two per row, exact down to 2^-24 of the row's largest value; the weights are fp16,
// relative to a power of two above the row scales of V that the row sees, and rounded once more with the factor. Maxima,
// sums and O are 32 bits. Rescaling is lazy, see attn_decode.cu.
#include <atomic>
#include <type_traits>

#include "attn_dev.cuh"
#include "tcgen05.cuh"

// Sticky status: VQ2_ERR_TIMEOUT once a bounded wait for a copy gave up.
__device__ int32_t g_decode4_status;

namespace vq2 {
namespace {

__device__ __forceinline__ uint32_t lds4(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
  uint2 v;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ float lds_f32(uint32_t addr) { return __uint_as_float(lds4(addr)); }
__device__ __forceinline__ uint32_t lds1(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}

__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                    float c0, float c1, float c2, float c3) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  mma(d, a0, a1, a2, a3, b0, b1, d[0], d[1], d[2], d[3]);
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

// Two e4m3 bytes (the low two of w) as fp16.
__device__ __forceinline__ uint32_t factors_f16(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// Shapes of one variant. DP: head size rounded up (values past D are zeros); NT: 8-row tiles.
template <int DP, int NT>
struct Shape4 {
  static constexpr int kRow = DP / 2;                   // bytes of a key's codes
  static constexpr int kG = DP / 64;                    // groups
  static constexpr int kU = DP == 64 ? 4 : 2;          // 16-key tiles a step
  static constexpr int kKeys = 16 * kU;
  static constexpr int kHalf = kKeys * kRow;            // K or V of a step
  static constexpr int kWarps = 4;
  static constexpr int kPerSm = NT == 2 ? 2 : DP == 256 ? 3 : 4;   // blocks an SM, as registers allow
  static constexpr int kRecords = kU * (64 + 16 * kG);  // scales of a half, at most
  static constexpr int kFit = (224 * 1024 / kPerSm - 10240) / (kWarps * (kHalf + kRecords));
  static constexpr int kSlots = kFit > 8 ? 8 : kFit;
  static constexpr int kRing = kWarps * kSlots * kHalf;
  static constexpr int kJoin = kWarps * NT * 8 * (DP + 4) * 4;   // the warps' O, over the ring
  static constexpr int kQ = NT * kG * 1024;             // query fragments
  static constexpr int kScaleSlots = kSlots / 2 + 1;    // steps under way
  static constexpr int kScales = kWarps * kScaleSlots * 2 * kRecords;
  static constexpr int kSmem = 1024 + (kRing > kJoin ? kRing : kJoin) + kQ + kScales;
  static_assert(kSlots >= 3, "a half in use, two in flight");
  static_assert(kScaleSlots * kU <= 32, "bits of the pages that are gone");
};

// The key of a tile that stands in row r (0..7) of the MMA's first 8; 8 on, that of row r + 8. Rows 0..3, rows 4..7,
// the even ones and the odd ones are each on four different 32-byte places of shared memory.
template <int DP>
__device__ __forceinline__ int key_of_row(int r) {
  const int place = (r & 3) ^ (r >> 2), other = r >> 2;
  if (DP == 256) return 2 * place + other;
  if (DP == 128) return (place & 1) | other << 1 | (place & 2) << 1;
  return place + 4 * other;
}

constexpr long long kWaitCycles = 4000000000LL;  // ~2 s at 1.965 GHz

__device__ __forceinline__ bool copy_wait(uint32_t bar, uint32_t parity) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity))
    if (clock64() - t0 > kWaitCycles) {
      atomicMax(&g_decode4_status, VQ2_ERR_TIMEOUT);
      return false;
    }
  return true;
}

template <int DP, int NT, typename T>
__global__ void __launch_bounds__(Shape4<DP, NT>::kWarps * 32, Shape4<DP, NT>::kPerSm)
    attn_decode4_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using S = Shape4<DP, NT>;
  constexpr int G = S::kG, U = S::kU, ROW = S::kRow;
  // weights 2^7 larger than the maximum asks for, so that those down to 2^-32 of the largest are more than 0
  constexpr float kLift = 7.f, kDrop = 1.f / 128.f;
  constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;
  extern __shared__ unsigned char decode4_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(decode4_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* q_s = sm + (S::kRing > S::kJoin ? S::kRing : S::kJoin);
  __shared__ uint64_t bars[S::kWarps][S::kSlots];
  __shared__ float2 ml_s[S::kWarps][NT * 8];
  __shared__ float qexp_s[NT * 8], qsum_s[NT * 8][G];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int split = blockIdx.y, h = blockIdx.z;
  const int b = blockIdx.x / a.row_blocks, rb = blockIdx.x - b * a.row_blocks;
  const AttnRows w = attn_rows(a, b, rb);
  blank_strays(a, w, b, ((int64_t)rb * a.kv.heads + h) * a.splits + split, (int64_t)a.row_blocks * a.kv.heads * a.splits);
  if (w.rows <= 0) return;
  int lo, hi;
  block_keys(a, w, lo, hi);
  if (split > 0 && (int64_t)split * a.chunk >= hi - lo) return;   // split 0 stays: it writes the rows that see nothing
  const int s0 = lo + split * a.chunk, s1 = s0 + min(a.chunk, hi - s0);   // no sum past 2^31
  const bool alone = hi - lo <= a.chunk;
  const int tiles = s1 > s0 ? (s1 - s0 + S::kKeys - 1) / S::kKeys : 0;

  // ---- the warp's ring: halves K0 V0 K1 V1 .. of its steps warp, warp + kWarps, ..
  const int groups = (a.D + 63) >> 6, record = 64 + 16 * groups;   // bytes of 16 keys' scales
  const uint32_t q_sm = su32(q_s), ring = su32(sm) + warp * S::kSlots * S::kHalf, bar0 = su32(&bars[warp][0]);
  const uint32_t scales = q_sm + S::kQ + warp * S::kScaleSlots * 2 * S::kRecords;
  const int32_t* table = a.kv.table + b * a.kv.table_stride;
  const int page_mask = (1 << a.kv.page_log2) - 1, seen = row_lo(a, w, w.r0 / a.G);
  const int halves = tiles > warp ? 2 * ((tiles - warp + S::kWarps - 1) / S::kWarps) : 0;
  auto key_of = [&](int i) { return s0 + S::kKeys * (warp + S::kWarps * i); };   // first key of the warp's step i
  // A copy is min(page, step) keys: this lane's, and the key it starts at.
  const int box_keys = min(1 << a.kv.page_log2, S::kKeys), sub = lane * box_keys;
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
  // gone: bit U i + u of 32 says that the page of tile u of step i is not in the pool: no such keys
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
      for (int u = 0; u < U; ++u) {   // of the lane whose copy holds tile u
        const uint32_t bit = (out >> (16 * u / box_keys)) & 1;
        const int at = (U * i + u) & 31;
        gone = (gone & ~(1u << at)) | (bit << at);
      }
      // a page that exists stands in for one that does not
      row = (((there ? ahead : 0) * a.kv.heads + h) << a.kv.page_log2) + ((k + sub) & page_mask);
      ahead = page_of(i + 1);
      if (lane == 0) mbar_arrive_tx(bar, S::kHalf + 2 * U * record);
      __syncwarp();
      if (copies) {
        const uint32_t dst = scales + put_scale * 2 * S::kRecords + (sub >> 4) * record;
        const int64_t from = (int64_t)(row >> 4) * record;
        const int bytes = (box_keys >> 4) * record;
        bulk_load(dst, reinterpret_cast<const unsigned char*>(a.kv.k_scale) + from, bytes, bar);
        bulk_load(dst + S::kRecords, reinterpret_cast<const unsigned char*>(a.kv.v_scale) + from, bytes, bar);
      }
      if (++put_scale == S::kScaleSlots) put_scale = 0;
    } else {
      if (lane == 0) mbar_arrive_tx(bar, S::kHalf);
      __syncwarp();
    }
    if (copies) tma_load_2d(ring + put_slot * S::kHalf + sub * ROW, put & 1 ? &vmap : &kmap, 0, row, bar);
    ++put;
    if (++put_slot == S::kSlots) put_slot = 0;
  };
#pragma unroll 1
  for (int j = 0; j < S::kSlots; ++j) fetch();

  // ---- queries as B fragments, in the order of K's codes: of a group's 16 values of lane t, word w holds 8 w .. 8 w + 7,
  // and its MMA j takes values 2 j, 2 j + 4 and 2 j + 1, 2 j + 5 (these by 16)
  for (int i = warp; i < NT; i += S::kWarps) {
    const int r = w.r0 + 8 * i + g;
    const bool ok = 8 * i + g < w.rows;
    const T* src = static_cast<const T*>(a.q);
    if (ok) src += (w.first + r / a.G) * a.q_ts + (h * a.G + r % a.G) * a.q_hs;
    uint4 v[G][2];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < G; ++k)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int d = 64 * k + 16 * t + 8 * c;
        v[k][c] = make_uint4(0, 0, 0, 0);
        if (ok && d < a.D) v[k][c] = *reinterpret_cast<const uint4*>(src + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 f = unpack2<T>((&v[k][c].x)[j]);
          top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
        }
      }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = fp16_lift(top);
    const float by = __int_as_float((127 + e) << 23);
    if (t == 0) qexp_s[8 * i + g] = __int_as_float((127 - e) << 23);
#pragma unroll
    for (int k = 0; k < G; ++k) {
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = unpack2<T>((&v[k][c].x)[j]);
          f[2 * j] = x.x * by;
          f[2 * j + 1] = x.y * by;
        }
        uint4 o;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t b0 = pack2<__half>(f[2 * j], f[2 * j + 4]);
          const uint32_t b1 = pack2<__half>(f[2 * j + 1] * 0.0625f, f[2 * j + 5] * 0.0625f);
          (&o.x)[2 * j] = b0;
          (&o.x)[2 * j + 1] = b1;
          const float2 x = unpack2<__half>(b0), y = unpack2<__half>(b1);
          sum += (x.x + x.y) + 16.f * (y.x + y.y);
        }
        *reinterpret_cast<uint4*>(q_s + ((i * G + k) * 2 + c) * 512 + lane * 16) = o;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) qsum_s[8 * i + g][k] = sum * (-8.f / 16777216.f);
    }
  }
  __syncthreads();

  // ---- this lane's two rows of each tile (columns 2t, 2t + 1 of S^T): what they see
  int klo[NT][2], khi[NT][2];
  float sc[NT][2], start[NT][G][2];   // start: what a group's sum starts at
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = 8 * i + 2 * t + c;
      const bool ok = r < w.rows;
      const int tok = (w.r0 + (ok ? r : 0)) / a.G;
      klo[i][c] = row_lo(a, w, tok);
      khi[i][c] = ok ? row_hi(a, w, tok) : 0;
      sc[i][c] = a.scale_log2 * qexp_s[r];
#pragma unroll
      for (int k = 0; k < G; ++k) start[i][k][c] = qsum_s[r][k];
    }
  // keys that every row sees need no mask
  const int all_lo = row_lo(a, w, (w.r0 + w.rows - 1) / a.G), all_hi = row_hi(a, w, w.r0 / a.G);

  // o: sums over the codes plus 8, of values d (0, 1) and, 16 times as large, d + 1 (2, 3); oc: row k of it, 8 2^-24 times the
  // weights of group k
  float o[NT][DP / 16][4], oc[NT][4], m[NT][2], base[NT][2], l[NT][2], vref[NT][2];
#pragma unroll
  for (int i = 0; i < NT; ++i) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
#pragma unroll
      for (int j = 0; j < DP / 16; ++j) o[i][j][c] = 0.f;
      oc[i][c] = 0.f;
    }
    m[i][0] = m[i][1] = -INFINITY;
    base[i][0] = base[i][1] = 0.f;   // m, or 0 while no key has been seen
    l[i][0] = l[i][1] = vref[i][0] = vref[i][1] = 0.f;
  }

  // this lane's places: K's key (another 8 on), V's keys of the MMA's rows 2t, 2t + 1 (others 8 on); 32 bytes a group
  auto swizzled = [](int key, int byte) {
    const int x = DP == 256 ? key & 7 : DP == 128 ? (key >> 1) & 3 : 0;
    return (uint32_t)(key * ROW + (byte ^ (x << 4)));
  };
  const int kkey = key_of_row<DP>(g), vkey0 = key_of_row<DP>(2 * t), vkey1 = key_of_row<DP>(2 * t + 1);
  const uint32_t kx = swizzled(kkey, 8 * t), vx[2] = {swizzled(vkey0, 4 * g), swizzled(vkey1, 4 * g)};
  // the factors of V's two keys out of the four bytes that both are in
  const uint32_t vword = vkey0 & 4, vsel = (uint32_t)(vkey0 & 3) | (uint32_t)(vkey1 & 3) << 4;
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
    const uint32_t k_rec = scales + scale_slot * 2 * S::kRecords, v_rec = k_rec + S::kRecords;
    if (++scale_slot == S::kScaleSlots) scale_slot = 0;
    // ---- S^T = K Q^T, a group's sum times its factor
    float s[U][NT][4];
#pragma unroll
    for (int k = 0; k < G; ++k) {
      uint4 q[NT][2];
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) q[i][c] = lds16(q_sm + ((i * G + k) * 2 + c) * 512 + lane * 16);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t at = src + u * 16 * ROW + (kx ^ (32 * k));
        const uint2 x = lds8(at), y = lds8(at + 8 * ROW);
        float f0 = 0.f, f1 = 0.f;   // factors, by 2^-8: their bits as fp16's
        if (k < groups) {
          const uint32_t fa = k_rec + u * record + 64 + 16 * k + kkey;
          const uint32_t two = (lds1(fa) | lds1(fa + 8) << 16) << 7;
          const float2 f = unpack2<__half>(two);
          f0 = f.x;
          f1 = f.y;
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          float acc[4];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t xw = c ? x.y : x.x, yw = c ? y.y : y.x, xs = xw >> 8, ys = yw >> 8;
            const float s0_ = start[i][k][0], s1_ = start[i][k][1];
            if (c == 0) mma(acc, xw & kLow, yw & kLow, xw & kHigh, yw & kHigh, q[i][c].x, q[i][c].y, s0_, s1_, s0_, s1_);
            else mma(acc, xw & kLow, yw & kLow, xw & kHigh, yw & kHigh, q[i][c].x, q[i][c].y);
            mma(acc, xs & kLow, ys & kLow, xs & kHigh, ys & kHigh, q[i][c].z, q[i][c].w);
          }
#pragma unroll
          for (int c = 0; c < 4; ++c) s[u][i][c] = k ? fmaf(acc[c], c < 2 ? f0 : f1, s[u][i][c]) : acc[c] * (c < 2 ? f0 : f1);
        }
      }
    }
    // ---- scores, masks
    const int k0 = key_of(n);
    const uint32_t none = (gone >> (U * n & 31)) & ((1u << U) - 1);
    const bool whole = k0 >= all_lo && k0 + S::kKeys <= all_hi && k0 + S::kKeys <= s1 && !none;
    float vs[U][2];
    bool high = false;
    float vlow = INFINITY;   // what every row's vref covers
#pragma unroll
    for (int i = 0; i < NT; ++i) vlow = fminf(vlow, fminf(vref[i][0], vref[i][1]));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float ks[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const uint32_t at = u * record + 4 * (kkey + 8 * e);
        ks[e] = lds_f32(k_rec + at);
        vs[u][e] = lds_f32(v_rec + at);
        // what lies past the keys, or on a page that does not exist, is no scale
        if (!whole && (((none >> u) & 1) || k0 + 16 * u + kkey + 8 * e >= s1)) vs[u][e] = 0.f;
        high |= vs[u][e] > vlow;
      }
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = s[u][i][c] * 4294967296.f * (sc[i][c & 1] * ks[c >> 1]);   // 2^24 of the codes, 2^8 of the factors
          if (!whole) {
            const int key = k0 + 16 * u + kkey + 8 * (c >> 1);
            if (((none >> u) & 1) || key >= s1 || key < klo[i][c & 1] || key >= khi[i][c & 1]) v = -INFINITY;
          }
          s[u][i][c] = v;
          high |= v > m[i][c & 1] + (8.f + kLift);
        }
    }
    if (__any_sync(0xffffffffu, high)) {
#pragma unroll
      for (int i = 0; i < NT; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float x = -INFINITY, y = 0.f;   // y: of the keys that the row sees: a hidden one's scale must not cost it bits
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              x = fmaxf(x, s[u][i][c + 2 * e]);
              if (s[u][i][c + 2 * e] != -INFINITY) y = fmaxf(y, vs[u][e]);
            }
#pragma unroll
          for (int f = 4; f <= 16; f <<= 1) {
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, f));
            y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, f));
          }
          float undo = 1.f;
          if (y > vref[i][c]) {
            const float ref = above(y);
            undo = vref[i][c] / ref;
            vref[i][c] = ref;
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
          oc[i][c] *= by * undo;
        }
    }
    step();
    // ---- P^T: columns summed, then turned into B fragments
    uint32_t p0[U][NT], p1[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        float p[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          p[c] = ex2(s[u][i][c] - base[i][c & 1]);
          l[i][c & 1] += p[c];
          const bool hidden = !whole && p[c] == 0.f;   // a masked key's scale may be anything
          // 1 / vref, a power of two (2^127 where no scale but 0 has been seen)
          const float vinv = __int_as_float(0x7f000000 - __float_as_int(vref[i][c & 1]));
          p[c] = hidden ? 0.f : p[c] * (vs[u][c >> 1] * vinv);
        }
        p0[u][i] = transpose8x8(pack2<__half>(p[0], p[1]));
        p1[u][i] = transpose8x8(pack2<__half>(p[2], p[3]));
      }
    ok = __all_sync(0xffffffffu, copy_wait(bar0 + 8 * slot, phase));
    if (!ok) break;
    src = ring + slot * S::kHalf;
    // ---- O^T += V^T P^T, P times the group's factors
#pragma unroll
    for (int k = 0; k < G; ++k) {
      if (k >= groups) continue;   // values past D
      const uint32_t ones = g == k ? 0x00080008u : 0u;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const uint32_t fa = v_rec + u * record + 64 + 16 * k + vword;
        uint32_t f01 = factors_f16(__byte_perm(lds4(fa), 0, vsel)), f89 = factors_f16(__byte_perm(lds4(fa + 8), 0, vsel));
        if (!whole) {   // factors past the keys may be anything, and 0 * NaN is not 0
          const int left = (none >> u) & 1 ? 0 : s1 - (k0 + 16 * u);
          f01 &= (vkey0 < left ? 0xffffu : 0u) | (vkey1 < left ? 0xffff0000u : 0u);
          f89 &= (vkey0 + 8 < left ? 0xffffu : 0u) | (vkey1 + 8 < left ? 0xffff0000u : 0u);
        }
        const uint32_t at = src + u * 16 * ROW, b0 = at + (vx[0] ^ (32 * k)), b1 = at + (vx[1] ^ (32 * k));
        const uint32_t w0 = lds4(b0), w1 = lds4(b1), w2 = lds4(b0 + 8 * ROW), w3 = lds4(b1 + 8 * ROW);
        uint32_t f0[NT], f1[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          f0[i] = hmul2(p0[u][i], f01);
          f1[i] = hmul2(p1[u][i], f89);
          mma(oc[i], ones, 0u, ones, 0u, f0[i], f1[i]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {   // values 2 j and 2 j + 1 of each lane's 8
          uint32_t x = __byte_perm(w0, w1, j < 2 ? 0x5410 : 0x7632), y = __byte_perm(w2, w3, j < 2 ? 0x5410 : 0x7632);
          if (j & 1) {
            x >>= 8;
            y >>= 8;
          }
#pragma unroll
          for (int i = 0; i < NT; ++i) mma(o[i][4 * k + j], x & kLow, x & kHigh, y & kLow, y & kHigh, f0[i], f1[i]);
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
    for (int k = 0; k < G; ++k)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float less = __shfl_sync(0xffffffffu, oc[i][c], 4 * k + t);   // row k, this column
        const float by = kDrop * vref[i][c];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int d = 64 * k + 8 * g + 2 * j;
          float2* dst = reinterpret_cast<float2*>(acc + (warp * NT * 8 + 8 * i + 2 * t + c) * LD + d);
          *dst = make_float2((o[i][4 * k + j][c] - less) * 16777216.f * by, (o[i][4 * k + j][c + 2] * 0.0625f - less) * 16777216.f * by);
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

// A pool's codes [rows, D / 2] as boxes of `keys` rows x DP / 2 bytes, swizzled over the row; bytes past D / 2 read as zeros.
bool make_code_map(CUtensorMap* map, const void* base, const AttnArgs& a, int DP, int keys) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.D / 2), (static_cast<cuuint64_t>(a.kv.pages) * a.kv.heads) << a.kv.page_log2};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.D / 2)};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(DP / 2), static_cast<cuuint32_t>(keys)};
  const cuuint32_t es[2] = {1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, es,
                     CU_TENSOR_MAP_INTERLEAVE_NONE,
                     DP == 256 ? CU_TENSOR_MAP_SWIZZLE_128B : DP == 128 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DP, int NT, typename T>
int launch(const AttnArgs& a, cudaStream_t st) {
  using S = Shape4<DP, NT>;
  auto kern = attn_decode4_kernel<DP, NT, T>;
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
  if (!make_code_map(&kmap, a.kv.k, a, DP, keys) || !make_code_map(&vmap, a.kv.v, a, DP, keys)) return VQ2_ERR_LAUNCH;
  return launch_kernel(kern, grid, dim3(S::kWarps * 32), S::kSmem, st, a, kmap, vmap);
}

template <typename T>
int launch_shape(const AttnArgs& a, cudaStream_t st) {
  const int nt = a.rows_per_block / 8;
  if (a.D > 128) return nt == 1 ? launch<256, 1, T>(a, st) : launch<256, 2, T>(a, st);
  if (a.D > 64) return nt == 1 ? launch<128, 1, T>(a, st) : launch<128, 2, T>(a, st);
  return nt == 1 ? launch<64, 1, T>(a, st) : launch<64, 2, T>(a, st);
}

}  // namespace

void plan_attn_decode4(AttnArgs& a, int64_t max_new, int64_t max_len) {
  // As plan_attn_decode, in pieces of 64 keys: a step's, which a page holds whole or in whole parts.
  const int64_t rows = max_new * a.G;
  const int nt = rows <= 8 ? 1 : 2;
  a.rows_per_block = 8 * nt;
  a.row_blocks = (int)((rows + 8 * nt - 1) / (8 * nt));
  if (a.row_blocks < 1) a.row_blocks = 1;
  a.lo_mask = ~63;
  const int64_t step = a.D > 128 ? 128 : 256;
  int64_t keys = max_len;
  if (a.window && a.window + max_new + 64 < keys) keys = a.window + max_new + 64;
  keys += 63;   // the first key is rounded down by up to 63
  const int64_t blocks = (int64_t)a.kv.seqs * a.kv.heads * a.row_blocks;
  const int64_t fill = (keys * blocks * 2 + 3 * sm_count() - 1) / (3 * sm_count());
  int64_t chunk = fill < 768 ? fill : 768;
  const int64_t least = (keys + 63) / 64 < fill ? (keys + 63) / 64 : fill;
  if (chunk < least) chunk = least;
  if (chunk < step) chunk = step;
  if (chunk < (keys + 255) / 256) chunk = (keys + 255) / 256;   // what the joining kernel takes
  if (keys <= 2 * step + 63) chunk = keys;
  chunk = (chunk + 63) & ~int64_t(63);
  a.chunk = (int)chunk;
  a.splits = (int)((keys + chunk - 1) / chunk);
  if (a.splits < 1) a.splits = 1;
}

int launch_attn_decode4(const AttnArgs& a, cudaStream_t st) {
  if (!encode_fn()) return VQ2_ERR_LAUNCH;
  return a.q_bf16 ? launch_shape<__nv_bfloat16>(a, st) : launch_shape<__half>(a, st);
}

int attn_decode4_status(int reset) {
  int32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_decode4_status, sizeof(v));
  if (e == cudaSuccess && reset) {
    const int32_t z = 0;
    e = cudaMemcpyToSymbol(g_decode4_status, &z, sizeof(z));
  }
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return VQ2_ERR_LAUNCH;
  }
  return v;
}

}  // namespace vq2
