// Attention of few query rows per key/value head over a 4-bit paged cache: the decode step.
//
// A cached value is code * factor * scale: a code of -7..7 (stored plus 8, two a byte), a factor of 8 bits for each 64
// values of a row, the row's scale in 32 bits. As over 16 and 8 bits a warp takes its own keys, 16 a tile, computes
//
//   S^T [16 keys x 8 rows] = K Q^T,   P = 2^(S - m),   O^T [D x 8 rows] += V^T P^T
//
// with mma.m16n8k16 and its own running maximum m and sum; warps, and blocks that split a long sequence, are joined at
// the end. HBM bounds it (half of int8's bytes) as long as the codes become operands in few instructions, and they still
// set the pace: 300 a warp for 16 keys of 128 values, K and V.
//
//   * A code's bits c in the low end of a 16-bit float are the number c 2^-24 (and one place of four further up,
//     16 c 2^-24), exactly: a mask takes two codes out of a word and they are an operand register. The 8 codes of a word take
//     five integer instructions (which run at half rate) and a subtraction; no conversion.
//   * What the 16 stands for is put right where it is free: in K in the queries' operand (half of it is divided by 16),
//     in V in what such codes are multiplied by.
//   * The 8 in every code: K's sums, of 64 products each, start at -8 sum q. V's sums run over all keys of a warp, and an MMA's
//     addition is off by up to 2^-22 of its largest operand, to zero's side: with the 8 left in, sums of positive numbers only, 56
//     sequences of 131,072 keys came out 12 % off (524,288: 35 %). So V's operand has it taken away.
//   * K's factors multiply a group's sum (4 numbers a lane). V's multiply its operand, in the multiply-add that takes the 8 away:
//     code * factor is exact in 16 bits. (On the weights, ahead of their rounding, they cost less: 88.3 us for 92.3. But a factor goes
//     down to 2^-9 and took up to 9 bits of what fp16 has for small weights: beside a key of 2^20 times their weight
//     a group with factors of 2^-8 came out 4 % off in bf16; now 0.2 %, the output's own rounding.)
//
// Where the codes are: a K operand wants 16 values of a group in the four lanes of a key's row, a V operand 8 in each
// of the eight lanes g: lane (g, t) reads the 8 bytes t of a group from keys of number g and the 4 bytes g from keys of
// number 2t, 2t + 1. With TMA's swizzle (none where a row is 32 bytes) all of these reads are free of bank conflicts if the
// keys are numbered as `key_of_row` does.
//
// A warp's 64 keys of a step (32 for heads above 128), K, V and scales, come into a ring of its own, two steps under way,
// issued by one of its threads; it waits for nobody but its copies. Lengths are ragged, and starts and ends cost a block as
// much as a few steps, so the launch has as many blocks as the card holds at once (3 an SM) and each finds its equal share of all
// keys from the lengths, see `my_units`.
//
// Queries become fp16 by a power of two per row, exact down to 2^-24 of the row's largest value; the weights are rounded to fp16 once,
// relative to a power of two above the row scales of V that the row sees. Maxima, sums and O are 32 bits. Rescaling is lazy, see
// attn_decode.cu.
//
// Measured (B200, calls side by side in one graph): 64 sequences of 800 to 8000, 16/2 heads of 256 (154 MB) 48.9 us, 4 sequences
// to 100,003, 32/8 heads of 128 in pages of 32 (372 MB) 86.3; pages of 16 91.2, of 64 and more 84.0. What earlier versions took, with V's
// factors on the weights and its codes not signed (81.3 the last of them): a warp a row, 32 bits, 1667 and
// 3483; the MMAs, splits of 768 keys, K and V fetched by halves 65.8 and 134; whole steps, masks in a branch 60 and 115; splits of
// 1536 keys 54 and 109, of 4800 117 and 116; equal shares 71 and 93, with the queries loaded ahead of the copies and by all warps
// (6 us a segment before) 57 and 92, with a pair's start counted as two units 48.7 and 85.7 (these with the copies for a block's four
// warps by one thread). Left out: one tile less a warp and step for 4 blocks an SM (59 and 93.5: spills, and a step's fixed
// cost), P through shared memory and a group of O a warp (66 and 114: two barriers' waits), the last warp done with a block's
// step fetching the next (49 and 92), groups and tiles in rolled loops (73 and 120).
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
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
               : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}

__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
  const __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), *reinterpret_cast<const __half2*>(&c));
  return *reinterpret_cast<const uint32_t*>(&r);
}

constexpr uint32_t kLow = 0x000f000fu, kHigh = 0x00f000f0u;   // codes of an even byte, as numbers 2^-24 and 16 2^-24

// The codes of bytes 0 and 2 (odd: 1 and 3) of w as two fp16 numbers each: low ones by 2^-24, high ones by 16 2^-24. Integer
// instructions run at half rate: the second mask of the odd bytes is a subtraction.
__device__ __forceinline__ void two_codes(bool odd, uint32_t w, uint32_t& low, uint32_t& high) {
  if (odd) {
    const uint32_t both = __byte_perm(w, 0, 0x4341);
    low = both & kLow;
    high = hsub2(both, low);
  } else {
    low = w & kLow;
    high = w & kHigh;
  }
}

// Two e4m3 bytes (the low two of w) as fp16.
__device__ __forceinline__ uint32_t factors_f16(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 h;\n\tcvt.u16.u32 h, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, h;\n\t}" : "=r"(r) : "r"(w));
  return r;
}

// Shapes of one variant. G: groups of a row (codes past D are zeros); NT: 8-row tiles.
template <int G, int NT>
struct Shape4 {
  static constexpr int kWarps = 4;
  static constexpr int kRow = G > 2 ? 128 : 32 * G;     // bytes of a key's codes in shared memory
  static constexpr int kU = G > 2 ? 2 : 4;              // 16-key tiles of a warp a step
  static constexpr int kKeys = 16 * kU * kWarps;        // of a step
  static constexpr int kHalf = kKeys * kRow;            // K or V of a step
  static constexpr int kRecord = 64 + 16 * G;           // scales of 16 keys
  static constexpr int kScales = kKeys / 16 * kRecord;
  static constexpr int kStages = 2;                     // steps under way
  static constexpr int kPerSm = NT == 2 ? 2 : 3;        // blocks an SM, as registers allow
  static constexpr int kQ = NT * G * 1024;              // query fragments
  static constexpr int kRing = kStages * 2 * kHalf;
  static constexpr int kWidth = 64 * G + 4;             // of a row of O
  static constexpr int kJoin = kWarps * NT * 8 * kWidth * 4;   // the warps' O, over the ring
  // (three blocks an SM: 76 KB each, static and reserved memory of 2.5 KB included)
  static constexpr int kSmem = 1024 + (kRing > kJoin ? kRing : kJoin) + kStages * 2 * kScales + kQ;
  static_assert(kPerSm * (kSmem + 2560) <= 228 * 1024, "blocks an SM");
};

// The key of a tile that stands in row r (0..7) of the MMA's first 8; 8 on, that of row r + 8. Rows 0..3, rows 4..7,
// the even ones and the odd ones are each on four different 32-byte places of shared memory.
template <int ROW>
__device__ __forceinline__ int key_of_row(int r) {
  const int place = (r & 3) ^ (r >> 2), other = r >> 2;
  if (ROW == 128) return 2 * place + other;
  if (ROW == 64) return (place & 1) | other << 1 | (place & 2) << 1;
  return place + 4 * other;
}

// Work is counted in units of a block step (a step of each warp). Every pair (block of rows, key/value head) has its keys' units, at least one, and,
// where a block's share of all units is four or more, two for its start and its end. The launch's blocks take equal shares in
// order, so that lengths of any kind fill the card evenly; what a block has of one pair is a segment. Only pairs of more than
// a.whole units are split.
struct Place {
  int64_t x;     // units before the pair
  int item, h;   // block of rows (sequence by sequence), head
  int k;         // the pair's units before this one, its start not counted
};
struct Share {
  int64_t of;    // a block's
  int start;     // units of a pair's start
};

// (Not inlined, as what follows: run a few times a block, they would push the loop out of the instruction cache.)
template <int UNIT>
__device__ __noinline__ int units_of(const AttnArgs& a, int item) {
  const int b = a.row_blocks == 1 ? item : item / a.row_blocks;
  const AttnRows w = attn_rows(a, b, item - b * a.row_blocks);
  if (w.rows <= 0) return 0;
  int lo, hi;
  block_keys(a, w, lo, hi);
  return hi > lo ? (hi - lo - 1) / UNIT + 1 : 1;
}

__device__ __forceinline__ int64_t quotient(int64_t x, int64_t y) {
  return (x | y) >> 31 ? x / y : (int64_t)((uint32_t)x / (uint32_t)y);
}

// Where this block's units start and end (block-wide, 128 threads; false: it has none). Each thread counts a run of the
// items; the runs' sums are added up, and the thread whose run a boundary falls in finds it there.
template <int UNIT>
__device__ __noinline__ bool my_units(const AttnArgs& a, Place* ends, int64_t* sums, Share& share) {
  const int items = a.kv.seqs * a.row_blocks, run = (items + 127) >> 7, i0 = min(items, (int)threadIdx.x * run), i1 = min(items, i0 + run);
  int64_t units = 0;
  int pairs = 0, last = 0;
#pragma unroll 1
  for (int i = i0; i < i1; ++i) {
    last = units_of<UNIT>(a, i);
    units += last;
    pairs += last > 0;
  }
  // up to this thread: units, items with rows
  int64_t upto_u = units, upto_p = pairs;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, upto_u, o), z = __shfl_up_sync(0xffffffffu, upto_p, o);
    if ((threadIdx.x & 31) >= o) {
      upto_u += y;
      upto_p += z;
    }
  }
  if ((threadIdx.x & 31) == 31) {
    sums[2 * (threadIdx.x >> 5)] = upto_u;
    sums[2 * (threadIdx.x >> 5) + 1] = upto_p;
  }
  __syncthreads();
  int64_t total_u = 0, total_p = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < (int)(threadIdx.x >> 5)) {
      upto_u += sums[2 * i];
      upto_p += sums[2 * i + 1];
    }
    total_u += sums[2 * i];
    total_p += sums[2 * i + 1];
  }
  share.start = total_u * a.kv.heads >= 4 * (int64_t)gridDim.x ? 2 : 0;
  const int64_t total = (total_u + share.start * total_p) * a.kv.heads, mine = (units + share.start * pairs) * a.kv.heads,
                upto = (upto_u + share.start * upto_p) * a.kv.heads;
  share.of = quotient(total + gridDim.x - 1, gridDim.x);
  if (blockIdx.x * share.of >= total) return false;
#pragma unroll 1
  for (int e = 0; e < 2; ++e) {
    const int64_t x = (blockIdx.x + e) * share.of;
    if (x >= total) {
      if (threadIdx.x == 0) ends[e] = {total, items, 0, 0};
    } else if (x >= upto - mine && x < upto) {
      Place p = {upto - mine, i0, 0, 0};
      int n;   // of a pair
#pragma unroll 1
      for (;; ++p.item) {
        n = run == 1 ? last : units_of<UNIT>(a, p.item);
        if (n == 0) continue;
        n += share.start;
        if (x < p.x + (int64_t)n * a.kv.heads) break;
        p.x += (int64_t)n * a.kv.heads;
      }
      p.h = (int)quotient(x - p.x, n);
      p.x += (int64_t)p.h * n;
      p.k = max(0, (int)(x - p.x) - share.start);
      n -= share.start;
      if (n <= a.whole) {   // whole: the nearer end
        if (2 * p.k >= n) {
          p.x += n + share.start;
          if (++p.h == a.kv.heads) {
            p.h = 0;
            do ++p.item; while (p.item < items && units_of<UNIT>(a, p.item) == 0);
          }
        }
        p.k = 0;
      }
      ends[e] = p;
    }
  }
  __syncthreads();
  return ends[0].item != ends[1].item || ends[0].h != ends[1].h || ends[0].k != ends[1].k;
}

// How many blocks, from that with unit x on, have the n units from there on.
__device__ __noinline__ int blocks_of(int64_t x, int n, int64_t share) {
  return (int)(quotient(x + n - 1, share) - quotient(x, share)) + 1;
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

template <int G, int NT, typename T>
__global__ void __launch_bounds__(Shape4<G, NT>::kWarps * 32, Shape4<G, NT>::kPerSm)
    attn_decode4_kernel(const __grid_constant__ AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using S = Shape4<G, NT>;
  constexpr int U = S::kU, ROW = S::kRow, UNIT = S::kKeys, ST = S::kStages, REC = S::kRecord;
  // weights 2^7 larger than the maximum asks for, so that those down to 2^-32 of the largest are more than 0 (of keys whose V scale
  // is the largest; 2^-32 over its share of that otherwise)
  constexpr float kLift = 7.f, kDrop = 1.f / 128.f;
  extern __shared__ unsigned char decode4_raw[];
  unsigned char* sm = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(decode4_raw) + 1023) & ~uintptr_t(1023));
  unsigned char* q_s = sm + (S::kRing > S::kJoin ? S::kRing : S::kJoin) + ST * 2 * S::kScales;
  __shared__ uint64_t full[S::kWarps][ST];
  __shared__ float2 red[S::kWarps][NT * 8];
  __shared__ float qexp_s[NT * 8], qtop_s[G][NT * 8];
  __shared__ float4 start_s[NT][G][4];
  __shared__ Place ends[2];
  __shared__ int64_t sums[8];
  if (threadIdx.x < 2)   // constant: ahead of the wait
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(threadIdx.x ? &vmap : &kmap)) : "memory");
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t ring = su32(sm), scales = su32(q_s) - ST * 2 * S::kScales, q_sm = su32(q_s), full0 = su32(&full[warp][0]);
  if (threadIdx.x == 0) {
    for (int i = 0; i < ST * S::kWarps; ++i) mbar_init(full0 + 8 * i, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    fence_proxy_async();
  }
  Share share;
  const bool any = my_units<UNIT>(a, ends, sums, share);
  const Place end = ends[1];
  const int page_mask = (1 << a.kv.page_log2) - 1;
  // A copy is a box of the warp's keys of a step, as many as a page has; boxes are found by a lane each and issued by one thread.
  const int box_keys = min(1 << a.kv.page_log2, 16 * U), boxes = 16 * U / box_keys, box_record = (box_keys >> 4) * REC;
  // this lane's places: K's key (another 8 on), V's keys of the MMA's rows 2t, 2t + 1 (others 8 on); 32 bytes a group
  auto swizzled = [](int key, int byte) {
    const int x = ROW == 128 ? key & 7 : ROW == 64 ? (key >> 1) & 3 : 0;
    return (uint32_t)(key * ROW + (byte ^ (x << 4)));
  };
  const int kkey = key_of_row<ROW>(g), vkey0 = key_of_row<ROW>(2 * t), vkey1 = key_of_row<ROW>(2 * t + 1);
  const uint32_t vkeys = vkey0 | vkey1 << 4;   // as bytes of 8 factors
  const uint32_t kx = swizzled(kkey, 8 * t), vx[2] = {swizzled(vkey0, 4 * g), swizzled(vkey1, 4 * g)};
  uint32_t done = 0;              // steps of the segments so far
  bool lost = false, ok = true;   // a wait of this warp, none of the block's has given up

  int item = ends[0].item, h = ends[0].h, unit0 = ends[0].k;
  int64_t x = ends[0].x;
#pragma unroll 1
  for (bool more = any; more;) {   // ---- a segment
    const int b = a.row_blocks == 1 ? item : item / a.row_blocks;
    const AttnRows w = attn_rows(a, b, item - b * a.row_blocks);
    int lo, hi;
    block_keys(a, w, lo, hi);
    const int n_units = hi > lo ? (hi - lo - 1) / UNIT + 1 : 1;
    const int take = (item == end.item && h == end.h ? end.k : n_units) - unit0;
    const int s0 = lo + unit0 * UNIT, s1 = (int)min((int64_t)hi, s0 + (int64_t)take * UNIT);
    const bool alone = take == n_units;
    if (unit0 == 0 && threadIdx.x == 0)   // for the joining launch: who has this pair
      a.segments[(int64_t)item * a.kv.heads + h] = make_int2(blockIdx.x, alone ? 1 : blocks_of(x + share.start, n_units, share.of));
    const int32_t* table = a.kv.table + b * a.kv.table_stride;
    const int seen = row_lo(a, w, w.r0 / a.G);
    const int steps = ok && s1 > s0 ? (s1 - s0 + S::kKeys - 1) / S::kKeys : 0;
    const uint32_t first = done;   // the segment's first step
    // The queries first, ahead of the copies that fill the memory's queues: a group of 8 rows a warp, 16 values a lane.
    constexpr int QW = (NT * G + 3) / 4;
    uint4 qv[QW][2];
#pragma unroll
    for (int p = 0; p < QW; ++p) {
      const int e = warp + 4 * p, i = e / G, r = 8 * i + g, d = 64 * (e % G) + 16 * t;
      qv[p][0] = qv[p][1] = make_uint4(0, 0, 0, 0);
      if (e < NT * G && r < w.rows && d < a.D) {
        const int tok = (w.r0 + r) / a.G;
        const uint4* from = reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (int64_t)(w.first + tok) * a.q_ts +
                                                           (int64_t)(h * a.G + w.r0 + r - tok * a.G) * a.q_hs + d);
        qv[p][0] = from[0];
        qv[p][1] = from[1];
      }
    }
    // page of the lane's box of step i; -1 where there is none or its keys are past (looked up a step ahead)
    auto page_of = [&](int i) {
      const int k = s0 + S::kKeys * i + 16 * U * warp + lane * box_keys;
      return lane < boxes && i < steps && k < s1 && (k | page_mask) >= seen ? table[k >> a.kv.page_log2] : -1;
    };
    int put = 0;   // the segment's step that the warp fetches next
    uint32_t gone = 0;   // a byte a stage: the boxes whose pages are not in the pool
    int ahead = page_of(0);
    auto fetch = [&]() {
      if (put >= steps) return;
      const uint32_t step = first + put, st = step % ST, bar = full0 + 8 * st;
      const bool there = ahead >= 0 && ahead < a.kv.pages;
      const uint32_t out = __ballot_sync(0xffffffffu, lane < boxes && !there);
      // a page that exists stands in for one that does not
      const int rows = (((there ? ahead : 0) * a.kv.heads + h) << a.kv.page_log2) + ((s0 + S::kKeys * put + 16 * U * warp + lane * box_keys) & page_mask);
      gone &= ~(0xffu << (8 * st));
      gone |= out << (8 * st);
      ahead = page_of(++put);
#pragma unroll 1
      for (int c = 0; c < boxes; ++c) {
        const int row = __shfl_sync(0xffffffffu, rows, c);
        if (elect_one()) {
          if (c == 0) mbar_arrive_tx(bar, 2 * (S::kHalf + S::kScales) / S::kWarps);
          const uint32_t to = ring + st * 2 * S::kHalf + (16 * U * warp + c * box_keys) * ROW, to_s = scales + st * 2 * S::kScales + warp * U * REC + c * box_record;
          const int64_t from = (int64_t)(row >> 4) * REC;
          tma_load_2d(to, &kmap, 0, row, bar);
          bulk_load(to_s, reinterpret_cast<const unsigned char*>(a.kv.k_scale) + from, box_record, bar);
          tma_load_2d(to + S::kHalf, &vmap, 0, row, bar);
          bulk_load(to_s + S::kScales, reinterpret_cast<const unsigned char*>(a.kv.v_scale) + from, box_record, bar);
        }
      }
    };
#pragma unroll 1
    for (int i = 0; i < ST; ++i) fetch();

    // ---- queries as B fragments, in the order of K's codes: of a group's 16 values of lane t, word w holds 8 w .. 8 w + 7,
    // and its MMA j takes values 2 j, 2 j + 4 and 2 j + 1, 2 j + 5 (these by 16)
#pragma unroll
    for (int p = 0; p < QW; ++p) {
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 f = unpack2<T>((&qv[p][j >> 2].x)[j & 3]);
        top = fmaxf(top, fmaxf(fabsf(f.x), fabsf(f.y)));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = warp + 4 * p;
      if (t == 0 && e < NT * G) qtop_s[e % G][8 * (e / G) + g] = top;
    }
    __syncthreads();
#pragma unroll
    for (int p = 0; p < QW; ++p) {
      const int n = warp + 4 * p, i = n / G, k = n % G;
      if (n >= NT * G) break;
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < G; ++c) top = fmaxf(top, qtop_s[c][8 * i + g]);
      const int e = fp16_lift(top);
      const float by = __int_as_float((127 + e) << 23);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float f[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 y = unpack2<T>((&qv[p][c].x)[j]);
          f[2 * j] = y.x * by;
          f[2 * j + 1] = y.y * by;
        }
        uint4 o;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const uint32_t b0 = pack2<__half>(f[2 * j], f[2 * j + 4]);
          const uint32_t b1 = pack2<__half>(f[2 * j + 1] * 0.0625f, f[2 * j + 5] * 0.0625f);
          (&o.x)[2 * j] = b0;
          (&o.x)[2 * j + 1] = b1;
          const float2 y = unpack2<__half>(b0), z = unpack2<__half>(b1);
          sum += (y.x + y.y) + 16.f * (z.x + z.y);
        }
        *reinterpret_cast<uint4*>(q_s + (n * 2 + c) * 512 + lane * 16) = o;
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      if (t == 0) {   // what a group's sum starts at, as the MMA's four of the lanes with row 8 i + g
        float* to = reinterpret_cast<float*>(&start_s[i][k][g >> 1]) + (g & 1);
        to[0] = to[2] = sum * (-8.f / 16777216.f);
        if (k == 0) qexp_s[8 * i + g] = __int_as_float((127 - e) << 23);
      }
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
        const bool there = r < w.rows;
        const int tok = (w.r0 + (there ? r : 0)) / a.G;
        klo[i][c] = row_lo(a, w, tok);
        khi[i][c] = there ? row_hi(a, w, tok) : 0;
        sc[i][c] = a.scale_log2 * qexp_s[r];
      }
    // keys that every row sees need no mask
    const int all_lo = row_lo(a, w, (w.r0 + w.rows - 1) / a.G), all_hi = min(s1, row_hi(a, w, w.r0 / a.G));

    // o: sums of values d (0, 1) and d + 1 (2, 3)
    float o[NT][4 * G][4], m[NT][2], l[NT][2], vref[NT][2];
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int j = 0; j < 4 * G; ++j) o[i][j][c] = 0.f;
      m[i][0] = m[i][1] = -INFINITY;
      l[i][0] = l[i][1] = vref[i][0] = vref[i][1] = 0.f;
    }

#pragma unroll 1
    for (int n = 0; n < steps; ++n) {
      const uint32_t step = first + n, st = step % ST;
      lost |= !copy_wait(full0 + 8 * st, (step / ST) & 1);
      if (__any_sync(0xffffffffu, lost)) break;
      const uint32_t src = ring + st * 2 * S::kHalf + warp * U * 16 * ROW;
      const uint32_t k_rec = scales + st * 2 * S::kScales + warp * U * REC, v_rec = k_rec + S::kScales;
      // ---- S^T = K Q^T, a group's sum times its factor
      float s[U][NT][4];
#pragma unroll
      for (int k = 0; k < G; ++k) {
        uint4 q[NT][2];
        float4 start[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          start[i] = start_s[i][k][t];
#pragma unroll
          for (int c = 0; c < 2; ++c) q[i][c] = lds16(q_sm + ((i * G + k) * 2 + c) * 512 + lane * 16);
        }
        uint2 kc[U], kd[U];
        float2 f[U];   // factors, by 2^-8: their bits as fp16's
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const uint32_t at = src + u * 16 * ROW + (kx ^ (32 * k)), fa = k_rec + u * REC + 64 + 16 * k + kkey;
          kc[u] = lds8(at);
          kd[u] = lds8(at + 8 * ROW);
          f[u] = unpack2<__half>((lds1(fa) | lds1(fa + 8) << 16) << 7);
        }
        // the tiles side by side: a sum's next MMA does not wait for the one before
        float acc[U][NT][4];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int u = 0; u < U; ++u) {
            uint32_t a0, a1, a2, a3;
            two_codes(c & 1, c & 2 ? kc[u].y : kc[u].x, a0, a2);
            two_codes(c & 1, c & 2 ? kd[u].y : kd[u].x, a1, a3);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
              const uint32_t b0 = c & 1 ? q[i][c >> 1].z : q[i][c >> 1].x, b1 = c & 1 ? q[i][c >> 1].w : q[i][c >> 1].y;
              if (c == 0) mma(acc[u][i], a0, a1, a2, a3, b0, b1, start[i].x, start[i].y, start[i].z, start[i].w);
              else mma(acc[u][i], a0, a1, a2, a3, b0, b1);
            }
          }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const float by = c < 2 ? f[u].x : f[u].y;
              s[u][i][c] = k ? fmaf(acc[u][i][c], by, s[u][i][c]) : acc[u][i][c] * by;
            }
      }
      float vs[U][2];   // V's row scales
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float ks[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t at = u * REC + 4 * (kkey + 8 * e);
          ks[e] = lds_f32(k_rec + at);
          vs[u][e] = lds_f32(v_rec + at);
        }
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) s[u][i][c] = s[u][i][c] * 4294967296.f * (sc[i][c & 1] * ks[c >> 1]);   // 2^24 of the codes, 2^8 of the factors
      }
      // ---- masks
      const int k0 = s0 + n * S::kKeys + warp * U * 16;
      const uint32_t out = gone >> (8 * st) & 0xffu;
      uint32_t hidden = 0;   // the masked ones of this lane's weights
      if (!(k0 >= all_lo && k0 + 16 * U <= all_hi && !out)) {
        static_assert(U * NT * 4 <= 32, "bits of hidden");
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int left = (out >> (16 * u / box_keys)) & 1 ? 0 : s1 - k0 - 16 * u;   // keys of the tile that there are
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (kkey + 8 * e >= left) vs[u][e] = 0.f;   // what lies past them is no scale
#pragma unroll
          for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              const int key = kkey + 8 * (c >> 1), p = k0 + 16 * u + key;
              if (key >= left || p < klo[i][c & 1] || p >= khi[i][c & 1]) {
                s[u][i][c] = -INFINITY;
                hidden |= 1u << ((u * NT + i) * 4 + c);
              }
            }
          // nor a factor: 0 * NaN would not be 0 (a group's 16 in the lanes 4 k .. 4 k + 3)
          if (lane < 4 * G) {
            const uint32_t at = v_rec + u * REC + 64 + 4 * lane;
            const int in = left - 4 * (lane & 3);
            if (in < 4) asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(in > 0 ? lds4(at) & ((1u << (8 * in)) - 1) : 0u) : "memory");
          }
        }
        fence_proxy_async();   // ahead of the copy that takes this place next
        __syncwarp();
      }
      // ---- the running maximum, and the V scale that weights are relative to
      bool high = false;
      float vlow = INFINITY;   // what every row's vref covers
#pragma unroll
      for (int i = 0; i < NT; ++i) vlow = fminf(vlow, fminf(vref[i][0], vref[i][1]));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        high |= vs[u][0] > vlow || vs[u][1] > vlow;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) high |= s[u][i][c] > m[i][c & 1] + (8.f + kLift);
      }
      if (__any_sync(0xffffffffu, high)) {
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = -INFINITY, y = 0.f;   // y: of the keys that the row sees: a hidden one's scale must not cost it bits
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                top = fmaxf(top, s[u][i][c + 2 * e]);
                if (s[u][i][c + 2 * e] != -INFINITY) y = fmaxf(y, vs[u][e]);
              }
#pragma unroll
            for (int f = 4; f <= 16; f <<= 1) {
              top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, f));
              y = fmaxf(y, __shfl_xor_sync(0xffffffffu, y, f));
            }
            float undo = 1.f;
            if (y > vref[i][c]) {
              const float ref = above(y);
              undo = vref[i][c] / ref;
              vref[i][c] = ref;
            }
            const float mn = fmaxf(m[i][c], top - kLift);
            const float by = mn == -INFINITY ? 1.f : ex2(m[i][c] - mn);
            m[i][c] = mn;
            l[i][c] *= by;
#pragma unroll
            for (int j = 0; j < 4 * G; ++j) {
              o[i][j][c] *= by * undo;
              o[i][j][c + 2] *= by * undo;
            }
          }
      }
      // ---- P^T: columns summed, weights relative to the V scale
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        // 1 / vref, a power of two (2^127 where no scale but 0 has been seen); m, or 0 while no key has been seen
        const float vinv[2] = {__int_as_float(0x7f000000 - __float_as_int(vref[i][0])), __int_as_float(0x7f000000 - __float_as_int(vref[i][1]))};
        const float base[2] = {m[i][0] == -INFINITY ? 0.f : m[i][0], m[i][1] == -INFINITY ? 0.f : m[i][1]};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const float p = ex2(s[u][i][c] - base[c & 1]);
            l[i][c & 1] += p;
            s[u][i][c] = p * (vs[u][c >> 1] * vinv[c & 1]);
          }
        if (hidden) {   // a masked key's scale may be anything: 0 * inf, 0 * NaN
#pragma unroll
          for (int u = 0; u < U; ++u)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (hidden >> ((u * NT + i) * 4 + c) & 1) s[u][i][c] = 0.f;
        }
      }
      // ---- O^T += V^T P^T, P rounded and turned into B fragments
      uint32_t p0[U][NT], p1[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < NT; ++i) {
          p0[u][i] = transpose8x8(pack2<__half>(s[u][i][0], s[u][i][1]));
          p1[u][i] = transpose8x8(pack2<__half>(s[u][i][2], s[u][i][3]));
        }
#pragma unroll
      for (int k = 0; k < G; ++k) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          // factors of keys 2t, 2t + 1 and of those 8 on; code * factor comes out 2^-9 times as large, a code of 2^-24 times
          // 2^15 factor: none of it is lost, as factors are multiples of 2^-9
          const uint4 fw = lds16(v_rec + u * REC + 64 + 16 * k);
          const uint32_t fy = factors_f16(__byte_perm(fw.x, fw.y, vkeys)), fz = factors_f16(__byte_perm(fw.z, fw.w, vkeys));
          const uint32_t yl = hmul2(fy, 0x78007800u), yh = hmul2(fy, 0x68006800u), y8 = hmul2(fy, 0xa400a400u);   // 2^15, 2^11, -2^-6 (8 codes)
          const uint32_t zl = hmul2(fz, 0x78007800u), zh = hmul2(fz, 0x68006800u), z8 = hmul2(fz, 0xa400a400u);
          const uint32_t at = src + S::kHalf + u * 16 * ROW, b0 = at + (vx[0] ^ (32 * k)), b1 = at + (vx[1] ^ (32 * k));
          const uint32_t w0 = lds4(b0), w1 = lds4(b1), w2 = lds4(b0 + 8 * ROW), w3 = lds4(b1 + 8 * ROW);
#pragma unroll
          for (int j = 0; j < 4; ++j) {   // values 2 j and 2 j + 1 of each lane's 8
            uint32_t y0, y1, z0, z1;
            two_codes(j & 1, __byte_perm(w0, w1, j < 2 ? 0x5410 : 0x7632), y0, y1);
            two_codes(j & 1, __byte_perm(w2, w3, j < 2 ? 0x5410 : 0x7632), z0, z1);
#pragma unroll
            for (int i = 0; i < NT; ++i)
              mma(o[i][4 * k + j], hfma2(y0, yl, y8), hfma2(y1, yh, y8), hfma2(z0, zl, z8), hfma2(z1, zh, z8), p0[u][i], p1[u][i]);
          }
        }
      }
      __syncwarp();   // the stage is used up
      fetch();
    }
    done += steps;
    if (__syncthreads_or(lost)) {   // copies under way have landed before the ring's memory is used for anything else
      ok = false;
      for (uint32_t i = first + max(0, put - ST); i < first + put; ++i) copy_wait(full0 + 8 * (i % ST), (i / ST) & 1);
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NT; ++i) l[i][0] = l[i][1] = __int_as_float(0x7fffffff);   // the rows come out as NaN
    } else if (!ok) {
#pragma unroll
      for (int i = 0; i < NT; ++i) l[i][0] = l[i][1] = __int_as_float(0x7fffffff);
    }

    // ---- join the warps: maximum, then sums relative to it
    constexpr float kUnit = 512.f * kDrop;        // 2^9 of code * factor
    constexpr int LD = S::kWidth;
    float* acc = reinterpret_cast<float*>(sm);    // [warp][row][64 G + 4]
#pragma unroll
    for (int i = 0; i < NT; ++i)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float y = l[i][c];
        y += __shfl_xor_sync(0xffffffffu, y, 4);
        y += __shfl_xor_sync(0xffffffffu, y, 8);
        y += __shfl_xor_sync(0xffffffffu, y, 16);
        if (g == 0) red[warp][8 * i + 2 * t + c] = make_float2(m[i][c] + kLift, y * kDrop);
#pragma unroll
        for (int k = 0; k < G; ++k)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            *reinterpret_cast<float2*>(acc + (warp * NT * 8 + 8 * i + 2 * t + c) * LD + 64 * k + 8 * g + 2 * j) =
                make_float2(o[i][4 * k + j][c] * kUnit * vref[i][c], o[i][4 * k + j][c + 2] * kUnit * vref[i][c]);
      }
    __syncthreads();
#pragma unroll 1
    for (int e = threadIdx.x; e < w.rows * (16 * G); e += S::kWarps * 32) {
      const int r = e / (16 * G), d = e % (16 * G) * 4;
      if (d >= a.D) continue;
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < S::kWarps; ++k) top = fmaxf(top, red[k][r].x);
      const float base = top == -INFINITY ? 0.f : top;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int k = 0; k < S::kWarps; ++k) {
        const float by = ex2(red[k][r].x - base);
        const float4 z = *reinterpret_cast<const float4*>(acc + (k * NT * 8 + r) * LD + d);
        sum += red[k][r].y * by;
        y.x += z.x * by;
        y.y += z.y * by;
        y.z += z.z * by;
        y.w += z.w * by;
      }
      if (alone) {
        const int row = w.r0 + r;
        const int64_t at = (int64_t)(w.first + row / a.G) * a.hq + h * a.G + row % a.G;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.D + d) =
            make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
        if (a.lse && d == 0) a.lse[at] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * kLn2;
      } else {
        // a block has at most one segment that a pair starts with and does not end with, and one that it goes on with
        const int64_t at = ((int64_t)blockIdx.x * 2 + (unit0 == 0)) * a.rows_per_block + r;
        *reinterpret_cast<float4*>(a.part_o + at * a.D + d) = y;
        if (d == 0) a.part_ml[at] = make_float2(top, sum);
      }
    }
    more = unit0 + take == n_units;   // the pair ends here
    if (more) {
      x += n_units + share.start;
      unit0 = 0;
      if (++h == a.kv.heads) {
        h = 0;
        do ++item; while (item < a.kv.seqs * a.row_blocks && units_of<UNIT>(a, item) == 0);
      }
      more = item != end.item || h != end.h || end.k != 0;
    }
    if (more) {
      fence_proxy_async();   // the ring's memory goes back to the copies
      __syncthreads();
    }
  }
  if (a.kv.starts) {   // tokens of no sequence
    const int first = max(0, min(a.kv.starts[0], a.T)), past = max(first, min(a.kv.starts[a.kv.seqs], a.T));
    if (first > 0) blank_tokens(a, 0, first, blockIdx.x, gridDim.x);
    if (past < a.T) blank_tokens(a, past, a.T, blockIdx.x, gridDim.x);
  }
}

// Joins the segments of a row (token, head) that has more than one: a block takes 4 * LANES of its values, LANES threads of
// them for each of 256 / LANES shares of the segments; the shares are then added in order.
template <typename T, int LANES>
__global__ void __launch_bounds__(256) attn_join4_kernel(const __grid_constant__ AttnArgs a) {
  __shared__ float4 acc[256];
  __shared__ float red[8], sum_s[256 / LANES];
  // Of what is read ahead of the wait nothing is written by the launch before, and that one has waited for all before it.
  const int t = blockIdx.x, hq = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = sequence_of(a.kv, t);
  int64_t row = -1, pair = 0;
  if (b >= 0) {
    row = (int64_t)(t - attn_rows(a, b, 0).first) * a.G + hq % a.G;
    if (row >= (int64_t)a.row_blocks * a.rows_per_block) row = -1;   // past max_new
  }
  int r = 0;
  if (row >= 0) {
    const int rb = (int)row / a.rows_per_block;
    r = (int)row - rb * a.rows_per_block;
    if (r >= attn_rows(a, b, rb).rows) row = -1;
    pair = ((int64_t)b * a.row_blocks + rb) * a.kv.heads + hq / a.G;
  }
  pdl_wait();   // by every block: what follows this launch takes its end for the end of the one before too
  pdl_trigger();
  if (row < 0) return;
  const int2 seg = a.segments[pair];
  if (seg.y <= 1) return;   // written already
  // part of segment i: the first one's is its block's second
  auto part = [&](int i) { return ((int64_t)(seg.x + i) * 2 + (i == 0)) * a.rows_per_block + r; };
  float top = -INFINITY;
  for (int i = threadIdx.x; i < seg.y; i += 256) top = fmaxf(top, a.part_ml[part(i)].x);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if (lane == 0) red[warp] = top;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) top = fmaxf(top, red[k]);
  const float base = top == -INFINITY ? 0.f : top;
  constexpr int kShares = 256 / LANES;
  const int share = threadIdx.x / LANES, d = 4 * (blockIdx.z * LANES + threadIdx.x % LANES);
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int i = share; i < seg.y; i += kShares) {
    const int64_t p = part(i);
    const float2 ml = a.part_ml[p];
    const float by = ex2(ml.x - base);
    sum += ml.y * by;
    if (d < a.D) {
      const float4 z = *reinterpret_cast<const float4*>(a.part_o + p * a.D + d);
      y.x += z.x * by;
      y.y += z.y * by;
      y.z += z.z * by;
      y.w += z.w * by;
    }
  }
  acc[threadIdx.x] = y;
  if (threadIdx.x % LANES == 0) sum_s[share] = sum;
  __syncthreads();
  if (share) return;
  sum = sum_s[0];
#pragma unroll
  for (int k = 1; k < kShares; ++k) {
    sum += sum_s[k];
    const float4 z = acc[LANES * k + threadIdx.x];
    y.x += z.x;
    y.y += z.y;
    y.z += z.z;
    y.w += z.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int64_t at = (int64_t)t * a.hq + hq;
  if (d < a.D)
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + at * a.D + d) =
        make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
  if (a.lse && d == 0) a.lse[at] = sum == 0.f ? -INFINITY : (base + log2f(sum)) * kLn2;
}

// A pool's codes [rows, D / 2] as boxes of `keys` rows x `row` bytes, swizzled over the row; bytes past D / 2 read as zeros.
bool make_code_map(CUtensorMap* map, const void* base, const AttnArgs& a, int row, int keys) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.D / 2), (static_cast<cuuint64_t>(a.kv.pages) * a.kv.heads) << a.kv.page_log2};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(a.D / 2)};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(row), static_cast<cuuint32_t>(keys)};
  const cuuint32_t es[2] = {1, 1};
  return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, boxes, es,
                     CU_TENSOR_MAP_INTERLEAVE_NONE,
                     row == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : row == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE,
                     CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int G, int NT, typename T>
int launch(AttnArgs a, cudaStream_t st) {
  using S = Shape4<G, NT>;
  auto kern = attn_decode4_kernel<G, NT, T>;
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
  CUtensorMap kmap, vmap;
  const int keys = 16 * S::kU < 1 << a.kv.page_log2 ? 16 * S::kU : 1 << a.kv.page_log2;
  a.lo_mask = ~(keys - 1);   // a box lies in a page
  if (!make_code_map(&kmap, a.kv.k, a, S::kRow, keys) || !make_code_map(&vmap, a.kv.v, a, S::kRow, keys)) return VQ2_ERR_LAUNCH;
  return launch_kernel(kern, dim3((unsigned)a.blocks), dim3(S::kWarps * 32), S::kSmem, st, a, kmap, vmap);
}

// f(shape, groups, row tiles) of the variant for `a`.
template <typename F>
auto with_shape(const AttnArgs& a, F f) {
  using std::integral_constant;
  auto rows = [&](auto groups) {
    return a.rows_per_block == 8 ? f(groups, integral_constant<int, 1>()) : f(groups, integral_constant<int, 2>());
  };
  if (a.D > 192) return rows(integral_constant<int, 4>());
  if (a.D > 128) return rows(integral_constant<int, 3>());
  return a.D > 64 ? rows(integral_constant<int, 2>()) : rows(integral_constant<int, 1>());
}

template <typename T>
int launch_shape(const AttnArgs& a, cudaStream_t st) {
  return with_shape(a, [&](auto g, auto nt) { return launch<decltype(g)::value, decltype(nt)::value, T>(a, st); });
}

}  // namespace

void plan_attn_decode4(AttnArgs& a, int64_t max_new, int64_t max_len) {
  const int64_t rows = max_new * a.G;
  const int nt = rows <= 8 ? 1 : 2;
  a.rows_per_block = 8 * nt;
  a.row_blocks = (int)((rows + 8 * nt - 1) / (8 * nt));
  if (a.row_blocks < 1) a.row_blocks = 1;
  a.splits = 1;
  a.chunk = 0x7fffffff;
  int unit = 0, per_sm = 0;
  with_shape(a, [&](auto g, auto nt) {
    using S = Shape4<decltype(g)::value, decltype(nt)::value>;
    unit = S::kKeys;
    per_sm = S::kPerSm;
    return 0;
  });
  int64_t keys = max_len;
  if (a.window && a.window + max_new < keys) keys = a.window + max_new;
  // the first key is rounded down by less than a unit
  const int64_t units = (keys + unit - 2) / unit + 1, pairs = (int64_t)a.kv.seqs * a.row_blocks * a.kv.heads;
  const int64_t room = (int64_t)sm_count() * per_sm;
  a.blocks = (int)(pairs >= room || units >= room || pairs * units >= room ? room : pairs * units);
  // Pairs of two units stay whole: a joining launch and a second start cost more than they take. Where no pair is longer, by the
  // caller's bounds, nothing is split and no joining launch follows; with pairs for a quarter of the blocks, where none is
  // longer than eight (32 sequences of 1100, 32/8 heads of 128: split 24.8 us, whole 22.5; 64 of 500, 16/2 of 256: 21.9, 20.6;
  // 8 of 600, 16/2 of 256, 16 pairs: 12.2, 16.9).
  a.whole = units <= (4 * pairs >= room ? 8 : 2) ? 0x7fffffff : 2;
}

int launch_attn_decode4(const AttnArgs& a, cudaStream_t st) {
  if (!encode_fn()) return VQ2_ERR_LAUNCH;
  const int s = a.q_bf16 ? launch_shape<__nv_bfloat16>(a, st) : launch_shape<__half>(a, st);
  if (s != VQ2_OK || a.whole == 0x7fffffff) return s;
  // Few rows of many segments: 64 values a block, 16 segments read at once; else whole rows.
  const int lanes = (int64_t)a.T * a.hq < 2 * sm_count() || a.D <= 64 ? 16 : a.D <= 128 ? 32 : 64;
  const dim3 grid((unsigned)a.T, (unsigned)a.hq, (unsigned)((a.D + 4 * lanes - 1) / (4 * lanes)));
  auto join = [&](auto type) {
    using T = decltype(type);
    return launch_kernel(lanes == 16 ? attn_join4_kernel<T, 16> : lanes == 32 ? attn_join4_kernel<T, 32> : attn_join4_kernel<T, 64>,
                         grid, dim3(256), 0, st, a);
  };
  return a.q_bf16 ? join(__nv_bfloat16()) : join(__half());
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
