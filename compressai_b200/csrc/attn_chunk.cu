// Attention of many query rows per key/value head over a paged cache: chunks and whole prompts, on
// the tensor cores (tcgen05) with scores and output in tensor memory.
//
//   S = Q K^T,   P = 2^(S * scale - m),   O += P V      (128 rows x 128 keys a step)
//
// Rows are (new token, head of the group) pairs, so one tile of keys serves every head that shares
// it. A block (head sizes above 128: a pair of blocks) owns 256 rows, O staying in tensor memory, and
// walks the keys once. Roles:
//   * one thread brings keys and values by TMA, straight from their pages: 16 KB blocks in a ring, a
//     K block being 128 keys x 64 values, a V block 8192 / DP keys x all values, 128-byte swizzle;
//   * one thread issues the MMAs: S from shared memory, O with P as the operand in tensor memory
//     (P overwrites its S, each softmax thread's within its own columns) and V with its values
//     contiguous (the descriptor's transposed form);
//   * 16 warps do the softmax, 2 or 4 threads a row: with one thread a row (a warp a scheduler and
//     row tile) the chain of its 128 maxima and exponentials set the pace: 3 us a step where the
//     MMAs take 1.1. The threads of a row agree through one named barrier whether any score asks
//     for a new maximum. Maxima, sums and O are 32 bits; P is rounded to the cache's 16 bits.
// Head sizes above 128 run as pairs of blocks (cluster of 2, cta_group::2): an MMA then spans both, each
// holding 128 of 256 rows in its tensor memory and half of K's keys and V's values in its shared memory,
// so that a step's 128 KB serve 256 rows as they do for smaller heads (prompt of 8192 tokens, 16/2 heads
// of 256: 684 us with one block per 128 rows, 502 with pairs, the loads as they were then).
//
// With two row tiles the tensor core works on one while the softmax works on the other; with one
// (head size 256, O takes half of tensor memory) S is double-buffered and QK of the next tile runs
// under the softmax.
//
// The running maximum moves only when a score passes it by 8 powers of two (P is at most 256; fp16: 2^15),
// which is rare after the first tiles: O is rescaled in tensor memory by the softmax threads
// themselves, and no separate correction stage stands in the loop.
//
// Bound: a step of 256 rows x 128 keys is 2048 cycles of MMA at head size 128 (in each block of a pair at
// 256) and, at 16 exponentials a clock an SM, 2048 (1024) of exponentials. Measured 3700 cycles at 128,
// the chain softmax -> weights -> O -> next scores of a row tile; 2350 at 256 (prompt of 8192 tokens
// 401 us, 1.37 PFLOP/s).
//
// 8-bit caches: a launch before this one writes the visible keys and values out once as exact fp16 (an
// int8 is; see attn_decode.cu, also for the scales: the key's multiplies the score, the value's the
// weight, relative to a power of two), in order and without pages, and this kernel reads those. Every
// block of rows would convert the same keys again: warps that did so inside this kernel, beside the
// softmax, took 4700 cycles an operand tile (two chunks of 257 tokens over 16385, 34 blocks a
// sequence: 359 us).
//
// Rows of a page past the keys that the block sees may hold anything, NaN too: their scores are
// replaced, and their V rows zeroed in shared memory by the loading warp before the MMA may read
// them (at most one block per launch block holds such rows; blocks and pages wholly outside are not
// read: the copy's coordinate is put past the pool, which fills zeros).
//
// Every wait is bounded by the SM clock (about 2 s): one that gives up raises the abort flag and
// vq2_attention_status, every role leaves its loop, copies and MMAs in flight are drained, the rows are NaN.
#include <atomic>
#include <type_traits>

#include "attn_dev.cuh"
#include "tcgen05.cuh"

// Sticky status of the chunk kernel: VQ2_ERR_TIMEOUT once any bounded wait gave up.
__device__ int32_t g_attention_status;

namespace vq2 {
namespace {

constexpr long long kWaitCycles = 4000000000LL;  // ~2 s at 1.965 GHz
constexpr int kBlock = 16384;                    // bytes of a ring block

template <int DP, bool I8>
struct ChunkShape {
  static constexpr bool Pair = DP > 128;             // two blocks work as one, each with half of K and V
  static constexpr int NQ = Pair ? 1 : 2;            // row tiles of 128 in a block
  static constexpr int QC = DP / 64;                 // 16 KB blocks of a row tile's queries
  static constexpr int B = Pair ? 2 : DP / 64;       // ring blocks of a 128-key tile, K or V
  static constexpr int KB = Pair ? 64 : 8192 / DP;   // keys of a V block
  static constexpr int Q = NQ * 128 * DP * 2;
  static constexpr int NB = I8 ? (DP == 64 ? 10 : 9) : DP == 64 ? 12 : 10;   // ring blocks
  static constexpr int TPR = 4 / NQ;                 // threads of a row in the softmax
  static constexpr int W = 128 / TPR;                // keys of a tile that one of them takes
  static constexpr int Mma = 16, LoadK = 17, LoadV = 18;   // warps: softmax before, MMA issuer, TMA
  static constexpr int Threads = 20 * 32;            // one warp idle: registers come in fours of warps

  static constexpr int Scales = I8 ? 8 * 1024 + 1024 + 2048 : 0;   // K's and V's of 8 tiles; the rows' powers of two; a word a softmax thread
  static constexpr int Smem = Q + NB * kBlock + 512 + 2048 + Scales;
  static_assert(Smem <= 232448, "shared memory");
  static constexpr uint32_t O0 = 256;                // first TMEM column of O; S buffers at 0 and 128
};

struct ChunkCtl {
  uint64_t full[12], empty[12];   // ring
  uint64_t s_full[2], p_full[2];  // score buffers: scores ready, weights ready
  uint64_t o_full[2];             // the last product of a row tile is in O
  uint64_t pv;                    // one row tile: each product into O (before a rescale)
  uint64_t tail;                  // V rows past the last key are zeroed
  uint64_t drain;
  uint64_t q_full;                // the queries are in shared memory (a pair: both blocks')
  uint64_t q_here, tail_here;     // a pair: this block's queries; its copy of the V block with the last key
  uint64_t scales[8];             // 8-bit cache: the scales of tile j (mod 8) are there
  uint32_t tmem_base;
  int abort;
  int page[2][2][8];              // of the key tiles being loaded: K, V; this one's and the next's
};
static_assert(sizeof(ChunkCtl) <= 512, "control block");

__device__ __forceinline__ void chunk_fail(ChunkCtl* c) {
  *reinterpret_cast<volatile int*>(&c->abort) = 1;
  atomicMax(&g_attention_status, VQ2_ERR_TIMEOUT);
}
template <bool CLUSTER = false>   // CLUSTER: arrivals come from the pair's other block too
__device__ __forceinline__ bool chunk_wait(uint32_t bar, uint32_t parity, ChunkCtl* c) {
  auto ready = [&] { return CLUSTER ? mbar_try_cluster(bar, parity) : mbar_try(bar, parity); };
  if (ready()) return true;
  const long long t0 = clock64();
  while (!ready()) {
    if (*reinterpret_cast<volatile int*>(&c->abort)) return false;
    if (clock64() - t0 > kWaitCycles) {
      chunk_fail(c);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void chunk_drain(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try(bar, parity))
    if (clock64() - t0 > kWaitCycles) {
      atomicMax(&g_attention_status, VQ2_ERR_TIMEOUT);
      return;
    }
}

// Descriptor of a V block: values contiguous (64 in a 128-byte swizzled row, the next 64 KB keys * 128
// bytes on: the leading byte offset), keys 128 bytes apart, 8-key groups 1024 (stride byte offset).
template <int KB>
__device__ __forceinline__ uint64_t v_desc(uint32_t saddr) {
  return static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(KB * 128 >> 4) << 16) |
         (static_cast<uint64_t>(1024 >> 4) << 32) | (static_cast<uint64_t>(1) << 46) | (static_cast<uint64_t>(2) << 61);
}

template <bool PAIR>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  if (PAIR) tma_load_3d_pair(dst, map, x, y, z, bar);
  else tma_load_3d(dst, map, x, y, z, bar);
}

// 64-value groups that one copy brings: `groups` where the head size is made of whole groups and the
// copy has all keys of the block (the groups then stand in shared memory as the block wants them).
__host__ __device__ constexpr int copy_groups(int D, bool all_keys, int groups) {
  return D % 64 == 0 && all_keys ? groups : 1;
}

template <bool PAIR>
__device__ __forceinline__ void umma(uint32_t d, uint64_t ad, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if (PAIR) umma2_f16(d, ad, bd, idesc, accumulate);
  else umma_f16(d, ad, bd, idesc, accumulate);
}
template <bool PAIR>
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t at, uint64_t bd, uint32_t idesc, uint32_t accumulate) {
  if (PAIR) umma2_f16_ts(d, at, bd, idesc, accumulate);
  else umma_f16_ts(d, at, bd, idesc, accumulate);
}
template <bool PAIR>   // of a pair: on the barrier in both blocks
__device__ __forceinline__ void commit(uint32_t bar) {
  if (PAIR) umma2_commit(bar);
  else umma_commit(bar);
}

// Barrier `id` of n threads (whole warps): whether any of them says p.
__device__ __forceinline__ bool any_of(int id, int n, bool p) {
  int r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %3, 0;\n\t"
      "barrier.cta.red.or.pred q, %1, %2, p;\n\t"
      "selp.b32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(n), "r"(static_cast<int>(p))
      : "memory");
  return r != 0;
}

// Two sums or products at once.
__device__ __forceinline__ uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 unpair(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 32 columns of this thread's lane, not yet waited for; tmem_wait passes the registers through the
// wait so that no use of them can be moved ahead of it.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_wait_ld(float* v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15])
               :
               : "memory");
  asm volatile("" : "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]), "+f"(v[23]),
                    "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]), "+f"(v[30]), "+f"(v[31])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
        "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
        "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

constexpr int kSorted = 32;   // sequences, at most, that blocks are ordered by

// Which split this block is: over an 8-bit cache read again where it is needed rather than kept in a
// register that spills (two int8 chunks 155 us kept, 147 so).
__device__ __forceinline__ int this_split(const AttnArgs& a) {
  uint32_t z;
  asm volatile("mov.u32 %0, %%ctaid.z;" : "=r"(z));
  return (int)(a.kv.seqs <= kSorted ? z / (uint32_t)a.kv.seqs : z);
}

// The sequence (of 32 at most) that stands at place n when they are ordered by length, longest first (warp-wide).
__device__ __forceinline__ int nth_longest(const PagedKV& kv, int n, int lane) {
  if (kv.seqs == 1) return 0;
  const int len = lane < kv.seqs ? length_of(kv, lane) : -1;
  int place = 0;
  for (int i = 0; i < kv.seqs; ++i) {
    const int l = __shfl_sync(0xffffffffu, len, i);
    place += l > len || (l == len && i < lane);
  }
  return __ffs(__ballot_sync(0xffffffffu, lane < kv.seqs && place == n)) - 1;
}

// T: of queries and output. The products run in T, over an 8-bit cache in fp16.
template <int DP, typename T, bool I8>
__global__ void __launch_bounds__(ChunkShape<DP, I8>::Threads, 1)
    attn_chunk_kernel(const AttnArgs a, const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap) {
  using S = ChunkShape<DP, I8>;
  using M = typename std::conditional<I8, __half, T>::type;
  constexpr int NQ = S::NQ, B = S::B, KB = S::KB, NB = S::NB;
  constexpr bool PAIR = S::Pair;
  constexpr bool BF = std::is_same<M, __nv_bfloat16>::value;
  // fp16 weights: 2^7 larger than in bf16, up to 2^15, so that those down to 2^-32 of the largest (2^-25 otherwise)
  // are more than 0: over 200,000 keys together they can outweigh a rounding. Taken back where splits are joined.
  constexpr float kLift = BF ? 0.f : 7.f, kDrop = BF ? 1.f : 1.f / 128.f;
  extern __shared__ __align__(1024) unsigned char sm[];
  unsigned char* ring = sm + S::Q;
  ChunkCtl* ctl = reinterpret_cast<ChunkCtl*>(ring + NB * kBlock);
  float* part_s = reinterpret_cast<float*>(ring + NB * kBlock + 512);   // a word of each softmax thread
  float* scale_s = part_s + 512;      // 8-bit: [8 tiles][K 128, V 128], then what undoes each row's power of two
  float* undo_s = scale_s + 8 * 256;
  float* vmax_s = undo_s + 256;
  pdl_wait();
  pdl_trigger();
  if (su32(sm) & 1023) {   // the swizzle needs it; the only shared memory here, so it starts a 1024-byte line
    if (threadIdx.x == 0) atomicMax(&g_attention_status, VQ2_ERR_ALIGN);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kMma = S::Mma, TPR = S::TPR, W = S::W;
  // Longest first, so that the last round of blocks is short: whole splits before what is left over, the
  // longest sequence first, of its rows the last, which see the most keys (208 blocks of three sequences
  // of 5659 to 8191 keys: 241 us in the sequences' order, 224 so).
  const int rank = PAIR ? blockIdx.x & 1 : 0;   // of a pair: which row tile, which half of K's keys and V's values
  const int bx = PAIR ? blockIdx.x >> 1 : blockIdx.x;
  const bool sorted = a.kv.seqs <= kSorted;
  const int nth = sorted ? blockIdx.z % a.kv.seqs : bx / a.row_blocks, split = sorted ? blockIdx.z / a.kv.seqs : blockIdx.z;
  const int rb = a.row_blocks - 1 - (sorted ? bx : bx - nth * a.row_blocks), h = blockIdx.y;
  const int b = sorted ? nth_longest(a.kv, nth, lane) : nth;
  const AttnRows w = attn_rows(a, b, rb);
  if (!I8)   // the widening kernel's work there: registers are short here (two int8 chunks 160 us for 163)
    blank_strays(a, w, b, (((int64_t)rb * a.kv.heads + h) * a.splits + split) * (PAIR ? 2 : 1) + rank,
                 (int64_t)a.row_blocks * a.kv.heads * a.splits * (PAIR ? 2 : 1));
  if (w.rows <= 0) return;
  int lo, hi;
  block_keys(a, w, lo, hi);
  if (split > 0 && (int64_t)split * a.chunk >= hi - lo) return;  // split 0 stays: it writes the rows that see nothing
  const int s0 = lo + split * a.chunk, s1 = s0 + min(a.chunk, hi - s0);   // no sum past 2^31
  const bool alone = hi - lo <= a.chunk;
  const int tiles = s1 > s0 ? (s1 - s0 + 127) >> 7 : 0;
  const int nq = NQ == 2 && w.rows > 128 ? 2 : 1;  // row tiles in use

  if (threadIdx.x == 0) {
    for (int i = 0; i < NB; ++i) {
      mbar_init(su32(&ctl->full[i]), 1);
      mbar_init(su32(&ctl->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(su32(&ctl->s_full[i]), 1);
      mbar_init(su32(&ctl->p_full[i]), 4 * TPR * (PAIR ? 2 : 1));
      mbar_init(su32(&ctl->o_full[i]), 1);
    }
    mbar_init(su32(&ctl->pv), 1);
    mbar_init(su32(&ctl->tail), PAIR ? 2 : 1);
    mbar_init(su32(&ctl->tail_here), 1);
    mbar_init(su32(&ctl->q_here), 4 * TPR);
    mbar_init(su32(&ctl->drain), 1);
    mbar_init(su32(&ctl->q_full), 4 * TPR * (PAIR ? 2 : nq));
    for (int i = 0; i < 8; ++i) mbar_init(su32(&ctl->scales[i]), 1);
    ctl->abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kMma) {
    if (PAIR) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&ctl->tmem_base)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(su32(&ctl->tmem_base)) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  if (PAIR) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  // A pair's MMAs are issued by its first block, which the other's copies, queries and weights report to.
  auto lead = [&](uint64_t* bar) { return PAIR ? in_block(su32(bar), 0) : su32(bar); };
  auto arrive = [&](uint64_t* bar) {
    if (PAIR) mbar_arrive_cluster(in_block(su32(bar), 0));
    else mbar_arrive(su32(bar));
  };
  const uint32_t tmem = ctl->tmem_base;
  const int gran = I8 ? KB : min(1 << a.kv.page_log2, KB);   // keys of one V copy
  const int tail = !I8 && (s1 & (gran - 1)) ? s1 : -1;    // rows from here on, up to the copy's end, hold anything

  const int32_t* table = a.kv.table + b * a.kv.table_stride;
  const int page_mask = (1 << a.kv.page_log2) - 1;
  const int seen = row_lo(a, w, w.r0 / a.G);   // pages that end before the first key seen may be gone

  if (warp == S::LoadK || warp == S::LoadV) {
    // ---------------------------------------------------------------------------- loads
    // One elected thread each for K and V, for the reason given at the MMA issuer: copies issued by several
    // lanes are serialised through the uniform registers one by one, and the MMAs waited for them. Small
    // pages are many copies (16 keys: 32 a step), so K's and V's are issued side by side.
    const int pool_rows = (a.kv.pages * a.kv.heads) << a.kv.page_log2;
    const int wide_row0 = I8 ? (b * a.kv.heads + h) * a.wide_len : 0;
    constexpr int KK = PAIR ? 64 : 128, KS = PAIR ? 2 : 1;   // keys and 64-value groups of a K block
    const int rk = I8 ? KK : min(1 << a.kv.page_log2, KK);   // keys of one K copy
    // 64-value groups of one copy: all of the block's where its keys are one copy too
    const int kg = copy_groups(a.D, rk == KK, KS), vg = copy_groups(a.D, gran == KB, B);
    int said = 0, issued = 0;   // tiles whose scales, ring blocks whose copies were started
    bool ok = true;
    const bool loads_v = warp == S::LoadV;
    // first ring block of K or V of key tile j: K0 V0 K1 V1 .. with two row tiles, K0 K1 V0 K2 V1 .. with one
    auto block_of = [&](bool v, int j) {
      if (NQ == 2) return (2 * j + (v ? 1 : 0)) * B;
      return v ? (j == tiles - 1 ? 2 * j + 1 : 2 * j + 2) * B : (j == 0 ? 0 : 2 * j - 1) * B;
    };
    if (tiles > 0 && elect_one()) {
      // The pages of a key tile (128 / page size, at least one) are looked up a tile ahead: a lookup right
      // before its copies would cost an L2 round trip each time.
      const int shift = a.kv.page_log2, count = max(1, 128 >> shift), first_page = seen >> shift, last_page = (s1 - 1) >> shift;
      auto look = [&](int j, int i) {
        const int p = ((s0 + 128 * j) >> shift) + i;
        return i < count && p >= first_page && p <= last_page ? table[p] : -1;
      };
      const uint32_t full0 = PAIR ? in_block(su32(&ctl->full[0]), 0) : su32(&ctl->full[0]), empty0 = su32(&ctl->empty[0]);
      const int part0 = a.D % 64 == 0 ? 0 : 64, part1 = a.D % 64 == 0;   // where a 64-value group stands in the map
      int (*pages)[8] = ctl->page[loads_v ? 1 : 0];   // of this key tile and the next
      // K or V of key tile j
      auto load = [&](auto is_v, int j) {
        constexpr bool V = decltype(is_v)::value;
        constexpr int keys = V ? KB : KK, groups = V ? B : KS;
        const int k0 = s0 + 128 * j, step = V ? gran : rk, per = V ? vg : kg;
        int slot = block_of(V, j) % NB, parity = block_of(V, j) / NB & 1 ^ 1;
        int next[8];
        if (!I8 && j + 1 < tiles) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < count) next[i] = look(j + 1, i);
        }
        if (I8 && !V) {   // the tile's scales, with K; their place is free long before the ring's is
          const uint32_t bar = su32(&ctl->scales[j & 7]), dst = su32(scale_s + (j & 7) * 256);
          mbar_arrive_tx(bar, 1024);
          bulk_load(dst, a.wide_ks + wide_row0 + k0, 512, bar);
          bulk_load(dst + 512, a.wide_vs + wide_row0 + k0, 512, bar);
          said = j + 1;
        }
#pragma unroll
        for (int c = 0; c < B; ++c) {
          if (!chunk_wait(empty0 + 8 * slot, parity, ctl)) return false;
          const uint32_t dst = su32(ring) + slot * kBlock;
          const int kb = c * KB;   // of the tile
          const bool last = V && tail > k0 + kb && tail < k0 + kb + KB;   // the block that holds the last key and what follows it
          const uint32_t bar = PAIR && last ? su32(&ctl->tail_here) : full0 + 8 * slot;
          if (!PAIR || last) mbar_arrive_tx(bar, kBlock);
          if (PAIR && rank == 0) {
            if (last) mbar_arrive(su32(&ctl->full[slot]));
            else mbar_arrive_tx(su32(&ctl->full[slot]), 2 * kBlock);   // both blocks' copies
          }
          const int key0 = V ? kb : KK * rank, g0 = V ? B * rank : KS * c;
#pragma unroll 1
          for (int i = 0; i < keys; i += step) {
            const int k = k0 + key0 + i;
            int row = wide_row0 + k;
            if (!I8) {   // past the pool (zeros) where there is no key, or no page
              const int page = pages[j & 1][(key0 + i) >> shift];
              row = k >= s1 || page < 0 || page >= a.kv.pages ? pool_rows : ((page * a.kv.heads + h) << shift) + (k & page_mask);
            }
#pragma unroll 1
            for (int g = 0; g < groups; g += per)
              load_3d<PAIR>(dst + g * keys * 128 + i * 128, V ? &vmap : &kmap, part0 * (g0 + g), row, part1 * (g0 + g), bar);
          }
          issued = block_of(V, j) + c + 1;
          if (++slot == NB) {
            slot = 0;
            parity ^= 1;
          }
        }
        if (!I8 && j + 1 < tiles) {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (i < count) pages[(j + 1) & 1][i] = next[i];
        }
        return true;
      };
      if (!I8)
        for (int i = 0; i < count; ++i) pages[0][i] = look(0, i);
      if (loads_v)
        for (int j = 0; j < tiles && ok; ++j) ok = load(std::true_type(), j);
      else
        for (int j = 0; j < tiles && ok; ++j) ok = load(std::false_type(), j);
    }
    __syncwarp();
    ok = __all_sync(0xffffffffu, ok);
    issued = __reduce_max_sync(0xffffffffu, issued);
    said = __reduce_max_sync(0xffffffffu, said);
    if (ok && loads_v && tail >= 0 && tiles > 0) {   // the whole warp zeroes what follows the last key in its copy
      const int kl = s0 + 128 * (tiles - 1), c = (tail - kl) / KB, at = (2 * tiles - 1) * B + c, kb = kl + c * KB;
      ok = __all_sync(0xffffffffu, chunk_wait(su32(PAIR ? &ctl->tail_here : &ctl->full[at % NB]), PAIR ? 0 : (at / NB) & 1, ctl));
      if (ok) {
        const int from = tail - kb, to = (from + gran - 1) / gran * gran;
        for (int e = lane; e < (to - from) * B * 8; e += 32) {
          const int rr = from + e / (B * 8), p = e % (B * 8);
          *reinterpret_cast<uint4*>(ring + at % NB * kBlock + (p >> 3) * KB * 128 + rr * 128 + ((p & 7) << 4)) =
              make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) arrive(&ctl->tail);
      }
    }
    // copies this warp started have landed before the block's shared memory goes away
    if (!ok) {
      if (PAIR) {   // the other block's copies, and this one's that nobody here can wait for: 100 us is ample
        const long long t0 = clock64();
        while (clock64() - t0 < 200000) {}
      }
      for (int i = max(0, issued - NB); !PAIR && i < issued; ++i) {
        const int j = i / B;
        if (NQ == 2 && (j & 1) == (loads_v ? 1 : 0)) chunk_drain(su32(&ctl->full[i % NB]), (i / NB) & 1);
      }
      if (I8)   // scales: at most 8 tiles' are under way; those waited for already answer at once
        for (int i = max(0, said - 8); i < said; ++i) chunk_drain(su32(&ctl->scales[i & 7]), (i >> 3) & 1);
    }
  } else if (warp == kMma) {
    // ---------------------------------------------------------------------------- MMA issuer
    // One elected thread. elect.sync rather than a lane number: the compiler then knows a single thread
    // runs and keeps descriptors in uniform registers; behind `lane == 0` each MMA was issued in about
    // 140 cycles, twice what it takes to execute.
    if (rank == 0 && elect_one()) {
      constexpr uint32_t QK = umma_idesc<128, BF>(false, PAIR ? 256 : 128), PV = umma_idesc<DP, BF>(true, PAIR ? 256 : 128);
      const uint64_t qd = sw128_desc(su32(sm)), kd = sw128_desc(su32(ring)), vd = v_desc<KB>(su32(ring));
      const uint32_t full0 = su32(&ctl->full[0]), empty0 = su32(&ctl->empty[0]);
      bool ok = tiles == 0 || chunk_wait<PAIR>(su32(&ctl->q_full), 0, ctl);
      int ks = 0, vs = 0, kp = 0, vp = 0;   // slot and parity of the next K and V tile's first block
      auto skip = [&](int& slot, int& parity, int n) {
        slot += n;
        if (slot >= NB) {
          slot -= NB;
          parity ^= 1;
        }
      };
      // scores of row tile i with the next key tile into buffer s
      auto qk = [&](int i, int s) {
        int slot = ks, parity = kp;
#pragma unroll
        for (int c = 0; c < B; ++c) {
          if (i == 0) {
            if (!chunk_wait<PAIR>(full0 + 8 * slot, parity, ctl)) return false;
            tc_fence_after();
          }
          constexpr int KS = PAIR ? 2 : 1;   // 64-value groups of the block
#pragma unroll
          for (int g = 0; g < KS; ++g) {
            const uint64_t ad = qd + (i * S::QC + KS * c + g) * (kBlock >> 4);
            const uint64_t bd = kd + slot * (kBlock >> 4) + g * (kBlock / KS >> 4);
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              umma<PAIR>(tmem + 128 * s, ad + 2 * kk, bd + 2 * kk, QK, (c | g | kk) != 0);
          }
          if (i == nq - 1) commit<PAIR>(empty0 + 8 * slot);
          skip(slot, parity, 1);
        }
        commit<PAIR>(su32(&ctl->s_full[s]));
        return true;
      };
      // O of row tile i += weights in buffer s times V tile j
      auto pv = [&](int i, int j, int s) {
        int slot = vs, parity = vp;
#pragma unroll
        for (int c = 0; c < B; ++c) {
          if (i == 0) {
            const int kb = s0 + 128 * j + c * KB;
            if (!chunk_wait<PAIR>(full0 + 8 * slot, parity, ctl)) return false;
            if (!I8 && tail > kb && tail < kb + KB && !chunk_wait<PAIR>(su32(&ctl->tail), 0, ctl)) return false;
            tc_fence_after();
          }
          const uint64_t bd = vd + slot * (kBlock >> 4);
#pragma unroll
          for (int kk = 0; kk < KB / 16; ++kk) {
            const int key = c * KB + 16 * kk;   // of the tile: its weights stand in the columns of its part's scores
            umma_ts<PAIR>(tmem + S::O0 + i * DP, tmem + 128 * s + key / S::W * S::W + key % S::W / 2, bd + 128 * kk, PV,
                          (c | kk) != 0 || j > 0);
          }
          if (i == nq - 1) commit<PAIR>(empty0 + 8 * slot);
          skip(slot, parity, 1);
        }
        if (NQ == 1) commit<PAIR>(su32(&ctl->pv));
        if (j == tiles - 1) commit<PAIR>(su32(&ctl->o_full[i]));
        return true;
      };
      // ring order K0 V0 K1 V1 .. with two row tiles, K0 K1 V0 K2 V1 .. with one
      if (NQ == 2) {
        if (tiles > 0)
          for (int i = 0; i < nq && ok; ++i) ok = qk(i, i);
        skip(vs, vp, B);
        skip(ks, kp, 2 * B);
        for (int j = 0; j < tiles && ok; ++j) {
          for (int i = 0; i < nq && ok; ++i) {
            ok = chunk_wait(su32(&ctl->p_full[i]), j & 1, ctl);
            if (!ok) break;
            tc_fence_after();
            ok = pv(i, j, i) && (j + 1 == tiles || qk(i, i));
          }
          skip(vs, vp, 2 * B);
          skip(ks, kp, 2 * B);
        }
      } else {
        if (tiles > 0 && ok) ok = qk(0, 0);
        skip(ks, kp, B);
        skip(vs, vp, tiles > 1 ? 2 * B : B);
        for (int j = 0; j < tiles && ok; ++j) {
          if (j + 1 < tiles) ok = qk(0, (j + 1) & 1);
          skip(ks, kp, 2 * B);
          ok = ok && chunk_wait<PAIR>(su32(&ctl->p_full[j & 1]), (j >> 1) & 1, ctl);
          if (!ok) break;
          tc_fence_after();
          ok = pv(0, j, j & 1);
          skip(vs, vp, j + 2 == tiles ? B : 2 * B);   // the last V follows the one before it
        }
      }
      // every MMA issued has completed before TMEM is freed
      if (PAIR) umma2_commit_here(su32(&ctl->drain));
      else umma_commit(su32(&ctl->drain));
      chunk_drain(su32(&ctl->drain), 0);
    }
    __syncwarp();
  } else if (warp / (4 * TPR) < nq) {
    // ---------------------------------------------------------------------------- softmax
    const int i = warp / (4 * TPR), part = (warp >> 2) % TPR, quarter = warp & 3;
    const int tile = PAIR ? rank : i;              // row tile of the rows
    const int r = 128 * tile + 32 * quarter + lane;   // row
    const bool mine = r < w.rows;
    // Row rr of the block is new token t0 + (g0 + rr) / G, head (g0 + rr) % G: small numbers, divided by
    // a multiplication.
    const int t0 = w.r0 / a.G, g0 = w.r0 - t0 * a.G;
    const uint32_t by_g = 0xffffffffu / a.G + 1;
    auto token_of = [&](int rr, int& head) {
      const int n = g0 + rr, q = a.G == 1 ? n : (int)__umulhi(n, by_g);
      head = n - q * a.G;
      return t0 + q;
    };
    // ---- the tile's queries into 128-byte swizzled blocks of 64 values; rows past the last are zeros.
    // The loads of a round go out together.
    if (tiles > 0) {
      constexpr int kThreads = 128 * TPR, N = 128 * (DP / 8) / kThreads, R = N < 8 ? N : 8;
      const int tid = (warp - 4 * TPR * i) * 32 + lane;
#pragma unroll 1
      for (int n0 = 0; n0 < N; n0 += R) {
        uint4 x[R];
#pragma unroll
        for (int n = 0; n < R; ++n) {
          const int e = tid + (n0 + n) * kThreads, rr = e / (DP / 8), v = e % (DP / 8);  // row of the tile, 8-value piece
          x[n] = make_uint4(0, 0, 0, 0);
          if (128 * tile + rr < w.rows && 8 * v < a.D) {
            int head;
            const int t = token_of(128 * tile + rr, head);
            x[n] = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (int64_t)(w.first + t) * a.q_ts +
                                                   (int64_t)(h * a.G + head) * a.q_hs + 8 * v);
          }
        }
#pragma unroll
        for (int n = 0; n < R; ++n) {
          const int e = tid + (n0 + n) * kThreads, rr = e / (DP / 8), v = e % (DP / 8);
          if (a.scale_log2 < 0.f)
            x[n] = make_uint4(x[n].x ^ 0x80008000u, x[n].y ^ 0x80008000u, x[n].z ^ 0x80008000u, x[n].w ^ 0x80008000u);
          if (I8) {   // fp16, from bf16 by a power of two that brings the row's largest value to 2^13 .. 2^14
            float back = 1.f;
            if (a.q_bf16) {
              float f[8], big = 0.f;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float2 y = unpack2<__nv_bfloat16>((&x[n].x)[j]);
                f[2 * j] = y.x;
                f[2 * j + 1] = y.y;
                big = fmaxf(big, fmaxf(fabsf(y.x), fabsf(y.y)));
              }
#pragma unroll
              for (int o = 1; o < DP / 8; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
              const int up = fp16_lift(big);
              const float by = __int_as_float((127 + up) << 23);
              back = __int_as_float((127 - up) << 23);
#pragma unroll
              for (int j = 0; j < 4; ++j) (&x[n].x)[j] = pack2<__half>(f[2 * j] * by, f[2 * j + 1] * by);
            }
            if (v == 0) undo_s[128 * i + rr] = back;
          }
          *reinterpret_cast<uint4*>(sm + (i * S::QC + (v >> 3)) * kBlock + rr * 128 + (((v & 7) ^ (rr & 7)) << 4)) = x[n];
        }
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        if (PAIR) mbar_arrive(su32(&ctl->q_here));
        arrive(&ctl->q_full);
      }
    }
    int head = 0;
    const int tok = token_of(mine ? r : 0, head);
    const uint32_t lanes = static_cast<uint32_t>(32 * quarter) << 16;
    const uint32_t o_col = tmem + lanes + S::O0 + i * DP;
    const int bar = 1 + 4 * i + quarter;           // of the warps that share these rows
    const int klo = mine ? row_lo(a, w, tok) : 0, khi = mine ? min(row_hi(a, w, tok), s1) : s1;
    const int all_lo = __reduce_max_sync(0xffffffffu, klo), all_hi = __reduce_min_sync(0xffffffffu, khi);
    bool ok = true, leave = false;   // a wait that gives up; all threads of the rows know of one
    float scale = fabsf(a.scale_log2);
    if (I8 && tiles > 0) {
      ok = chunk_wait(su32(PAIR ? &ctl->q_here : &ctl->q_full), 0, ctl);
      scale *= undo_s[128 * i + 32 * quarter + lane];
    }
    // Masked scores are -inf before they are scaled, and -inf * 0 is not -inf: a scale of 0 (or one that has
    // underflowed) becomes the smallest number, which takes every finite score to less than 5e-7.
    scale = fmaxf(scale, __int_as_float(1));
    // what the threads of this row leave for one another
    float* said = part_s + (warp - 4 * part) * 32 + lane;   // part p: said[128 * p]
    float m = -INFINITY, l = 0.f, vref = 0.f, vinv = 0.f;   // vref: a power of two above the V scales that the row has seen
    auto page_at = [&](int k) { return lane < W / 16 && k + 16 * lane < s1 ? table[(k + 16 * lane) >> a.kv.page_log2] : 0; };
    int page = page_at(s0 + W * part);   // a tile ahead
    for (int j = 0; j < tiles && !leave; ++j) {
      const int k0 = s0 + 128 * j + W * part, buf = NQ == 2 ? i : j & 1;   // this thread's first key
      // 16-key groups whose page does not exist (past the keys khi masks)
      const uint32_t missing = __ballot_sync(0xffffffffu, page < 0 || page >= a.kv.pages);
      page = page_at(k0 + 128);
      float vmax = 0.f;
      const float *ks = nullptr, *vs = nullptr;
      if (I8) {
        ok = ok && chunk_wait(su32(&ctl->scales[j & 7]), (j >> 3) & 1, ctl);
        ks = scale_s + (j & 7) * 256 + W * part;
        vs = ks + 128;
        // the largest of the tile's keys that the row sees (a hidden one's scale must not cost the row bits), where
        // some are hidden of this thread's part of them; a NaN or an infinity (a value that was stored as such) sets
        // no reference
        const float* tile_vs = scale_s + (j & 7) * 256 + 128;
        const int tile0 = s0 + 128 * j;
        uint32_t x = 0;
        if (tile0 >= all_lo && tile0 + 128 <= all_hi) {
          const float4 f = *reinterpret_cast<const float4*>(tile_vs + 4 * lane);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t y = __float_as_uint((&f.x)[e]);
            if (y < 0x7f800000u) x = max(x, y);
          }
          x = __reduce_max_sync(0xffffffffu, x);
        } else {
#pragma unroll 4
          for (int k = 0; k < W; k += 4) {
            const float4 f = *reinterpret_cast<const float4*>(vs + k);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t y = __float_as_uint((&f.x)[e]);
              if (y < 0x7f800000u && k0 + k + e >= klo && k0 + k + e < khi) x = max(x, y);
            }
          }
        }
        vmax = __uint_as_float(x);
      }
      ok = __all_sync(0xffffffffu, ok && chunk_wait(su32(&ctl->s_full[buf]), (NQ == 2 ? j : j >> 1) & 1, ctl));
      tc_fence_after();
      const uint32_t own = tmem + lanes + 128 * buf + W * part;
      const bool masked = k0 < all_lo || k0 + W > all_hi || missing;
      // The scores are read twice, 32 at a time, rather than held: 64 of them do not fit beside the
      // weights in 96 registers (three chunks to 611 tokens over 8191: 247 us so, 591 spilled; weighed
      // before the maximum is agreed on, and again where it moves: 474 us).
      auto scores = [&](int c, float* s) {
        tmem_ld32(own + c, s);
        tmem_wait_ld(s);
        if (I8) {
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(ks + c + k);
            const float2 x = unpair(mul2(pair(s[k], s[k + 1]), f.x)), y = unpair(mul2(pair(s[k + 2], s[k + 3]), f.y));
            s[k] = x.x;
            s[k + 1] = x.y;
            s[k + 2] = y.x;
            s[k + 3] = y.y;
          }
        }
        if (masked) {
#pragma unroll
          for (int k = 0; k < 32; ++k)
            if (k0 + c + k < klo || k0 + c + k >= khi || ((missing >> ((c + k) >> 4)) & 1)) s[k] = -INFINITY;
        }
      };
      float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < W; c += 32) {
        float s[32];
        scores(c, s);
#pragma unroll
        for (int k = 0; k < 32; k += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], fmaxf(s[k + e], s[k + e + 4]));
      }
      const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale;
      // One that gave up waiting says so here, so that all leave together.
      if (any_of(bar, 32 * TPR, mx > m + (8.f + kLift) || vmax > vref || !ok)) {
        said[128 * part] = mx;
        float* said_v = vmax_s + (said - part_s);
        if (I8) said_v[128 * part] = vmax;
        leave = any_of(bar, 32 * TPR, !ok);
        if (leave) break;
        float all = mx;
#pragma unroll
        for (int q = 0; q < TPR; ++q) {
          all = fmaxf(all, said[128 * q]);
          if (I8) vmax = fmaxf(vmax, said_v[128 * q]);
        }
        const float mn = fmaxf(m, all - kLift), by = mn == -INFINITY ? 1.f : ex2(m - mn);
        float undo = 1.f;
        if (I8 && vmax > vref) {
          const float ref = above(vmax);
          undo = vref / ref;
          vref = ref;
          vinv = 1.f / ref;
        }
        m = mn;
        l *= by;
        if (j > 0) {
          // scores of tile j follow the product of tile j - 1 (two row tiles) or j - 2 (one)
          if (NQ == 1) {
            ok = __all_sync(0xffffffffu, chunk_wait(su32(&ctl->pv), (j - 1) & 1, ctl));
            tc_fence_after();
          }
#pragma unroll 1
          for (int c = part * (DP / TPR); c < (part + 1) * (DP / TPR); c += 32) {
            float o[32];
            tmem_ld32(o_col + c, o);
            tmem_wait_ld(o);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] *= by * undo;
            tmem_st32(o_col + c, reinterpret_cast<const uint32_t*>(o));
          }
        }
        any_of(bar, 32 * TPR, false);   // `said` has been read by all
      }
      const float base = m == -INFINITY ? 0.f : m;
      const uint64_t scale2 = pair(scale, scale), base2 = pair(-base, -base);
      const uint64_t vinv2 = pair(vinv, vinv);
      // The tile's sum by itself: beside a running sum of 1, weights of 2^-25 would vanish one by one.
      uint64_t l2 = pair(0.f, 0.f);
      auto weigh = [&](auto hides, int c) {   // hides: some keys of the tile are masked
        float s[32];
        uint32_t p[16];
        scores(c, s);
#pragma unroll
        for (int k = 0; k < 32; k += 4) {
          const float2 x = unpair(fma2(pair(s[k], s[k + 1]), scale2, base2));
          const float2 z = unpair(fma2(pair(s[k + 2], s[k + 3]), scale2, base2));
          uint64_t y = pair(ex2(x.x), ex2(x.y)), w = pair(ex2(z.x), ex2(z.y));
          l2 = add2(l2, add2(y, w));
          if (I8) {
            const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(vs + c + k);
            y = mul2(y, mul2(f.x, vinv2));
            w = mul2(w, mul2(f.y, vinv2));
          }
          float2 u = unpair(y), v = unpair(w);
          if (I8 && decltype(hides)::value) {   // a masked key's scale may be anything, and 0 * NaN is not 0
            if (s[k] == -INFINITY) u.x = 0.f;
            if (s[k + 1] == -INFINITY) u.y = 0.f;
            if (s[k + 2] == -INFINITY) v.x = 0.f;
            if (s[k + 3] == -INFINITY) v.y = 0.f;
          }
          p[k / 2] = pack2<M>(u.x, u.y);
          p[k / 2 + 1] = pack2<M>(v.x, v.y);
        }
        tmem_st16(own + c / 2, p);   // over scores that this thread has read
      };
#pragma unroll
      for (int c = 0; c < W; c += 32) {
        if (I8 && masked) weigh(std::true_type(), c);
        else weigh(std::false_type(), c);
      }
      const float2 l01 = unpair(l2);
      l += l01.x + l01.y;
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {   // the weights are in tensor memory: nothing else to release
        if (PAIR) mbar_arrive_cluster_relaxed(in_block(su32(&ctl->p_full[buf]), 0));
        else mbar_arrive(su32(&ctl->p_full[buf]));
      }
    }
    // ---- the rows' output, or their share of it
    if (ok && !leave && tiles > 0) ok = __all_sync(0xffffffffu, chunk_wait(su32(&ctl->o_full[i]), 0, ctl));
    said[128 * part] = l;
    ok = !any_of(bar, 32 * TPR, !ok || leave);
    tc_fence_after();
    l = 0.f;
#pragma unroll
    for (int p = 0; p < TPR; ++p) l += said[128 * p];
    if (!ok) l = __int_as_float(0x7fffffff);   // gave up: the rows come out as NaN
    const float inv = l == 0.f ? 0.f : 1.f / l;
    // 16 values of 32 rows at a time through 2 KB of the tile's queries, which nobody reads any more:
    // a row's 16 values then go out as whole sectors.
    unsigned char* mine_s = sm + i * S::QC * kBlock + (warp - 4 * TPR * i) * 2048;
#pragma unroll 1
    for (int c = part * (DP / TPR); c < (part + 1) * (DP / TPR); c += 16) {
      float o[16];
      __syncwarp();
      if (tiles > 0) tmem_ld16(o_col + c, o);
      else
#pragma unroll
        for (int k = 0; k < 16; ++k) o[k] = 0.f;
      const float by = (alone ? inv : kDrop) * (I8 ? vref : 1.f);
#pragma unroll
      for (int k = 0; k < 16; ++k) o[k] *= by;
      if (alone) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          *reinterpret_cast<uint4*>(mine_s + lane * 32 + ((k ^ (lane >> 2 & 1)) << 4)) =
              make_uint4(pack2<T>(o[8 * k], o[8 * k + 1]), pack2<T>(o[8 * k + 2], o[8 * k + 3]),
                         pack2<T>(o[8 * k + 4], o[8 * k + 5]), pack2<T>(o[8 * k + 6], o[8 * k + 7]));
        __syncwarp();
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const int rl = 16 * n + (lane >> 1), k = lane & 1, rr = 128 * tile + 32 * quarter + rl;
          int hd;
          const int t = token_of(rr, hd);
          if (rr < w.rows && c + 8 * k < a.D)
            *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + ((int64_t)(w.first + t) * a.hq + h * a.G + hd) * a.D + c + 8 * k) =
                *reinterpret_cast<const uint4*>(mine_s + rl * 32 + ((k ^ (rl >> 2 & 1)) << 4));
        }
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<float4*>(mine_s + lane * 64 + ((k ^ (lane >> 1 & 3)) << 4)) =
              make_float4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        __syncwarp();
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int rl = 8 * n + (lane >> 2), k = lane & 3, rr = 128 * tile + 32 * quarter + rl;
          int hd;
          const int t = token_of(rr, hd);
          if (rr < w.rows && c + 4 * k < a.D)
            *reinterpret_cast<float4*>(
                a.part_o + (((int64_t)(w.first + t) * a.hq + h * a.G + hd) * a.splits + (I8 ? this_split(a) : split)) * a.D + c + 4 * k) =
                *reinterpret_cast<const float4*>(mine_s + rl * 64 + ((k ^ (rl >> 1 & 3)) << 4));
        }
      }
    }
    const int64_t at = (int64_t)(w.first + tok) * a.hq + h * a.G + head;
    if (mine && part == 0) {
      if (!alone) a.part_ml[at * a.splits + (I8 ? this_split(a) : split)] = make_float2(m + kLift, l * kDrop);
      else if (a.lse) a.lse[at] = l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2;
    }
  }

  tc_fence_before();
  if (PAIR) cluster_sync();   // neither block's memory goes away while the other may still reach it
  else __syncthreads();
  if (warp == kMma) {
    tc_fence_after();
    if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// A pool [rows, D] (every page's every head) as copies of `groups` x `box` rows x 64 values, 128-byte
// swizzle: three dimensions, 64 values, rows, 64-value groups (head sizes not made of whole groups: D
// values, rows, 1, a copy a group). Values past D and rows past the pool read as zeros.
bool make_pool_map(CUtensorMap* map, const void* base, int64_t rows, int D, int box, int groups, bool bf16) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  const bool whole = D % 64 == 0;
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(whole ? 64 : D), static_cast<cuuint64_t>(rows),
                              static_cast<cuuint64_t>(whole ? D / 64 : 1)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(D) * 2, static_cast<cuuint64_t>(whole ? 128 : D * 2)};
  const cuuint32_t boxes[3] = {64, static_cast<cuuint32_t>(box), static_cast<cuuint32_t>(groups)};
  const cuuint32_t es[3] = {1, 1, 1};
  return fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base), dims,
            strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kWidenKeys = 64;

// The visible keys and values of an 8-bit cache as fp16 integers [seqs, heads, wide_len, D], their scales
// [seqs, heads, wide_len] beside them; zeros past a sequence's end (to the next 128 keys) and where a
// page does not exist. 64 keys a block; bound by memory (a key of 256 values: 516 bytes read, 1032
// written).
__global__ void __launch_bounds__(256) widen_kernel(const AttnArgs a) {
  pdl_wait();
  pdl_trigger();
  const int per = a.wide_len / kWidenKeys;
  const int bh = blockIdx.x / per, k0 = (blockIdx.x - bh * per) * kWidenKeys;
  const int b = bh / a.kv.heads, h = bh - b * a.kv.heads;
  AttnArgs all = a;
  all.rows_per_block = 0x7fffffff;
  const AttnRows w = attn_rows(all, b, 0);
  blank_strays(a, w, b, blockIdx.x - b * a.kv.heads * per, a.kv.heads * per);
  if (w.rows <= 0) return;
  const int first = row_lo(a, w, 0) & a.lo_mask, end = min((w.len + 127) & ~127, a.wide_len);
  if (k0 + kWidenKeys <= first || k0 >= end) return;
  const int32_t* table = a.kv.table + b * a.kv.table_stride;
  const int page_mask = (1 << a.kv.page_log2) - 1, seen = row_lo(a, w, 0);
  __shared__ int row_s[kWidenKeys];
  if (threadIdx.x < kWidenKeys) {
    const int k = k0 + threadIdx.x;
    int row = -1;
    if (k < w.len && (k | page_mask) >= seen) {
      const int page = table[k >> a.kv.page_log2];
      if (page >= 0 && page < a.kv.pages) row = ((page * a.kv.heads + h) << a.kv.page_log2) + (k & page_mask);
    }
    row_s[threadIdx.x] = row;
    const int64_t at = (int64_t)bh * a.wide_len + k;
    a.wide_ks[at] = row < 0 ? 0.f : a.kv.k_scale[row];
    a.wide_vs[at] = row < 0 ? 0.f : a.kv.v_scale[row];
  }
  __syncthreads();
  // 256 / pieces keys a round; the loads of two rounds, K's and V's, go out together
  const int pieces = a.D >> 4, per_round = 256 / pieces, key0 = threadIdx.x / pieces, p = threadIdx.x - key0 * pieces;
  if (key0 >= per_round) return;
  const int64_t out0 = ((int64_t)bh * a.wide_len + k0) * a.D + 16 * p;
  for (int k = key0; k < kWidenKeys; k += 2 * per_round) {
    uint4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = k + (i >> 1) * per_round, row = key < kWidenKeys ? row_s[key] : -1;
      const char* src = static_cast<const char*>(i & 1 ? a.kv.v : a.kv.k);
      x[i] = make_uint4(0, 0, 0, 0);
      if (row >= 0) x[i] = *reinterpret_cast<const uint4*>(src + (int64_t)row * a.D + 16 * p);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = k + (i >> 1) * per_round;
      if (key >= kWidenKeys) continue;
      uint4 y[2];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t u = (&x[i].x)[j] ^ 0x80808080u;   // offset binary
        (&y[j >> 1].x)[2 * (j & 1)] = bytes_f16(u, 0x4140);
        (&y[j >> 1].x)[2 * (j & 1) + 1] = bytes_f16(u, 0x4342);
      }
      uint4* to = reinterpret_cast<uint4*>(static_cast<unsigned char*>(i & 1 ? a.wide_v : a.wide_k) + (out0 + (int64_t)key * a.D) * 2);
      to[0] = y[0];
      to[1] = y[1];
    }
  }
}

template <int DP, typename T, bool I8>
int launch(const AttnArgs& a, cudaStream_t st) {
  using S = ChunkShape<DP, I8>;
  auto kern = attn_chunk_kernel<DP, T, I8>;
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaGetDevice(&dev);
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(done.load() & bit)) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, S::Smem);
    if (e != cudaSuccess) {
      set_last_cuda_error(e);
      return VQ2_ERR_LAUNCH;
    }
    done.fetch_or(bit);
  }
  CUtensorMap kmap, vmap;
  constexpr int KK = S::Pair ? 64 : 128;   // keys of a K block
  const int page = I8 ? 128 : 1 << a.kv.page_log2, kbox = page < KK ? page : KK, vbox = page < S::KB ? page : S::KB;
  const int64_t rows = I8 ? (int64_t)a.kv.seqs * a.kv.heads * a.wide_len : ((int64_t)a.kv.pages * a.kv.heads) << a.kv.page_log2;
  if (!make_pool_map(&kmap, I8 ? a.wide_k : a.kv.k, rows, a.D, kbox, copy_groups(a.D, kbox == KK, S::Pair ? 2 : 1), !I8 && a.q_bf16) ||
      !make_pool_map(&vmap, I8 ? a.wide_v : a.kv.v, rows, a.D, vbox, copy_groups(a.D, vbox == S::KB, S::B), !I8 && a.q_bf16))
    return VQ2_ERR_LAUNCH;
  const bool sorted = a.kv.seqs <= kSorted;
  const dim3 grid((unsigned)(sorted ? a.row_blocks : a.kv.seqs * a.row_blocks), (unsigned)a.kv.heads,
                  (unsigned)(sorted ? a.kv.seqs * a.splits : a.splits));
  if (S::Pair)
    return launch_cluster(kern, dim3(2 * grid.x, grid.y, grid.z), dim3(S::Threads), S::Smem, 2, st, a, kmap, vmap);
  return launch_kernel(kern, grid, dim3(S::Threads), S::Smem, st, a, kmap, vmap);
}

template <typename T, bool I8>
int launch_shape(const AttnArgs& a, cudaStream_t st) {
  return a.D > 128 ? launch<256, T, I8>(a, st) : a.D > 64 ? launch<128, T, I8>(a, st) : launch<64, T, I8>(a, st);
}

}  // namespace

void plan_attn_chunk(AttnArgs& a, int64_t max_new, int64_t max_len) {
  const int64_t rows = max_new * a.G;
  a.rows_per_block = 256;   // head size above 128: of a pair of blocks
  a.row_blocks = (int)((rows + a.rows_per_block - 1) / a.rows_per_block);
  if (a.row_blocks < 1) a.row_blocks = 1;
  a.lo_mask = ~127;
  // One block an SM. Where the blocks do not fill the card, the keys are split for one round of blocks,
  // 256 keys at least: a split costs its start and, per row, its share of O written and read again
  // (9 sequences of 5 drafts over 1024 keys, 18 blocks: 128 keys 22.3 us, 256 17.0, 512 21.6, whole 34;
  // 64 tokens over 8000, 8 blocks in pairs: 256 35, 512 23.2, 1024 27.4). From a quarter of the card on
  // rows are so many that a split has to take 2048 keys to pay (2048 tokens, 64 blocks: 1024 100 us, 2048
  // 91, whole 71; two int8 chunks of 257 over 16385, 72 blocks: 4096 160, half 147, whole 235).
  int64_t keys = max_len;
  if (a.window && a.window + max_new + 128 < keys) keys = a.window + max_new + 128;
  const int64_t blocks = (int64_t)a.kv.seqs * a.kv.heads * a.row_blocks * (a.D > 128 ? 2 : 1);
  const int64_t want = blocks >= sm_count() ? 1 : sm_count() / blocks;
  int64_t chunk = (keys + 127 + want - 1) / want;
  if (chunk < (keys + 127 + 63) / 64) chunk = (keys + 127 + 63) / 64;
  const int64_t least = 4 * blocks > sm_count() ? 2048 : 256;
  if (chunk < least) chunk = least;
  chunk = (chunk + 127) & ~int64_t(127);
  a.chunk = (int)chunk;
  a.splits = (int)((keys + 127 + chunk - 1) / chunk);   // the first key is rounded down by up to 127
  if (a.splits < 1) a.splits = 1;
}

int launch_attn_chunk(const AttnArgs& a, bool i8, cudaStream_t st) {
  if (i8) {
    const int64_t blocks = (int64_t)a.kv.seqs * a.kv.heads * (a.wide_len / kWidenKeys);
    const int s = launch_kernel(widen_kernel, dim3((unsigned)blocks), dim3(256), 0, st, a);
    if (s != VQ2_OK) return s;
    return a.q_bf16 ? launch_shape<__nv_bfloat16, true>(a, st) : launch_shape<__half, true>(a, st);
  }
  return a.q_bf16 ? launch_shape<__nv_bfloat16, false>(a, st) : launch_shape<__half, false>(a, st);
}

int attn_chunk_status(int reset) {
  int32_t v = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&v, g_attention_status, sizeof(v));
  if (e == cudaSuccess && reset) {
    const int32_t z = 0;
    e = cudaMemcpyToSymbol(g_attention_status, &z, sizeof(z));
  }
  if (e != cudaSuccess) {
    set_last_cuda_error(e);
    return VQ2_ERR_LAUNCH;
  }
  return v;
}

}  // namespace vq2
