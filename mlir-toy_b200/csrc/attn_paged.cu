// Attention of the new tokens of a ragged batch over the paged KV cache (f16 / bf16, D = 128, pages of 64 rows).
//
// Token t of sequence b (cu_seqlens[b] <= t < cu_seqlens[b+1]) sits at position p = seq_lens[b] - cu_seqlens[b+1] + t and
// sees the cached rows j <= p, its own among them:  out[t, h] = sum_j softmax_j(q[t, h] . k_j * scale) v_j, query head h
// reading kv head h / (Hq / Hkv).  One pass over the rows with the running maximum and sum of the softmax in fp32.
//
// Tiles.  The `group` query heads of a kv head share its K and V, so a tile's 128 rows are floor(128 / group) tokens times
// group heads (row = token * group + head).  Tiles run over sequence, kv head, chunk of tokens; each has a number of KV
// blocks of 128 rows (two pages) that follows from the device-side lengths.  The blocks of all tiles form one line, which
// is cut into equal ranges, one per CTA: a few drafted tokens over one long cache keep every SM as busy as a long prompt
// does, and all CTAs end together, whatever the lengths.  (One exception: see kWaveBytes.)  A range that covers a whole
// tile writes its output; the (at most two) tiles that a CTA has in part leave un-normalised fp32 partials (o, m, l),
// which a second kernel joins in the order of the line, so results do not depend on timing.
//
// Inside a CTA the blocks of its ranges form one stream, numbered g = 0, 1, 2, ..., that does not stop at tile borders:
//
//   S(g) = Q K(g)^T      8 x tcgen05.mma 128x128x16, both operands in shared memory, into TMEM buffer g % 3
//   softmax(g)           warpgroup g & 1 (thread = row = TMEM lane): row maximum, p = 2^(s - m), P(g) as packed 16-bit
//                        over the first 64 columns of the same TMEM buffer
//   O += P(g) V(g)       8 x tcgen05.mma 128x128x16 with P read from TMEM
//
// (64x128x16 for a tile of at most 64 rows: no faster, but the products' power counts where the clock is at the limit.)
//
//   warps 0-3 / 4-7  softmax of even / odd blocks      warps 8-11   epilogue
//   warp 12, 15      TMA producers: Q and K (and the list of tiles); V (warp 15 also allocates the 512 TMEM columns)
//   warp 13, 14      issuers of the score products and of the PV products (one lane each)
//
// The 512 TMEM columns are four regions of 128: three score buffers and O.  Reading a finished O takes the epilogue 2 to 3
// us, and a tile of a chunk may be over in two blocks, so the next tile does not wait for it: its O takes over the region
// of the score buffer whose turn comes last, and that buffer moves to the old O's region once it has been read, two blocks
// later.
//
// What bounds it.  A block takes 0.9 us where its products need 0.53: three blocks are in flight and the chain from PV(g-3)
// over S(g) and its softmax to PV(g) is 2.6 us long.  A change of tiles costs about 2 us more.  Under sustained load the
// power limit takes the clock from 1.9 to 1.3 - 1.5 GHz and both grow with it.  Measured, 32 / 8 heads, bf16:
//   4096 tokens, nothing cached     141 us alone (975 TFLOP/s), 160 - 167 sustained; tensor pipe 48 % busy
//   2048 tokens over 30000 rows     850 us alone (1225 TFLOP/s), 955 - 982 sustained
//   32 sequences of up to 7 tokens, 40 / 8 heads, up to 16001 rows: 166 us, 1.04 GB read once at 6.3 TB/s; 171 - 182 sustained
//   32 single tokens over 8000 rows each: 174 us sustained, 1.05 GB at 6.0 TB/s
//
// P is rounded to the storage type because the second product takes both operands in one 16-bit type; the row sum adds
// the unrounded values.  The running maximum passes between the warpgroups through shared memory, O is rescaled only when
// it grows by more than 2^8.  A weight is then at most 2^8; in fp16 all are taken times 2^7 (at most 2^15, of 2^16), so that
// the least that is not 0 is 2^-32 of the maximum's, not 2^-25: a long cache has many small ones.
//
// What is masked.  A table entry that is not needed or not in the pool becomes a coordinate outside the tensor map, which
// TMA fills with zeros; nothing outside the pool is addressed.  Scores of hidden columns are replaced, not added to, so K
// may hold anything there.  V may not, since 0 * NaN is NaN: in the blocks that some row of the tile does not see
// whole, the epilogue warps (idle then) clear V rows behind the sequence's end in shared memory, and look for infinities
// and NaN in the rows that only some of the tile's rows see, before the PV product of that block.  Such a value is
// replaced by 0 and noted, and the epilogue adds it to that column of exactly those rows that see it, so that it gives
// what the product gives in the other blocks: an infinity, or NaN beside one of the other sign.
//
// Every wait is bounded; on expiry the role records a code in the status words and unwinds.
#include <cuda.h>

#include <atomic>
#include <cstddef>

#include "nb200_common.cuh"
#include "sm100_primitives.cuh"
#include "tma_host.cuh"

namespace nb200 {
namespace {

using namespace sm100;

constexpr int kPageRows = 64;
constexpr int kBM = 128;
constexpr int kBN = 128;                        // rows of a KV block: two pages
constexpr int kD = 128;
constexpr int kThreads = 512;
constexpr int kTileBytes = 128 * kD * 2;        // 32 KB: two halves of 64 columns, 16 KB each
constexpr int kBox = kTileBytes / 2;
constexpr int kPageBox = kPageRows * 128;       // one page's half: 8 KB
constexpr int kSBufs = 3;
constexpr int kTmemCols = 512;                  // four regions of 128 columns
constexpr float kRescaleThreshold = 8.0f;
template <int DT> constexpr float kLift = DT == NB200_F16 ? 7.0f : 0.0f;   // weights are held times 2^kLift, in P, in O and in l
constexpr int kSched = 16;                      // ring of tile descriptors handed from the K producer to the other roles
constexpr int kMaxCtas = 160;                   // CTAs that the workspace has room for
// Cut like that, the CTAs of a head are all over its K and V at any time, which is fine while those stay in the L2.  A
// single sequence whose K and V do not, and whose tiles are about equally long, is dealt out in waves first: every CTA
// takes the same number of whole tiles, in order, so that neighbours read the same blocks at the same time, and only what
// is left is cut.  2048 tokens over 30000 cached rows (131 MB): 0.15 GB of DRAM reads and 971 us under sustained load, 2.46 GB
// and 1117 us without.  "About equally long" (the shortest tile within an eighth of the longest) is on the safe side: a wave
// lasts as long as its longest tile.  Sustained, as it is / in waves whatever the tiles' lengths / never in waves:
//   8192 tokens over 30000 rows   5.08 / 4.39 / 4.98 ms        16384 over 8192    4.23 / 4.19 / 4.22
//   20000, nothing cached         3.16 / 3.20 / 3.15           32768, nothing     9.11 / 8.49 / 9.05
// So the bound gives something away at long caches.  Batches of more than one sequence have not been tried.
constexpr long long kWaveBytes = 1ll << 26;     // half of the L2
constexpr int kTileUnits = 2;                   // what changing tiles costs (2 us), in blocks, on the line that is cut

enum : int { kErrProducer = 41, kErrMma = 42, kErrSoftmax = 43, kErrEpilogue = 44 };

// Part of a tile that one CTA works on.
struct Segment {
  int more;                  // 0: the list ends here
  int b, kvh;
  int tok0, ntok;            // first row of the batch, tokens
  int pos0;                  // position of the first token
  int len;                   // rows of the sequence's cache
  int blk0, nblk;            // KV blocks
  int check;                 // blocks from this one on (of nblk) have V rows that not every row of the tile sees
  int slot;                  // -1: the whole tile; 0 / 1: partial that ends / begins a tile
};
// Tile that begins in a CTA and goes on in the next ones.
struct Owner {
  int parts;                 // 0: none
  int kvh, tok0, ntok;
};
struct Args {
  const int *block_table, *cu_seqlens, *seq_lens;
  uint4 *out;
  unsigned out_t, out_h;     // in 16 bytes
  int T, B, Hkv, group, tok_tile, num_pages, max_pages;
  int inv_group;             // ceil(2^16 / group): row * inv_group >> 16 is row / group for rows of a tile
  float scale_log2;
  float *part_o;             // [kMaxCtas][2][128][128]
  float2 *part_ml;           // [kMaxCtas][2][128]
  Owner *owners;             // [kMaxCtas]
  int *status;
};
constexpr size_t kPartO = static_cast<size_t>(kMaxCtas) * 2 * kBM * kD * sizeof(float);
constexpr size_t kPartMl = static_cast<size_t>(kMaxCtas) * 2 * kBM * sizeof(float2);

// New tokens of a sequence, where they sit and what there is to see.  Clamped, so that no device-side value leads out of
// the tensors: rows stay inside [0, T), positions inside [-T - 1, len].
struct Seq {
  int first, n, pos, len;
};
struct Shared {
  uint64_t q_full[2], q_empty[2], k_full[2], k_empty[2], v_full[2], v_empty[2];
  uint64_t s_full[kSBufs], p_full[kSBufs], pv_done[kSBufs];
  uint64_t o_full[4], o_free[4], m_ready[2], lm_ready[2], lm_free[2], notes_read;
  uint64_t look[2], looked[2];       // V of a block to be looked through is on its way / has been looked through, per stage
  uint64_t sched_full[kSched];
  alignas(16) unsigned long long taint[2][3][kD];   // of NaN, inf, -inf per column: (tile number + 1) << 32 | (2^31 - 1 - first KV row that is so)
  unsigned scan[kThreads / 32];
  int waves;                         // whole tiles that every CTA takes first
  unsigned base;                     // units of the tiles dealt out like that
  unsigned before, units;                  // in front of the sequence that the CTA's range begins in, and its own
  Segment seg[kSched];
  int start_b;
  Seq start_seq;                     // what that sequence brings
  int taint_any[2];                  // tile number + 1
  uint32_t tmem_base;
  int skip;
  int error[3];                      // code (0: none), detail, thread
  int k_issued;                      // K blocks asked for: whoever waits for a whole tile sees that it goes on
  float mslot[2][kBM];               // running maximum decided by block g, slot g & 1
  float2 lm[2][2][kBM];              // of tile n in [n & 1], per warpgroup: (maximum last used, partial row sum)
};
constexpr int kStage = 32 * 64;      // a warp's 32 rows of 64 bytes on their way out
constexpr int kOffStage = 6 * kTileBytes, kOffShared = kOffStage + 4 * kStage;
constexpr int kSmemBytes = kOffShared + 1024 + static_cast<int>(sizeof(Shared));
static_assert(kSmemBytes <= 232448, "shared memory of one CTA");

// Notes an expired wait; the CTA records one of its notes in the status words at its end.
__device__ __forceinline__ void report(Shared *sh, int code, int detail) {
  if (sh->error[0] == 0) sh->error[0] = code, sh->error[1] = detail, sh->error[2] = static_cast<int>(threadIdx.x);
}

// Waits for a phase with a limit on the turns: about 2 s if every turn suspends the thread for its microsecond, at least
// 0.1 s.  A role whose wait runs out leaves, and the waits of the others then run out too.  Less code than a clock and
// a flag to look at, and code is what this kernel is short of: its roles' paths at a change of tiles share the
// instruction cache (117 KB of it took 221 us at a 4096-token first chunk, 86 KB 185 us).
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity) {
#pragma unroll 1
  for (int i = 0; i < 2000000; ++i)
    if (mbar_try_wait_suspend(bar, parity, 1000u)) return true;
  return false;
}
__device__ __forceinline__ Seq seq_of(const Args &a, int b) {
  const int c0 = a.cu_seqlens[b], c1 = a.cu_seqlens[b + 1], len = a.seq_lens[b];
  Seq s;
  s.first = max(c0, 0);
  s.n = max(min(c1, a.T) - s.first, 0);
  s.len = min(max(len, 0), a.max_pages * kPageRows);
  const long long pos = static_cast<long long>(len) - c1 + s.first;
  s.pos = static_cast<int>(max(min(pos, static_cast<long long>(s.len)), -static_cast<long long>(a.T) - 1));
  return s;
}
// KV blocks of the tile that starts at token j0 of the sequence: what its last token sees, at least one.
__device__ __forceinline__ int tile_blocks(const Seq &s, int j0, int tok_tile) {
  const int sees = min(s.pos + min(s.n, j0 + tok_tile), s.len);
  return max((sees + kBN - 1) >> 7, 1);
}
// Units of a sequence's tiles for one kv head, those of tiles first, first + step, ...
__device__ __forceinline__ unsigned seq_units(const Seq &s, int tok_tile, int first, int step) {
  unsigned sum = 0;
#pragma unroll 1
  for (int j0 = first * tok_tile; j0 < s.n; j0 += step * tok_tile) sum += tile_blocks(s, j0, tok_tile) + kTileUnits;
  return sum;
}
__device__ __forceinline__ unsigned warp_scan(unsigned x, int lane) {
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned up = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += up;
  }
  return x;
}

// A tile of at most 64 rows takes products of M = 64, whose rows lie 16 to a warp's 32 lanes.  Row of the tile at a lane of
// the accumulator (128: none).
__device__ __forceinline__ bool is_small(int ntok, int group) { return ntok * group <= 64; }
__device__ __forceinline__ int token_of(const Args &a, int row) { return (row * a.inv_group) >> 16; }
__device__ __forceinline__ int row_at(int lane, bool small) { return !small ? lane : ((lane & 16) ? kBM : (lane >> 5) * 16 + (lane & 15)); }

// Which TMEM region the three score buffers (bytes 0 to 2) and O (byte 3) are in.  Tile n > 0, whose first block is g,
// takes the region of buffer (g + 2) % 3 for its O and leaves its predecessor's to that buffer.
constexpr uint32_t kRegions = 0x03020100u;
__device__ __forceinline__ uint32_t next_regions(uint32_t map, int g) {
  const int sh = 8 * ((g + 2) % kSBufs);
  const uint32_t o = map >> 24, s = (map >> sh) & 0xffu;
  return (map & ~(0xff000000u | (0xffu << sh))) | (s << 24) | (o << sh);
}
__device__ __forceinline__ uint32_t region(uint32_t map, int i) { return ((map >> (8 * i)) & 0xffu) * 128u; }   // its first column

// fma(x, 0, acc) on packed 16-bit pairs: stays 0 while every x is finite, becomes NaN for good otherwise.
template <int DT> __device__ __forceinline__ uint32_t finite_probe(uint32_t x, uint32_t acc) {
  uint32_t r;
  if constexpr (DT == NB200_BF16)
    asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(acc));
  else
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(x), "r"(0u), "r"(acc));
  return r;
}
// 0: NaN, 1: inf, 2: -inf, of a value that is not finite.
template <int DT> __device__ __forceinline__ int kind16(uint32_t h) {
  return (h & (DT == NB200_BF16 ? 0x7fu : 0x3ffu)) ? 0 : 1 + ((h >> 15) & 1);
}
template <int DT> __device__ __forceinline__ bool not_finite16(uint32_t h) {
  return DT == NB200_BF16 ? (h & 0x7f80u) == 0x7f80u : (h & 0x7c00u) == 0x7c00u;
}

template <int DT>
__global__ void __launch_bounds__(kThreads, 1)
attn_paged_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                  const __grid_constant__ CUtensorMap tm_v, const Args a) {
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char *smem = smem_raw + (base - raw);
  const uint32_t sQ = base;                                   // buffer n & 1 of tile n
  const uint32_t sK = base + 2 * kTileBytes;                  // stage g & 1
  const uint32_t sV = base + 4 * kTileBytes;
  Shared *sh = reinterpret_cast<Shared *>(smem + kOffShared);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  static_assert(sizeof(sh->taint) <= kThreads * sizeof(uint4), "one store per thread");
  if (threadIdx.x < sizeof(sh->taint) / sizeof(uint4)) reinterpret_cast<uint4 *>(sh->taint)[threadIdx.x] = make_uint4(0u, 0u, 0u, 0u);
  if (warp == 15) {
    tmem_alloc(smem_u32(&sh->tmem_base), kTmemCols);
    tmem_relinquish();
  }
  if (warp == 14 && lane == 0) {
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    sh->start_b = 0;
    sh->start_seq = Seq{0, 0, 0, 0};
    sh->before = sh->units = sh->base = 0;
    sh->waves = 0;
    sh->taint_any[0] = sh->taint_any[1] = 0;
    sh->k_issued = 0;
    sh->error[0] = 0;
  }
  if (warp == 13) {
    // one barrier per lane and turn
    uint64_t *const bars = sh->q_full;
    constexpr int kBars = (offsetof(Shared, taint) - offsetof(Shared, q_full)) / sizeof(uint64_t);
    for (int i = lane; i < kBars; i += 32) {
      uint64_t *const bar = bars + i;
      uint32_t count = 1;
      if ((bar >= sh->p_full && bar < sh->p_full + kSBufs) || (bar >= sh->o_free && bar < sh->o_free + 4) || bar == &sh->notes_read || (bar >= sh->m_ready && bar < sh->m_ready + 2) ||
          (bar >= sh->lm_free && bar < sh->lm_free + 2) || (bar >= sh->looked && bar < sh->looked + 2))
        count = 128;
      if (bar >= sh->lm_ready && bar < sh->lm_ready + 2) count = 256;
      mbar_init(smem_u32(bar), count);
    }
    fence_barrier_init();
    fence_proxy_async_smem();
  }

  // Launched as a programmatic dependent: up to here the kernel before may still run.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");   // the joining kernel waits for this grid's end itself
  if (warp == 14 && lane == 0) {
    const int code = a.status ? *reinterpret_cast<volatile int *>(a.status) : 0;
    sh->skip = status_stops(code) ? 1 : 0;
    a.owners[blockIdx.x].parts = 0;
  }

  // ---- the CTA's range of the line: the units in front of each sequence ----
  // Up to 16 sequences: a warp each, its lanes over the tiles.  More: a thread per sequence and a scan, chunk by chunk.
  const bool few = a.B <= kThreads / 32;
  unsigned total = 0, before = 0, mine = 0;
  auto scan = [&](int b0, unsigned &running) {
    const int b = b0 + static_cast<int>(threadIdx.x);
    mine = b < a.B ? seq_units(seq_of(a, b), a.tok_tile, 0, 1) * a.Hkv : 0;
    const unsigned incl = warp_scan(mine, lane);
    __syncthreads();
    if (lane == 31) sh->scan[warp] = incl;
    __syncthreads();
    before = running + incl - mine;
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += sh->scan[w];
      running += sh->scan[w];
    }
  };
  if (few) {
    const Seq seq = warp < a.B ? seq_of(a, warp) : Seq{0, 0, 0, 0};
    const unsigned sum = warp_scan(seq_units(seq, a.tok_tile, lane, 32), lane);
    if (lane == 31) sh->scan[warp] = mine = sum * a.Hkv;
    __syncthreads();
    if (a.B == 1 && warp == 0 && static_cast<long long>(a.Hkv) * seq.len * (4 * kD) > kWaveBytes) {
      const unsigned tiles = (seq.n + a.tok_tile - 1) / a.tok_tile, waves = tiles * a.Hkv / gridDim.x;
      const int shortest = tile_blocks(seq, 0, a.tok_tile), longest = tile_blocks(seq, max(seq.n - 1, 0) / a.tok_tile * a.tok_tile, a.tok_tile);
      if (waves > 0 && 8 * (longest - shortest) <= longest) {
        const unsigned dealt = waves * gridDim.x, rest = dealt % tiles;
        Seq part = seq;                                        // the last head's tiles, as far as they are dealt out
        part.n = min(static_cast<int>(rest) * a.tok_tile, seq.n);
        const unsigned of_part = warp_scan(seq_units(part, a.tok_tile, lane, 32), lane);
        if (lane == 31) {
          sh->waves = static_cast<int>(waves);
          sh->base = dealt / tiles * sum + of_part;
        }
      }
    }
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w == warp) before = total;
      total += sh->scan[w];
    }
  } else {
    for (int b0 = 0; b0 < a.B; b0 += kThreads) scan(b0, total);
  }
  // CTA c takes `share` units, and one more if c < more_until
  const unsigned base_units = sh->base, ctas = min(gridDim.x, total), share = (total - base_units) / max(ctas, 1u),
                 more_until = total - base_units - share * ctas;
  const bool idle = sh->skip || blockIdx.x >= ctas;            // the same for every thread of the CTA
  const unsigned r0 = base_units + share * blockIdx.x + min(blockIdx.x, more_until), r1 = r0 + share + (blockIdx.x < more_until ? 1 : 0);
  auto claim = [&](int b) {                                    // the thread whose sequence holds unit r0
    if (idle || before > min(r0, total - 1) || min(r0, total - 1) >= before + mine) return;
    sh->start_b = b;
    sh->start_seq = seq_of(a, b);
    sh->before = before;
    sh->units = mine;
  };
  if (few) {
    if (lane == 31) claim(warp);
  } else if (a.B <= kThreads) {
    claim(threadIdx.x);
  } else {
    unsigned running = 0;
    for (int b0 = 0; b0 < a.B; b0 += kThreads) {
      scan(b0, running);
      claim(b0 + static_cast<int>(threadIdx.x));
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh->tmem_base;
  if (idle) {
    if (warp == 15) tmem_dealloc(tmem, kTmemCols);
    return;
  }

  const uint32_t b_q_full = smem_u32(&sh->q_full[0]), b_q_empty = smem_u32(&sh->q_empty[0]),
                 b_k_full = smem_u32(&sh->k_full[0]), b_k_empty = smem_u32(&sh->k_empty[0]),
                 b_v_full = smem_u32(&sh->v_full[0]), b_v_empty = smem_u32(&sh->v_empty[0]),
                 b_s_full = smem_u32(&sh->s_full[0]), b_p_full = smem_u32(&sh->p_full[0]),
                 b_pv_done = smem_u32(&sh->pv_done[0]), b_o_full = smem_u32(&sh->o_full[0]),
                 b_o_free = smem_u32(&sh->o_free[0]), b_notes_read = smem_u32(&sh->notes_read), b_m_ready = smem_u32(&sh->m_ready[0]),
                 b_lm_ready = smem_u32(&sh->lm_ready[0]), b_lm_free = smem_u32(&sh->lm_free[0]),
                 b_look = smem_u32(&sh->look[0]), b_looked = smem_u32(&sh->looked[0]),
                 b_sched = smem_u32(&sh->sched_full[0]);  // element i at + 8 * i

  // The K producer lists the CTA's tiles in a ring that every other role reads.  The roles are never more than 10 tiles
  // apart (two Q buffers, two stages, three score buffers, O's of three tiles), so 16 slots need no "empty" barrier.
  // Null: an expired wait.
  auto segment_at = [&](int n) -> const volatile Segment * {
    if (!wait(b_sched + 8 * (n % kSched), (n / kSched) & 1)) return nullptr;
    return &sh->seg[n % kSched];
  };

  if (warp >= 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 96;");
    if (warp == 12 || warp == 15) {
      // ================================ TMA producers ================================
      // warp 12: the list of tiles, Q of every tile and the K blocks; warp 15: the V blocks.  Lane i reads the table
      // entry of page i of the next 16 blocks, lane 0 waits and issues.
      const bool is_k = warp == 12;
      const CUtensorMap *tm = is_k ? &tm_k : &tm_v;
      const uint32_t s_dst = is_k ? sK : sV, b_full = is_k ? b_k_full : b_v_full, b_empty = is_k ? b_k_empty : b_v_empty;
      const uint32_t q_bytes = a.group * a.tok_tile * 256;
      const int outside = a.num_pages * a.Hkv;             // a slice that the tensor map does not have: zeros
      // the scheduler's place: sequence, kv head, first token of the tile, block in it
      int sb = 0, shd = 0, sj = 0, sblk = 0;
      unsigned at = 0;
      Seq seq{};
      const int waves = sh->waves;
      auto list_next = [&](int n) {                        // lane 0 of the K producer: tile n goes into the ring
        Segment w{};
        unsigned stop = r1;
        if (n <= waves) {
          // tile n of the waves, which are of the only sequence, or the place where the CTA's range of the line begins
          sb = sh->start_b;
          seq = sh->start_seq;
          const unsigned in_head = n < waves ? (seq.n + a.tok_tile - 1) / a.tok_tile : sh->units / a.Hkv;
          unsigned rem = n < waves ? n * gridDim.x + blockIdx.x : r0 - sh->before;
          shd = static_cast<int>(rem / max(in_head, 1u));
          rem -= shd * in_head;
          sj = sblk = 0;
          if (n < waves) {
            sj = static_cast<int>(rem) * a.tok_tile;
            at = 0;
            stop = 0x7fffffffu;
          } else {
            at = r0;
            if (shd >= a.Hkv) at = r1;                     // the waves were all, or cu_seqlens is not a running sum
#pragma unroll 1
            while (sj < seq.n) {
              const unsigned units = tile_blocks(seq, sj, a.tok_tile) + kTileUnits;
              if (rem < units) break;
              rem -= units;
              sj += a.tok_tile;
            }
            sblk = static_cast<int>(rem);
          }
        }
#pragma unroll 1
        while (at < stop) {
          if (sj >= seq.n) {                               // on to the next kv head, or sequence with new tokens
            sj = 0;
            if (++shd == a.Hkv) {
              shd = 0;
#pragma unroll 1
              do {
                if (++sb < a.B) seq = seq_of(a, sb);
              } while (seq.n == 0 && sb < a.B);
              if (sb >= a.B) break;                        // not with a running sum in cu_seqlens
            }
          }
          const int blocks = tile_blocks(seq, sj, a.tok_tile);
          if (sblk < blocks) {
            const int take = static_cast<int>(min(static_cast<unsigned>(blocks - sblk), stop - at));
            w.more = 1;
            w.b = sb, w.kvh = shd;
            w.tok0 = seq.first + sj, w.ntok = min(a.tok_tile, seq.n - sj);
            w.pos0 = seq.pos + sj, w.len = seq.len;
            w.blk0 = sblk, w.nblk = take;
            w.check = max(max(min(w.pos0 + 1, w.len), 0) / kBN - sblk, 0);
            w.slot = take == blocks ? -1 : (sblk > 0 ? 0 : 1);
            if (w.slot == 1) {                             // goes on in the CTAs up to the one that has its last block
              const unsigned x = at + blocks - 1 - base_units, longer = more_until * (share + 1);
              // (the bound holds back only a cu_seqlens whose sequences overlap so often that the units wrapped around)
              const unsigned last = min(x < longer ? x / (share + 1) : more_until + (x - longer) / share, gridDim.x - 1);
              a.owners[blockIdx.x] = Owner{static_cast<int>(last - blockIdx.x) + 1, w.kvh, w.tok0, w.ntok};
            }
            at += take;
            sblk += take;
          }
          if (sblk >= blocks) {                            // the tile's blocks are dealt out: the rest of its units is nobody's
            at += blocks + kTileUnits - sblk;
            sblk = 0;
            sj += a.tok_tile;
          }
          if (w.more) break;
        }
        sh->seg[n % kSched] = w;
        mbar_arrive(b_sched + 8 * (n % kSched));
      };
      int kvh = 0, blk0 = 0, pages = 0;
      const int *table = nullptr;
      auto slice_of = [&](int j) -> int {                  // of page (2 * (blk0 + j) + lane): its slice of the pool's map
        const int page = 2 * (blk0 + j) + lane;
        if (page >= pages) return outside;
        const int e = table[page];
        if (e >= 0 && e < a.num_pages) return e * a.Hkv + kvh;
        if (is_k) status_record(a.status, kStatusBadPage, static_cast<int>(blockIdx.x), e, static_cast<int>(threadIdx.x));
        return outside;
      };
      bool ok = true;
      int g = 0, issued = 0, q_issued = 0;
      for (int n = 0;; ++n) {
        // the next tile's lengths and table entries are fetched while the ring of blocks is full
        if (is_k && lane == 0) list_next(n);
        __syncwarp();
        const volatile Segment *seg = segment_at(n);
        ok = __all_sync(0xffffffffu, seg != nullptr);
        if (!ok || !seg->more) break;
        kvh = seg->kvh, blk0 = seg->blk0;
        const int nblk = seg->nblk, check = seg->check;
        pages = min((seg->len + kPageRows - 1) / kPageRows, 2 * (blk0 + nblk));   // needed here
        table = a.block_table + static_cast<long long>(seg->b) * a.max_pages;
        int next = slice_of(0);
        if (is_k && lane == 0) {
          ok = wait(b_q_empty + 8 * (n & 1), ((n >> 1) & 1) ^ 1);
          if (ok) {
            const int tok0 = seg->tok0;
            mbar_arrive_expect_tx(b_q_full + 8 * (n & 1), q_bytes);
            tma_load_3d(sQ + (n & 1) * kTileBytes, &tm_q, 0, kvh * a.group, tok0, b_q_full + 8 * (n & 1));
            tma_load_3d(sQ + (n & 1) * kTileBytes + kBox, &tm_q, 64, kvh * a.group, tok0, b_q_full + 8 * (n & 1));
            ++q_issued;
          }
        }
        ok = __all_sync(0xffffffffu, ok);
        for (int j0 = 0; j0 < nblk && ok; j0 += 16) {
          const int slices = next;
          if (j0 + 16 < nblk) next = slice_of(j0 + 16);
          const int j1 = min(nblk, j0 + 16);
          for (int j = j0; j < j1 && ok; ++j, ++g) {
            const int s0 = __shfl_sync(0xffffffffu, slices, 2 * (j - j0)), s1 = __shfl_sync(0xffffffffu, slices, 2 * (j - j0) + 1);
            if (lane == 0) {
              const int st = g & 1;
              ok = wait(b_empty + 8 * st, ((g >> 1) & 1) ^ 1);
              if (ok) {
                const uint32_t dst = s_dst + st * kTileBytes, bar = b_full + 8 * st;
                mbar_arrive_expect_tx(bar, kTileBytes);
                tma_load_3d(dst, tm, 0, 0, s0, bar);
                tma_load_3d(dst + kPageBox, tm, 0, 0, s1, bar);
                tma_load_3d(dst + kBox, tm, 64, 0, s0, bar);
                tma_load_3d(dst + kBox + kPageBox, tm, 64, 0, s1, bar);
                ++issued;
                if (is_k) *const_cast<volatile int *>(&sh->k_issued) = issued;
                if (!is_k && j >= check) mbar_arrive(b_look + 8 * st);   // PV(g-2) is done: v_full is at V(g)'s phase
              }
            }
            ok = __all_sync(0xffffffffu, ok);
          }
        }
        if (!ok) break;
      }
      if (!ok && lane == 0) {
        report(sh, kErrProducer, 2 * g + (is_k ? 0 : 1));
        // Unwinding: let the copies already in flight land before the CTA's shared memory goes away.
        for (int spin = 0; spin < 100000; ++spin) {
          bool done = true;
          for (int i = 1; i <= 2; ++i) {
            const int jg = issued - i, jq = q_issued - i;
            if (jg >= 0) done = done && mbar_try_wait(b_full + 8 * (jg & 1), (jg >> 1) & 1);
            if (jq >= 0) done = done && mbar_try_wait(b_q_full + 8 * (jq & 1), (jq >> 1) & 1);
          }
          if (done) break;
          __nanosleep(100);
        }
      }
      __syncwarp();
    } else if (warp == 13) {
      // ================================ score-product issuer ==================================
      // A thread of its own for each of the two products: issuing one and testing barriers for the other in between
      // does not keep the pipe fed.  S(g) goes into the buffer P(g-3) was read from: wait for that PV product first, and
      // in a tile's third block also for the epilogue of the tile before, whose O that buffer takes over.
      if (lane == 0) {
        constexpr int fmt = (DT == NB200_BF16) ? 1 : 0;
        const uint32_t d_hi = static_cast<uint32_t>(umma_desc_sw128(0, 16, 1024) >> 32);
        const uint32_t dq = static_cast<uint32_t>(umma_desc_sw128(sQ, 16, 1024)), dk = static_cast<uint32_t>(umma_desc_sw128(sK, 16, 1024));
        constexpr uint32_t kStageStep = kTileBytes >> 4;   // of buffer / stage 1
        bool ok = true;
        int g = 0, freed = 0;                    // tiles whose O's region has been given back
        int third[3] = {0, 0, 0};                // first block + 2 of the tiles freed + 1 .. (at most three are open)
        uint32_t map = kRegions;
        for (int n = 0; ok; ++n) {
          const volatile Segment *seg = segment_at(n);
          if (!seg) { ok = false; break; }
          if (!seg->more) break;
          const int nblk = seg->nblk;
          if (n > 0) {
            map = next_regions(map, g);
            third[n % 3] = g + 2;
          }
          ok = wait(b_q_full + 8 * (n & 1), (n >> 1) & 1);
          if (!ok) break;
          const uint32_t q_step = (n & 1) * kStageStep;
          const uint32_t idesc_qk = is_small(seg->ntok, a.group) ? umma_idesc_f16(fmt, 0, kBM / 2, kBN) : umma_idesc_f16(fmt, 0, kBM, kBN);
          for (int j = 0; j < nblk && ok; ++j, ++g) {
            const int sb = g % kSBufs;
            ok = wait(b_k_full + 8 * (g & 1), (g >> 1) & 1);
            if (!ok) break;
            if (freed < n && third[(freed + 1) % 3] == g) {
              ok = wait(b_o_free + 8 * (freed & 3), (freed >> 2) & 1);
              if (!ok) break;
              ++freed;
            }
            if (g >= kSBufs) {
              ok = wait(b_pv_done + 8 * sb, ((g - kSBufs) / kSBufs) & 1);
              if (!ok) break;
            }
            tc_fence_after();
            const uint32_t d_tmem = tmem + region(map, sb);
#pragma unroll 1
            for (int half = 0; half < 2; ++half) {          // 64 columns each: 16 of them are 32 bytes of a swizzled row
              const uint32_t q_at = dq + q_step + half * (kBox >> 4), k_at = dk + (g & 1) * kStageStep + half * (kBox >> 4);
#pragma unroll
              for (int kk = 0; kk < 4; ++kk) umma_ss_lo(d_tmem, q_at + kk * 2, k_at + kk * 2, d_hi, idesc_qk, half | kk);
            }
            umma_commit(b_s_full + 8 * sb);
            umma_commit(b_k_empty + 8 * (g & 1));
          }
          if (ok) umma_commit(b_q_empty + 8 * (n & 1));
        }
        if (!ok) report(sh, kErrMma, 2 * g);
      }
      __syncwarp();
    } else {
      // ================================ PV-product issuer ==================================
      if (lane == 0) {
        constexpr int fmt = (DT == NB200_BF16) ? 1 : 0;
        // V is MN-major: 16 kv rows = 2 KB, the two 64-column halves kBox apart
        const uint32_t d_hi = static_cast<uint32_t>(umma_desc_sw128(0, 16, 1024) >> 32);
        const uint32_t dv = static_cast<uint32_t>(umma_desc_sw128(sV, kBox, 1024));
        constexpr uint32_t kStageStep = kTileBytes >> 4;
        bool ok = true;
        int g = 0;
        uint32_t looks = 0;                                  // bit st: parity of the looks at stage st so far
        uint32_t map = kRegions;
        for (int n = 0; ok; ++n) {
          const volatile Segment *seg = segment_at(n);
          if (!seg) { ok = false; break; }
          if (!seg->more) break;
          const int nblk = seg->nblk, check = seg->check;
          if (n > 0) map = next_regions(map, g);
          const uint32_t o_tmem = tmem + region(map, 3);
          const uint32_t idesc_pv = is_small(seg->ntok, a.group) ? umma_idesc_f16(fmt, 1, kBM / 2, kD) : umma_idesc_f16(fmt, 1, kBM, kD);
          for (int j = 0; j < nblk && ok; ++j, ++g) {
            const int sb = g % kSBufs;
            ok = wait(b_v_full + 8 * (g & 1), (g >> 1) & 1);
            if (!ok) break;
            if (j == 0 && g > 0) {   // O goes where P(g-1) was
              ok = wait(b_pv_done + 8 * ((g - 1) % kSBufs), ((g - 1) / kSBufs) & 1);
              if (!ok) break;
            }
            if (j >= check) {
              ok = wait(b_looked + 8 * (g & 1), (looks >> (g & 1)) & 1);
              if (!ok) break;
              looks ^= 1u << (g & 1);
            }
            ok = wait(b_p_full + 8 * sb, (g / kSBufs) & 1);
            if (!ok) break;
            tc_fence_after();
            const uint32_t p_tmem = tmem + region(map, sb), v_at = dv + (g & 1) * kStageStep;
#pragma unroll 1
            for (int k0 = 0; k0 < kBN / 16; k0 += 4) {
#pragma unroll
              for (int kk = 0; kk < 4; ++kk)   // P: 16 packed 16-bit values = 8 TMEM columns per product
                umma_ts_lo(o_tmem, p_tmem + (k0 + kk) * 8, v_at + (k0 + kk) * 128, d_hi, idesc_pv, k0 | kk | j);
            }
            umma_commit(b_pv_done + 8 * sb);
            umma_commit(b_v_empty + 8 * (g & 1));
            if (j + 1 == nblk) umma_commit(b_o_full + 8 * (n & 3));
          }
        }
        if (!ok) report(sh, kErrMma, 2 * g + 1);
      }
      __syncwarp();
    }
  } else if (warp >= 8) {
    // ================================ epilogue: O / l -> out, or (O, m, l) -> workspace ==========================
    const int r = (warp & 3) * 32 + lane;
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    // rows leave through a stage of 32 x 64 bytes per warp, four lanes to a row: whole sectors, eight rows to a store
    unsigned char *const stage = smem + kOffStage + (warp & 3) * kStage;
    uint32_t looks = 0, notes = 0, map = kRegions;
    bool ok = true;
    // A tile's first two blocks are looked through before the epilogue of the tile before, which their products do not
    // wait for; its further blocks after it, because their scores do.  (A tile's tokens are at no more than 128 positions,
    // so the blocks to look through are its last two at most, and the next tile is listed before they are waited for:
    // listing it takes the issue of the tile's last K block, which waits for the PV product of the sixth last.)
    int g0 = 0, done = 0;                                    // first block of tile n, its blocks looked through
    for (int n = 0; ok; ++n) {
      const volatile Segment *seg = segment_at(n);
      ok = __all_sync(0xffffffffu, seg != nullptr);
      if (!ok || !seg->more) break;
      const int nblk = seg->nblk;
      if (n > 0) map = next_regions(map, g0);
      // Listed when tile n's last K block has been asked for, which may take longer than a wait lasts (4 s for 2^29 cached
      // rows): as long as blocks are being asked for, the wait begins again.
      const volatile Segment *after = nullptr;
      for (int then = -1, now; after == nullptr && (now = *const_cast<volatile int *>(&sh->k_issued)) != then; then = now)
        after = segment_at(n + 1);
      ok = __all_sync(0xffffffffu, after != nullptr);
      if (!ok) break;
      const int early = after->more ? min(after->nblk, 2) : 0;
      // ---- V rows that not every row of the tile sees; thread = row of V here ----
      const int from = max(seg->check, done), turns = max(nblk - from, 0), after_from = early ? after->check : 0;
      done = early;
#pragma unroll 1
      for (int i = 0; i < turns + max(early - after_from, 0); ++i) {
        const bool here = i < turns;
        const volatile Segment *of = here ? seg : after;
        const int m = here ? n : n + 1, j = here ? from + i : after_from + i - turns;
        const int g = (here ? g0 : g0 + nblk) + j, st = g & 1, col0 = (of->blk0 + j) * kBN;
        const int lo = of->pos0 + 1 - col0, hi = of->len - col0;   // from lo on the first token sees nothing; the cache ends at hi
        // the producer's word first: v_full alone tells two phases apart, not three
        ok = wait(b_look + 8 * st, (looks >> st) & 1) && wait(b_v_full + 8 * st, (g >> 1) & 1);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        looks ^= 1u << st;
        unsigned char *row = smem + (4 + st) * kTileBytes + r * 128;
        if (r >= hi) {
#pragma unroll 4
          for (int c = 0; c < 16; ++c)
            *reinterpret_cast<uint4 *>(row + (c >> 3) * kBox + ((c + r) & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
        } else if (r >= lo) {
          uint32_t probe[4] = {0u, 0u, 0u, 0u};
#pragma unroll 4
          for (int c = 0; c < 16; ++c) {
            const uint4 x = *reinterpret_cast<const uint4 *>(row + (c >> 3) * kBox + ((c + r) & 7) * 16);
            probe[0] = finite_probe<DT>(x.x, probe[0]);
            probe[1] = finite_probe<DT>(x.y, probe[1]);
            probe[2] = finite_probe<DT>(x.z, probe[2]);
            probe[3] = finite_probe<DT>(x.w, probe[3]);
          }
          bool clean = true;
#pragma unroll
          for (int c = 0; c < 4; ++c) clean = clean && !not_finite16<DT>(probe[c] & 0xffffu) && !not_finite16<DT>(probe[c] >> 16);
          if (!clean) {
#pragma unroll 1
            for (int c = 0; c < kD; ++c) {   // column c: 16-byte piece (c / 8) % 8 of its half, swizzled with the row
              uint16_t *x = reinterpret_cast<uint16_t *>(row + (c >> 6) * kBox + (((c >> 3) ^ r) & 7) * 16) + (c & 7);
              if (not_finite16<DT>(*x)) {
                const int kind = kind16<DT>(*x);
                *x = 0;
                atomicMax(&sh->taint[m & 1][kind][c], (static_cast<unsigned long long>(m + 1) << 32) | (0x7fffffffu - static_cast<unsigned>(col0 + r)));
                *reinterpret_cast<volatile int *>(&sh->taint_any[m & 1]) = m + 1;
              }
            }
          }
        }
        fence_proxy_async_smem();
        mbar_arrive(b_looked + 8 * st);
        __syncwarp();
      }
      if (!ok) break;
      g0 += nblk;
      const int slot = seg->slot;
      const int ntok = seg->ntok;
      const bool small = is_small(ntok, a.group);
      const int row = row_at(r, small), tok = token_of(a, row);
      int out_row[4];                                        // token << 8 | head
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = row_at((warp & 3) * 32 + 8 * i + (lane >> 2), small), tok = token_of(a, row);
        out_row[i] = tok << 8 | (row - tok * a.group);
      }
      const int last_seen = min(seg->pos0 + tok, seg->len - 1);
      uint4 *const dst = a.out + static_cast<size_t>(seg->tok0) * a.out_t + static_cast<size_t>(seg->kvh * a.group) * a.out_h;
      const uint32_t tO = tmem + region(map, 3) + lane_addr;
      // a table entry outside the pool among the pages read: NaN instead of a sum that lacks them
      bool bad = false;
      {
        const int *table = a.block_table + static_cast<long long>(seg->b) * a.max_pages;
        const int end = min(2 * (seg->blk0 + seg->nblk), (seg->len + kPageRows - 1) / kPageRows);
#pragma unroll 1
        for (int p = 2 * seg->blk0 + lane; p < end; p += 32) bad = bad || static_cast<unsigned>(table[p]) >= static_cast<unsigned>(a.num_pages);
        bad = __any_sync(0xffffffffu, bad);
      }
      ok = __all_sync(0xffffffffu, wait(b_lm_ready + 8 * (n & 1), (n >> 1) & 1));
      if (!ok) break;
      const float2 lm0 = sh->lm[n & 1][0][r], lm1 = sh->lm[n & 1][1][r];
      mbar_arrive(b_lm_free + 8 * (n & 1));
      const float mf = fmaxf(lm0.x, lm1.x);   // the running maximum never decreases: the later one is the larger
      float l = (lm0.y == 0.f ? 0.f : lm0.y * ex2(lm0.x - mf)) + (lm1.y == 0.f ? 0.f : lm1.y * ex2(lm1.x - mf));
      // A row that sees nothing is 0: every weight was 0 and every V looked through, so O is.  One that sees scores of -inf
      // alone has l = 0 too, and 0 / 0 = NaN as the softmax of such a row is.
      const bool empty = last_seen < 0;
      if (bad) l = __int_as_float(0x7fffffff);
      const float inv = slot >= 0 || (empty && !bad) ? 1.f : 1.f / l;
      const uint64_t inv2 = f2_pack(inv, inv);
      float *po = nullptr;
      if (slot >= 0) {
        const long long pr = (static_cast<long long>(blockIdx.x) * 2 + slot) * kBM + row;
        po = a.part_o + pr * kD;
        if (tok < ntok) a.part_ml[pr] = make_float2(mf, l);
      }
      ok = __all_sync(0xffffffffu, wait(b_o_full + 8 * (n & 3), (n >> 2) & 1));
      if (!ok) break;
      tc_fence_after();
      // the PV products waited for every look at the tile's V, so the notes of all the warps are there
      const bool tainted = *reinterpret_cast<volatile int *>(&sh->taint_any[n & 1]) == n + 1;
#pragma unroll 1
      for (int c = 0; c < kD / 32; ++c) {
        uint32_t o[32];
        tmem_ld32(tO + c * 32, o);
        tmem_wait_ld();
        if (c == kD / 32 - 1) {   // O is in registers: its region may be overwritten
          tc_fence_before();
          mbar_arrive(b_o_free + 8 * (n & 3));
        }
        if (slot < 0) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float2 x = f2_unpack(f2_mul(f2_pack(__uint_as_float(o[8 * k + 2 * i]), __uint_as_float(o[8 * k + 2 * i + 1])), inv2));
              w[i] = pack2<DT>(x.x, x.y);
            }
            *reinterpret_cast<uint4 *>(stage + lane * 64 + ((k ^ (lane >> 1)) & 3) * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = 8 * i + (lane >> 2);
            const uint4 x = *reinterpret_cast<const uint4 *>(stage + row * 64 + ((lane ^ (row >> 1)) & 3) * 16);
            if ((out_row[i] >> 8) < ntok)
              dst[static_cast<size_t>(out_row[i] >> 8) * a.out_t + static_cast<size_t>(out_row[i] & 0xff) * a.out_h + c * 4 + (lane & 3)] = x;
          }
          __syncwarp();
        } else {   // twice per CTA at most: straight from the registers
          if (tok < ntok) {
#pragma unroll
            for (int k = 0; k < 8; ++k)
              *reinterpret_cast<uint4 *>(po + c * 32 + 4 * k) = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
          }
          __syncwarp();
        }
      }
      if (tainted) {   // columns with values that are not finite: added in the rows that see them
        __syncwarp();
        uint16_t *const mine = reinterpret_cast<uint16_t *>(dst + static_cast<size_t>(tok) * a.out_t + static_cast<size_t>(row - tok * a.group) * a.out_h);
#pragma unroll 1
        for (int c = 0; c < kD && tok < ntok; ++c) {
          float add = 0.f;
#pragma unroll 1
          for (int kind = 0; kind < 3; ++kind) {
            const unsigned long long note = *reinterpret_cast<volatile unsigned long long *>(&sh->taint[n & 1][kind][c]);
            if (static_cast<int>(note >> 32) == n + 1 && static_cast<int>(0x7fffffffu - static_cast<uint32_t>(note)) <= last_seen)
              add += __int_as_float(kind == 0 ? 0x7fffffff : (kind == 1 ? 0x7f800000 : 0xff800000));
          }
          if (add == 0.f) continue;
          if (slot < 0)
            store1<DT>(mine, c, load1<DT>(mine, c) + add);
          else
            po[c] += add;
        }
        __syncwarp();
        // every warp has read its notes before any looks on and writes over them
        mbar_arrive(b_notes_read);
        ok = __all_sync(0xffffffffu, wait(b_notes_read, notes));
        notes ^= 1;
      }
    }
    if (!ok && lane == 0) report(sh, kErrEpilogue, g0);
  } else {
    // ================================ softmax: warpgroup w takes the blocks g with g & 1 == w ================
    asm volatile("setmaxnreg.inc.sync.aligned.u32 144;");
    const int w = warp >> 2;
    const int r = (warp & 3) * 32 + lane;                     // row in the tile == TMEM lane
    const uint32_t lane_addr = static_cast<uint32_t>((warp & 3) * 32) << 16;
    int tok = 0;
    int n = -1, g0 = 0;
    uint32_t map = kRegions;
    bool ok = true, more = true;
    int nblk = 0, blk0 = 0, pos0 = 0, len = 0, ntok = 0;
    float m_mine = -INFINITY, l = 0.f;
#pragma unroll 1
    for (int g = w; ok; g += 2) {
      // tiles that end before block g: hand (maximum, partial sum) to the epilogue and move on
#pragma unroll 1
      while (more && g >= g0 + nblk) {
        if (n > 1) ok = __all_sync(0xffffffffu, wait(b_lm_free + 8 * (n & 1), ((n >> 1) & 1) ^ 1));   // tile n - 2's have been read
        if (n >= 0 && ok) {
          sh->lm[n & 1][w][r] = make_float2(m_mine, l);
          mbar_arrive(b_lm_ready + 8 * (n & 1));
        }
        m_mine = -INFINITY;
        l = 0.f;
        g0 += nblk;
        if (++n > 0) map = next_regions(map, g0);
        const volatile Segment *seg = segment_at(n);
        ok = __all_sync(0xffffffffu, ok && seg != nullptr);
        if (!ok) break;
        more = seg->more;
        nblk = seg->nblk, blk0 = seg->blk0, pos0 = seg->pos0, len = seg->len, ntok = seg->ntok;
        tok = token_of(a, row_at(r, is_small(ntok, a.group)));
      }
      if (!ok || !more) break;
      const int j = g - g0;
      const int sb = g % kSBufs;
      const int col0 = (blk0 + j) * kBN;                       // cache row of the block's first column
      const uint32_t tS = tmem + region(map, sb) + lane_addr;
      ok = __all_sync(0xffffffffu, wait(b_s_full + 8 * sb, (g / kSBufs) & 1));
      if (!ok) break;
      tc_fence_after();
      float m_prev = -INFINITY;
      if (g > 0) {
        // block g-1 has decided on its maximum (and, before that, has read the slot this block will overwrite)
        ok = __all_sync(0xffffffffu, wait(b_m_ready + 8 * ((g - 1) & 1), ((g - 1) >> 1) & 1));
        if (!ok) break;
        if (j > 0) m_prev = sh->mslot[(g - 1) & 1][r];
      }
      // column c of the block is seen by this row iff c <= vis
      const int vis = tok < ntok ? min(pos0 + tok, len - 1) - col0 : -1;
      const bool warp_works = __any_sync(0xffffffffu, vis >= 0);   // else P may hold anything: no row of the warp is used, or none sees the block
      float m_new = m_prev;
      if (!warp_works) {
        // a row that sees nothing here still must not take anything from the products: P = 0
        sh->mslot[g & 1][r] = m_prev;
        mbar_arrive(b_m_ready + 8 * (g & 1));
        const uint32_t zero[16] = {};
#pragma unroll
        for (int c = 0; c < kBN / 32; ++c) tmem_st16(tS + c * 16, zero);
      } else {
        if (__any_sync(0xffffffffu, vis < kBN - 1)) {   // hidden columns, in place: once per tile or twice, so as little code as possible
#pragma unroll 1
          for (int c = 0; c < kBN; c += 16) {
            uint32_t x[16];
            tmem_ld16(tS + c, x);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = (c + k > vis) ? 0xff800000u : x[k];
            tmem_st16(tS + c, x);
          }
          tmem_wait_st();
        }
        // Two passes over the scores, read from tensor memory 64 columns at a time: holding all 128 in registers takes 176 of
        // them, which the epilogue and the producers then lack, and twice the code (176 against 164 us at a 4096-token
        // first chunk under sustained load, and 120 against 100 us for 512 sequences of 32 tokens over 128 rows).
        float mc[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) mc[c] = -INFINITY;
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t v[64];
          tmem_ld32p(tS + h * 64, v);
          tmem_ld32p(tS + h * 64 + 32, v + 32);
          tmem_wait_ld();
#pragma unroll
          for (int k = 0; k < 8; k += 2) {
#pragma unroll
            for (int c = 0; c < 8; ++c) mc[c] = max3(mc[c], __uint_as_float(v[c * 8 + k]), __uint_as_float(v[c * 8 + k + 1]));
          }
        }
        const float mx = fmaxf(max3(mc[0], mc[1], mc[2]), fmaxf(max3(mc[3], mc[4], mc[5]), fmaxf(mc[6], mc[7])));
        const float m_blk = mx * a.scale_log2;                   // -inf if the row sees nothing of this block
        // ---- the maximum to use: the one block g-1 decided on, unless this block exceeds it by more than 2^8 ----
        const bool need = j > 0 && m_blk > m_prev + kRescaleThreshold;
        m_new = (j == 0 || need) ? m_blk : m_prev;
        sh->mslot[g & 1][r] = m_new;
        mbar_arrive(b_m_ready + 8 * (g & 1));
        if (__any_sync(0xffffffffu, need)) {
          // O must hold every product up to block g-1 and none may be in flight
          ok = __all_sync(0xffffffffu, wait(b_pv_done + 8 * ((g - 1) % kSBufs), ((g - 1) / kSBufs) & 1));
          if (!ok) break;
          tc_fence_after();
          const float f = need ? ex2(m_prev - m_blk) : 1.f;
          const uint32_t tO = tmem + region(map, 3) + lane_addr;
#pragma unroll 1
          for (int c = 0; c < kD / 16; ++c) {
            uint32_t o[16];
            tmem_ld16(tO + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
            tmem_st16(tO + c * 16, o);
          }
          tmem_wait_st();
        }
        if (m_mine != m_new) {   // bring the partial sum to the new maximum (2^(-inf) = 0 on the first block)
          l *= ex2(m_mine - m_new);
          m_mine = m_new;
        }
        // ---- p = 2^(s*scale - m), row sum, pack to 16 bit; P overwrites columns 0..63 of S ----
        const float m_use = m_new == -INFINITY ? 0.f : m_new;    // nothing seen so far: every p is 2^(-inf) = 0
        const uint64_t c2 = f2_pack(a.scale_log2, a.scale_log2), nm2 = f2_pack(kLift<DT> - m_use, kLift<DT> - m_use);
        uint64_t lsum2 = f2_pack(0.f, 0.f);
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
          uint32_t v[64];
          tmem_ld32p(tS + h * 64, v);
          tmem_ld32p(tS + h * 64 + 32, v + 32);
          tmem_wait_ld();
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              const uint64_t x2 = f2_fma(
                  f2_pack(__uint_as_float(v[c * 32 + 2 * k]), __uint_as_float(v[c * 32 + 2 * k + 1])), c2, nm2);
              const float2 x = f2_unpack(x2);
              const float p0 = ex2(x.x), p1 = ex2(x.y);
              lsum2 = f2_add(lsum2, f2_pack(p0, p1));
              pk[k] = pack2<DT>(p0, p1);
            }
            tmem_st16(tS + h * 32 + c * 16, pk);
          }
        }
        const float2 ls = f2_unpack(lsum2);
        l += ls.x + ls.y;
      }
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(b_p_full + 8 * sb);
    }
    if (!ok && lane == 0) report(sh, kErrSoftmax, g0);
  }

  // ================================ tear-down =====================================
  tc_fence_before();
  __syncthreads();
  if (threadIdx.x == 0 && sh->error[0] != 0)
    status_record(a.status, sh->error[0], static_cast<int>(blockIdx.x), sh->error[1], sh->error[2]);
  if (warp == 15) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

// Joins the parts of the tiles that were cut, in the order of the line: part 0 in slot 1 of the CTA where the tile begins,
// part i in slot 0 of the i-th CTA behind it.  One warp per row.
constexpr int kJoinWarps = 8;
template <int DT> __global__ void __launch_bounds__(kJoinWarps * 32) attn_paged_join_kernel(const Args a) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int lane = threadIdx.x & 31;
  const int r = blockIdx.y * kJoinWarps + (threadIdx.x >> 5);
  auto place = [&](int i) { return (static_cast<long long>(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * kBM + r; };
  const Owner own = a.owners[blockIdx.x];
  const float2 first = a.part_ml[place(min(lane, kMaxCtas - 1 - static_cast<int>(blockIdx.x)))];   // asked for with the owner, used if there is a part
  if (own.parts == 0 || r >= own.ntok * a.group) return;
  // lane i holds (m, l) of parts i, i + 32, ...; m is a maximum that the part's weights are relative to
  float big = -INFINITY;
#pragma unroll 1
  for (int i = lane; i < own.parts; i += 32) {
    const float2 ml = i == lane ? first : a.part_ml[place(i)];
    if (ml.y != 0.f) big = fmaxf(big, ml.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float l = 0.f;
#pragma unroll 1
  for (int i0 = 0; i0 < own.parts; i0 += 32) {
    const int here = min(32, own.parts - i0);
    float w = -1.f;                                       // of part i0 + lane; negative: the row saw nothing of it
    if (lane < here) {
      const float2 ml = i0 == 0 ? first : a.part_ml[place(i0 + lane)];
      if (ml.y != 0.f) {
        w = ex2(ml.x - big);
        l = fmaf(w, ml.y, l);
      }
    }
#pragma unroll 1
    for (int i = 0; i < here; i += 8) {
      float4 o[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i + k < here) o[k] = reinterpret_cast<const float4 *>(a.part_o + place(i0 + i + k) * kD)[lane];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float wk = __shfl_sync(0xffffffffu, w, (i + k) & 31);
        if (i + k < here && !(wk < 0.f)) {
          acc.x = fmaf(wk, o[k].x, acc.x);
          acc.y = fmaf(wk, o[k].y, acc.y);
          acc.z = fmaf(wk, o[k].z, acc.z);
          acc.w = fmaf(wk, o[k].w, acc.w);
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
  // Every row of a tile that was cut sees something: the tile has two blocks or more, its tokens are at 128 positions at most.
  const float inv = 1.f / l;
  uint4 *dst = a.out + static_cast<size_t>(own.tok0 + token_of(a, r)) * a.out_t + static_cast<size_t>(own.kvh * a.group + r - token_of(a, r) * a.group) * a.out_h;
  reinterpret_cast<uint2 *>(dst)[lane] = make_uint2(pack2<DT>(acc.x * inv, acc.y * inv), pack2<DT>(acc.z * inv, acc.w * inv));
}

int map_3d(CUtensorMap *tm, const void *ptr, const cuuint64_t (&dims)[3], const cuuint64_t (&strides)[2],
           const cuuint32_t (&box)[3], int dtype) {
  EncodeTiledFnT enc = tma_encode_fn();
  NB200_REQUIRE(enc, NB200_ERR_LAUNCH, "attn_paged: cuTensorMapEncodeTiled is not available from the driver");
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = tma_encode(enc, tm, dtype == NB200_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
                         const_cast<void *>(ptr), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                         CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  NB200_REQUIRE(r == CUDA_SUCCESS, NB200_ERR_LAUNCH, "attn_paged: cuTensorMapEncodeTiled failed with code %d", (int)r);
  return NB200_OK;
}

// Multiprocessors of the current device, looked up once per device together with the kernel's shared-memory limit.
template <int DT> int device_sms(int *sms) {
  static std::atomic<int> known[64];
  int dev = 0;
  NB200_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && (*sms = known[dev].load(std::memory_order_acquire)) > 0) return NB200_OK;
  NB200_CHECK_CUDA(cudaFuncSetAttribute(attn_paged_kernel<DT>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBytes));
  NB200_CHECK_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  if (dev < 64) known[dev].store(*sms, std::memory_order_release);
  return NB200_OK;
}

template <int DT> int launch(const CUtensorMap &tq, const CUtensorMap &tk, const CUtensorMap &tv, const Args &a, cudaStream_t st) {
  int sms = 0, rc;
  if ((rc = device_sms<DT>(&sms)) != NB200_OK) return rc;
  const int grid = sms < kMaxCtas ? sms : kMaxCtas;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;   // both wait on the device for what is before them
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  NB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attn_paged_kernel<DT>, tq, tk, tv, a));
  const int rows = a.T < a.tok_tile ? a.T * a.group : a.tok_tile * a.group;   // of the fullest tile
  cfg.gridDim = dim3(grid, (rows + kJoinWarps - 1) / kJoinWarps);
  cfg.blockDim = dim3(kJoinWarps * 32);
  cfg.dynamicSmemBytes = 0;
  NB200_CHECK_CUDA(cudaLaunchKernelEx(&cfg, attn_paged_join_kernel<DT>, a));
  return NB200_OK;
}

}  // namespace
}  // namespace nb200

using namespace nb200;

extern "C" size_t nb200_attn_paged_workspace_bytes(void) { return kPartO + kPartMl + kMaxCtas * sizeof(Owner); }

extern "C" int nb200_attn_paged(const void *q, const void *k_pages, const void *v_pages, const int *block_table,
                                const int *cu_seqlens, const int *seq_lens, void *workspace, void *out,
                                const long long *strides, int T, int B, int Hq, int Hkv, int num_pages, int max_pages,
                                int page_size, int D, int dtype, float scale_log2, int *status, void *stream) {
  const char *who = "attn_paged";
  NB200_REQUIRE(q && k_pages && v_pages && block_table && cu_seqlens && seq_lens && workspace && out && strides,
                NB200_ERR_BAD_ARG, "%s: null pointer", who);
  NB200_REQUIRE(T > 0 && B > 0 && Hq > 0 && Hkv > 0 && num_pages > 0 && max_pages > 0 && D > 0, NB200_ERR_BAD_ARG,
                "%s: non-positive extent", who);
  NB200_REQUIRE(scale_log2 > 0.f, NB200_ERR_BAD_ARG, "%s: scale_log2 must be positive", who);
  NB200_REQUIRE(dtype == NB200_F16 || dtype == NB200_BF16, NB200_ERR_UNSUPPORTED, "%s: dtype %d (f16 and bf16 only)", who, dtype);
  NB200_REQUIRE(D == kD, NB200_ERR_UNSUPPORTED, "%s: D = %d, only 128 is implemented", who, D);
  NB200_REQUIRE(page_size == kPageRows, NB200_ERR_UNSUPPORTED, "%s: page_size = %d, only %d rows per page is implemented", who,
                page_size, kPageRows);
  NB200_REQUIRE(Hq % Hkv == 0, NB200_ERR_UNSUPPORTED, "%s: Hq %% Hkv != 0", who);
  NB200_REQUIRE(Hq / Hkv <= kBM, NB200_ERR_UNSUPPORTED, "%s: more than 128 query heads per kv head", who);
  NB200_REQUIRE(Hq <= 65535, NB200_ERR_UNSUPPORTED, "%s: too many heads", who);
  NB200_REQUIRE(T < (1 << 30) && max_pages <= (1 << 30) / kPageRows, NB200_ERR_UNSUPPORTED,
                "%s: T or max_pages * page_size does not fit 30 bits", who);
  // the device counts blocks in 32 bits: tiles (their number bounded by full tiles and one remainder per sequence) times
  // the longest sequence's blocks
  const double tiles = (static_cast<double>(T) / (kBM / (Hq / Hkv)) + B) * Hkv;
  NB200_REQUIRE(tiles * (max_pages / 2 + 2.0 + kTileUnits) < 4.0e9, NB200_ERR_UNSUPPORTED,
                "%s: T and max_pages are too large for one call", who);
  NB200_REQUIRE(static_cast<long long>(num_pages) * Hkv < (1ll << 31) - 1, NB200_ERR_UNSUPPORTED,
                "%s: num_pages * Hkv does not fit 31 bits", who);
  NB200_REQUIRE(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out) && aligned16(workspace),
                NB200_ERR_BAD_ARG, "%s: q, out, the page pools and the workspace must be 16-byte aligned", who);
  const int extents[4] = {T, Hq, T, Hq};
  long long s[4];
  for (int i = 0; i < 4; ++i) {
    s[i] = extents[i] == 1 ? kD : strides[i];              // a stride that is never taken
    NB200_REQUIRE(s[i] >= kD && s[i] % 8 == 0 && s[i] < (1ll << 34), NB200_ERR_BAD_ARG,
                  "%s: the strides of q and out must be multiples of 16 bytes, at least a row", who);
  }
  NB200_REQUIRE(rows_apart(kD, {T, Hq}, {s[2], s[3]}), NB200_ERR_BAD_ARG, "%s: the rows of out must lie apart", who);
  NB200_REQUIRE(q != out, NB200_ERR_BAD_ARG, "%s: out must not be q", who);   // a tile that is cut is read by several CTAs
  Args a{};
  a.block_table = block_table, a.cu_seqlens = cu_seqlens, a.seq_lens = seq_lens;
  a.out = static_cast<uint4 *>(out), a.out_t = static_cast<unsigned>(s[2] / 8), a.out_h = static_cast<unsigned>(s[3] / 8);
  a.T = T, a.B = B, a.Hkv = Hkv, a.group = Hq / Hkv, a.tok_tile = kBM / a.group, a.inv_group = ((1 << 16) + a.group - 1) / a.group;
  a.num_pages = num_pages, a.max_pages = max_pages, a.scale_log2 = scale_log2, a.status = status;
  char *ws = static_cast<char *>(workspace);
  a.part_o = reinterpret_cast<float *>(ws);
  a.part_ml = reinterpret_cast<float2 *>(ws + kPartO);
  a.owners = reinterpret_cast<Owner *>(ws + kPartO + kPartMl);
  CUtensorMap tq, tk, tv;
  int rc;
  // rows of a Q tile: tokens, and the group's heads inside a token
  if ((rc = map_3d(&tq, q, {kD, static_cast<cuuint64_t>(Hq), static_cast<cuuint64_t>(T)},
                   {static_cast<cuuint64_t>(s[1]) * 2, static_cast<cuuint64_t>(s[0]) * 2},
                   {64, static_cast<cuuint32_t>(a.group), static_cast<cuuint32_t>(a.tok_tile)}, dtype)) != NB200_OK)
    return rc;
  const cuuint64_t slices = static_cast<cuuint64_t>(num_pages) * Hkv;
  if ((rc = map_3d(&tk, k_pages, {kD, kPageRows, slices}, {kD * 2, kPageRows * kD * 2}, {64, kPageRows, 1}, dtype)) != NB200_OK)
    return rc;
  if ((rc = map_3d(&tv, v_pages, {kD, kPageRows, slices}, {kD * 2, kPageRows * kD * 2}, {64, kPageRows, 1}, dtype)) != NB200_OK)
    return rc;
  auto st = static_cast<cudaStream_t>(stream);
  if (dtype == NB200_BF16) return launch<NB200_BF16>(tq, tk, tv, a, st);
  return launch<NB200_F16>(tq, tk, tv, a, st);
}
