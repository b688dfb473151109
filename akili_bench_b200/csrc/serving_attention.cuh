// serving_attention.cuh — attention of packed queries over packed keys
// (prompts) or over a paged cache (new tokens, drafted trees), on tcgen05:
//
//   o_i = sum_j softmax_j(scale q_i.k_j) v_j   over the keys j that i sees
//
// This file holds the forms with the query rows on the M side of the tensor
// core; decode_attention.cuh the one for few rows.
//
// Rows.  The G = q_heads / kv_heads query heads of a key head share its keys,
// so the rows of a 128-row tile are tokens times P heads, P = G (or its
// largest divisor up to 128): row r is token r / P, head r % P of the group.
// Short sequences fill the tensor core that way, keys are loaded once for the
// group, and a causal tile spans few tokens, so that its diagonal wastes
// little.
//
// One CTA per SM, 640 threads, two streams of scores, each with its own S/P
// and O accumulators in tensor memory (S_t and P_t at columns 128 t, O_t at
// 256 + 128 t), so that the tensor core works on one stream while the
// softmax of the other runs:
//   pair form   stream t is tile t of two; both read every key block.  For
//               prompts and large trees.
//   single form both streams are the same tile, stream t reads the key blocks
//               of parity t, and the two are merged at the end.  For trees of
//               65 to 128 rows, and prompts whose tiles all run at once.
// Warps:
//   0, 18        key and value loads: blocks of 128 keys into two rings, one
//                TMA box per block (packed) or one per page part (paged).
//   1            TMEM owner and MMA issuer: per step O_t += P_t V of the
//                stream's previous block, then S_t = Q_t K^T of its next one
//                (over the columns of that P_t; the MMAs run in order).
//   2..9, 10..17 softmax of stream 0 and 1: two threads per row with 64 of a
//                block's 128 scores each.  The running maximum only matters
//                where it grows by more than 2^8 (a stale one cancels in
//                O / l), so their two warps vote behind one barrier a block
//                and exchange maxima through shared memory, and rescale O_t,
//                only then.  P = exp2(scale log2e s - m) goes over S_t in two
//                parts, each announced to the MMA warp on its own.
//   19           scheduler: finds the next piece of work, hands it to the
//                others through a small ring, and loads its Q by TMA as soon
//                as the last scores of the piece before are done.  A piece
//                used to cost 16000 cycles beyond its blocks (Q loaded row by
//                row 7900 of them); now its start overlaps the end of the last.
//
// Work.  Prompts: a grid of one block per (tile pair, head group), the tiles
// with the most keys first; a CTA that is done takes over the next block that
// has not started (cluster launch control).  Cache: the key blocks of all
// (sequence, head group, tile) items form one line that is cut into equal
// shares, one per CTA, so uneven lengths and few long sequences fill the GPU
// alike; an item that is cut leaves its parts (O, m, l in fp32) in the
// workspace and a join kernel adds them up in order.
//
// Bound by the chain of a block: scores, TMEM load, maximum, exponentials, P,
// product.  One stream alone would take 2300 cycles a block; the two overlap to
// 60% of the tensor pipe (and of the exponential unit; a copy without
// exponentials took the same time, at a clock that was not recorded).
// Measured: 8 causal prompts of 4096 tokens, 32 heads of 128, fp16: 1.19 ms, 925
// TFLOP/s of visible pairs; six uneven bf16 prompts with 32/8 heads: 949
// TFLOP/s; 24 short ones with 14/2 heads of 64: 12 us; 16 drafted trees over 700
// to 5999 tokens: 73 us (77 with nothing in L2).  Of the 96 registers that 640
// threads leave, the single-tile forms spill 22 to 32 bytes a thread, the paged
// pair form 12 to 16.
#pragma once
#include <type_traits>

#include "cache.cuh"
#include "flash.cuh"
#include "rope.cuh"
#include "sm100.cuh"

namespace akili {

constexpr int kSvRows = 128;  // rows of a tile
constexpr int kSvKeys = 128;  // keys of a block
constexpr int kSvThreads = 640;
constexpr int kSvJoinThreads = 256;
// Blocks that share a cut item: the rows of the few-row form (8 a block), the
// columns of the row forms (a thread takes 16 of a row).
template <int kTileRows, int DP>
constexpr int kSvJoinSplit = kTileRows < kSvRows ? (kTileRows + 7) / 8 : DP / 16 * kTileRows / kSvJoinThreads;

struct ServingArgs {
  const void* q;
  void* o;
  float* lse;
  const int* cu_q;
  const int* cu_k;  // packed keys
  const int* ctx;   // paged keys
  const int* page_table;
  const unsigned int* mask;
  float* parts;  // paged keys: O, m and l of cut items
  int4* cuts;    // row forms, paged keys: the cut item that starts in each share
  int q_heads, kv_heads, group, head_dim, batch, total_q, total_k, causal;
  int pack;         // heads of a token in one tile; the head groups are q_heads / pack
  int head_groups;  // q_heads / pack
  int groups_per_kv;
  int tile_tokens;  // of a 128-row tile: 128 / pack
  int num_pages, page_size, max_pages, mask_words;
  int box_rows;     // paged keys: rows of a TMA box, a divisor of page_size
  int chunk_heads;  // packed keys: head groups that are scheduled together
  float scale_log2;
  long long q_st[2], o_st[2];
  long long table_stride, mask_stride;
};

// ------------------------------------------------------------------- work --
struct SvSeq {
  int q0, n;       // query rows
  int k0, m;       // key rows (k0: packed only)
  int sure;        // keys every row sees (cache), or m - n (prompts)
};

template <bool kPaged>
__device__ __forceinline__ SvSeq sv_sequence(const ServingArgs& a, int b, bool* clamped) {
  SvSeq s;
  s.q0 = min(max(a.cu_q[b], 0), a.total_q);
  s.n = min(max(a.cu_q[b + 1], s.q0), a.total_q) - s.q0;
  if constexpr (kPaged) {
    const int c = max(a.ctx[b], 0);
    const long long cap = static_cast<long long>(a.max_pages) * a.page_size;
    const long long m = static_cast<long long>(c) + s.n;
    *clamped = m > cap;
    s.k0 = 0;
    s.m = static_cast<int>(min(m, cap));
    s.sure = min(c, s.m);
  } else {
    s.k0 = min(max(a.cu_k[b], 0), a.total_k);
    s.m = min(max(a.cu_k[b + 1], s.k0), a.total_k) - s.k0;
    s.sure = s.m - s.n;
    *clamped = false;
  }
  return s;
}

// A run of key blocks of one (sequence, head group, tile).
struct SvPiece {
  SvSeq s;
  int b, hk, tile;
  int kb, loads;    // first key block, blocks
  int part;         // slot of the workspace, or -1: the whole item
  long long first;  // place of the item's first block on the line
};

// An item's start and end take about as long as this many blocks, and count as
// such on the line that is cut into shares (before its first block).  25 drawn
// batches, geometric mean: 1 block 26.7 us, 2 25.6, 3 25.4, 4 24.0, 6 23.9; 16
// long drafted trees: 77.5, 77.8, 78.8, 80.5, 84.6.
constexpr int kSvItemCost = 4;

// A CTA's share of the line of key blocks.  kTileRows: rows of an item, 128
// or 256 of the row forms, 16 to 64 of the few-row form (whose tiles hold
// consecutive rows and need not start at a token).
template <int kTileRows>
struct SvWalk {
  long long pos, begin, end, off;  // off: position within sequence b
  int b;
  SvSeq s;
  int tiles, blocks;
  long long size;

  __device__ __forceinline__ void load(const ServingArgs& a, bool* clamped) {
    s = sv_sequence<true>(a, b, clamped);
    if constexpr (kTileRows >= kSvRows) {
      const int per = (kTileRows / kSvRows) * a.tile_tokens;
      tiles = (s.n + per - 1) / per;
    } else {
      tiles = (s.n * a.group + kTileRows - 1) / kTileRows;
    }
    blocks = (s.m + kSvKeys - 1) / kSvKeys;
    size = static_cast<long long>(a.head_groups) * tiles * (blocks > 0 ? blocks + kSvItemCost : 0);
  }
  __device__ __forceinline__ bool next(const ServingArgs& a, int cta, SvPiece& p) {
    while (pos < end) {
      while (off >= size) {
        off -= size;
        if (++b >= a.batch) return false;
        bool clamped;
        load(a, &clamped);
      }
      const int units = blocks + kSvItemCost;
      long long item;
      int at;  // unit within the item
      if ((off >> 32) == 0) {  // (a 64-bit division costs some 100 cycles more)
        const uint32_t i = static_cast<uint32_t>(off) / static_cast<uint32_t>(units);
        item = i;
        at = static_cast<int>(static_cast<uint32_t>(off) - i * static_cast<uint32_t>(units));
        p.hk = static_cast<int>(i / static_cast<uint32_t>(tiles));
      } else {
        item = off / units;
        at = static_cast<int>(off - item * units);
        p.hk = static_cast<int>(item / tiles);
      }
      const int take = static_cast<int>(min(static_cast<long long>(units - at), end - pos));
      p.s = s;
      p.b = b;
      p.tile = static_cast<int>(item - static_cast<long long>(p.hk) * tiles);
      p.kb = max(at - kSvItemCost, 0);
      p.loads = max(at + take - kSvItemCost, 0) - p.kb;
      p.part = p.loads == blocks ? -1 : 2 * cta + (pos == begin ? 0 : 1);
      p.first = pos - at + kSvItemCost;
      pos += take;
      off += take;
      if (p.loads > 0) return true;  // (a share may end before the item's first block)
    }
    return false;
  }
};

__device__ __forceinline__ long long warp_sum(long long v) {
#pragma unroll
  for (int x = 16; x; x >>= 1) v += __shfl_xor_sync(0xffffffffu, v, x);
  return v;
}
__device__ __forceinline__ long long warp_scan(long long v) {  // inclusive
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const long long u = __shfl_up_sync(0xffffffffu, v, x);
    if (lane >= x) v += u;
  }
  return v;
}

// Sequence b's place on the line (no blocks past the batch).
template <int kTileRows>
__device__ __forceinline__ void sv_line_sequence(const ServingArgs& a, int b, bool record, SvWalk<kTileRows>& w) {
  w.b = b;
  w.size = 0;
  if (b >= a.batch) return;
  bool clamped;
  w.load(a, &clamped);
  if (record && clamped) record_bad_index();
}

// The share of CTA `cta` of `ctas` (one warp): false if it is empty.
template <int kTileRows>
__device__ __forceinline__ bool sv_share(const ServingArgs& a, int cta, int ctas, SvWalk<kTileRows>& w,
                                         long long* quota_out, long long* total_out) {
  const int lane = threadIdx.x & 31;
  SvWalk<kTileRows> mine;
  sv_line_sequence<kTileRows>(a, lane, cta == 0, mine);
  long long total = mine.size;
  for (int b0 = 32; b0 < a.batch; b0 += 32) {
    SvWalk<kTileRows> more;
    sv_line_sequence<kTileRows>(a, b0 + lane, cta == 0, more);
    total += more.size;
  }
  total = warp_sum(total);
  // (a 64-bit division costs some 100 cycles more)
  const long long quota = total + ctas <= 0xffffffffll
                              ? static_cast<uint32_t>(total + ctas - 1) / static_cast<uint32_t>(ctas)
                              : (total + ctas - 1) / ctas;
  *quota_out = quota;
  *total_out = total;
  w.begin = w.pos = cta * quota;
  w.end = min(w.begin + quota, total);
  if (w.begin >= total) return false;
  long long before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    if (b0 > 0) sv_line_sequence<kTileRows>(a, b0 + lane, false, mine);
    const long long upto = before + warp_scan(mine.size);
    const unsigned hit = __ballot_sync(0xffffffffu, upto > w.begin);
    if (hit) {
      const int at = __ffs(hit) - 1;
      w.b = b0 + at;
      w.off = w.begin - __shfl_sync(0xffffffffu, upto - mine.size, at);
      w.size = __shfl_sync(0xffffffffu, mine.size, at);
      w.tiles = __shfl_sync(0xffffffffu, mine.tiles, at);
      w.blocks = __shfl_sync(0xffffffffu, mine.blocks, at);
      w.s.q0 = __shfl_sync(0xffffffffu, mine.s.q0, at);
      w.s.n = __shfl_sync(0xffffffffu, mine.s.n, at);
      w.s.k0 = 0;
      w.s.m = __shfl_sync(0xffffffffu, mine.s.m, at);
      w.s.sure = __shfl_sync(0xffffffffu, mine.s.sure, at);
      return true;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// Prompts: block `id` of the grid -> (sequence, head group, tile or tile
// pair), one warp; false past the last.  chunk_heads head groups of all
// sequences are taken together (their keys and values fit in L2 then), within
// them the tiles level by level from the last (the one with the most keys
// under a causal mask) to the first, so that the longest start earliest.
template <bool kPair>
struct SvPromptLine {
  SvSeq mine;   // sequence `lane`
  int levels;   // its tiles (tile pairs)
  int top;      // most tiles of any sequence
  int tiles;    // of a head group
  __device__ __forceinline__ int levels_of(const ServingArgs& a, const SvSeq& s) const {
    const int per = (kPair ? 2 : 1) * a.tile_tokens;
    return (s.n + per - 1) / per;
  }
  __device__ __forceinline__ int levels_at(const ServingArgs& a, int b) const {
    bool clamped;
    return b < a.batch ? levels_of(a, sv_sequence<false>(a, b, &clamped)) : 0;
  }
  __device__ __forceinline__ int at_least(const ServingArgs& a, int l) const {  // tiles of level l and above
    int c = max(levels - l, 0);
    for (int b0 = 32; b0 < a.batch; b0 += 32) c += max(levels_at(a, b0 + static_cast<int>(lane_id())) - l, 0);
    return __reduce_add_sync(0xffffffffu, c);
  }
  __device__ __forceinline__ void load(const ServingArgs& a) {
    const int b = static_cast<int>(lane_id());
    levels = 0;
    if (b < a.batch) {
      bool clamped;
      mine = sv_sequence<false>(a, b, &clamped);
      levels = levels_of(a, mine);
    }
    top = levels;
    for (int b0 = 32; b0 < a.batch; b0 += 32) top = max(top, levels_at(a, b0 + b));
    top = __reduce_max_sync(0xffffffffu, top);
    tiles = at_least(a, 0);
  }
  // (the grid has fewer than 2^31 blocks, so 32 bits hold every count)
  __device__ __forceinline__ bool find(const ServingArgs& a, uint32_t id, SvPiece& p) const {
    const uint32_t all = static_cast<uint32_t>(tiles);
    if (tiles == 0 || id / all >= static_cast<uint32_t>(a.head_groups)) return false;
    const uint32_t per = all * static_cast<uint32_t>(a.chunk_heads);  // of a chunk
    const uint32_t chunk = id / per, rem = id - chunk * per;
    const uint32_t heads = min(a.chunk_heads, a.head_groups - static_cast<int>(chunk) * a.chunk_heads);
    const int x = static_cast<int>(rem / heads);
    p.hk = static_cast<int>(chunk) * a.chunk_heads + static_cast<int>(rem - static_cast<uint32_t>(x) * heads);
    int lo = 0, hi = top - 1;  // the last level with more than x tiles at or above it
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (at_least(a, mid) > x) lo = mid;
      else hi = mid - 1;
    }
    p.tile = lo;
    int left = x - at_least(a, lo + 1);
    const uint32_t lane = lane_id();
    for (int b0 = 0; b0 < a.batch; b0 += 32) {
      SvSeq s = mine;
      int l = levels;
      if (b0 > 0) {
        l = 0;
        if (b0 + static_cast<int>(lane) < a.batch) {
          bool clamped;
          s = sv_sequence<false>(a, b0 + lane, &clamped);
          l = levels_of(a, s);
        }
      }
      const unsigned on = __ballot_sync(0xffffffffu, l > lo);
      const int c = __popc(on);
      if (left < c) {
        const unsigned hit = __ballot_sync(0xffffffffu, l > lo && __popc(on & ((1u << lane) - 1)) == left);
        const int at = __ffs(hit) - 1;
        p.b = b0 + at;
        p.s.q0 = __shfl_sync(0xffffffffu, s.q0, at);
        p.s.n = __shfl_sync(0xffffffffu, s.n, at);
        p.s.k0 = __shfl_sync(0xffffffffu, s.k0, at);
        p.s.m = __shfl_sync(0xffffffffu, s.m, at);
        p.s.sure = __shfl_sync(0xffffffffu, s.sure, at);
        return true;
      }
      left -= c;
    }
    return false;
  }
};

// ---------------------------------------------------------- shared memory --
template <int DP, bool kPair>
struct SvSmem {
  static constexpr int kQ = kSvRows * DP * 2;   // one row tile
  static constexpr int kKV = kSvKeys * DP * 2;  // one key or value block
  static constexpr int kStages = DP == 64 ? (kPair ? 5 : 6) : kPair ? 2 : 3;  // of each ring
  static constexpr int kKOff = (kPair ? 2 : 1) * kQ;
  static constexpr int kVOff = kKOff + kStages * kKV;
  // the two threads of a row exchange maxima and sums: [stream][half][row],
  // in the pair form in two alternating buffers
  static constexpr int kXBufs = kPair ? 2 : 1;
  static constexpr int kXOff = kVOff + kStages * kKV;
  static constexpr int kCtlOff = kXOff + kXBufs * 2 * 2 * kSvRows * 4;
  static constexpr int kBytes = kCtlOff + 1024;
  static_assert(kBytes <= 232448, "227 KB of shared memory per CTA");
};

// A piece as the scheduler hands it out.
struct SvTask {
  int q0, n, k0, m, sure;  // of the sequence
  int b, hk, tok0;         // sequence, head group, first token of the tile(s)
  int kb, loads;           // first key block, blocks loaded; loads < 0: no more work
  int blocks[2];           // blocks of each stream
  int part;
  int pad[3];
};
constexpr int kSvTasks = 4;

template <int kStages>
struct SvControl {
  uint64_t task_full[kSvTasks], task_empty[kSvTasks];
  uint64_t q_full[2], q_empty[2];  // pair form: of each tile; single form: the first
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], o_done[2];
  uint64_t p_part[4][2];
  uint64_t drain, cancel;
  uint4 cancelled;  // the answer to a request for a block that has not started
  uint32_t tmem;
  // a wait that gave up, for the threads that the next barrier joins: [pair of warps][parity], [quad][parity]
  volatile int pair_abort[8][2];
  volatile int quad_abort[4][2];
  SvTask task[kSvTasks];
};

template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float x, float y) { return pack_half2(x, y); }
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float x, float y) {
  __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Executed by the whole (converged) warp with warp-uniform operands; one
// elected lane issues.
__device__ __forceinline__ void tma_load_4d_warp(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y, int z,
                                                 int w) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, "
      "%6}], [%2];\n\t}" ::"r"(dst),
      "l"(m), "r"(bar), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}

// Ask for a block of this grid that has not started: its index, or that there
// is none, arrives in `answer` (16 bytes counted on `bar`).
__device__ __forceinline__ void request_block(uint4* answer, uint64_t* bar) {
  asm volatile(
      "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
          smem_u32(answer)),
      "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ bool answered_block(const uint4* answer, uint32_t* index) {
  uint32_t ok, x;
  asm volatile(
      "{\n\t.reg .b128 h;\n\t.reg .pred p;\n\t"
      "ld.shared.b128 h, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t"
      "mov.u32 %1, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %1, h;\n\t}"
      : "=r"(ok), "=r"(x)
      : "r"(smem_u32(answer))
      : "memory");
  *index = x;
  return ok != 0;
}

// Executed by the whole (converged) warp, as tma_load_4d_warp.
__device__ __forceinline__ void tma_load_3d_warp(uint32_t dst, const CUtensorMap* m, uint32_t bar, int x, int y,
                                                 int z) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], "
      "[%2];\n\t}" ::"r"(dst),
      "l"(m), "r"(bar), "r"(x), "r"(y), "r"(z)
      : "memory");
}

// 4 x 4 transpose of 16-byte units between four neighbouring lanes: lane i
// gives its unit j to lane j as unit i.
__device__ __forceinline__ void exchange_units(uint32_t (&u)[4][4]) {
  const uint32_t lane = lane_id();
#pragma unroll
  for (int b = 1; b <= 2; b <<= 1) {
    const bool upper = (lane & b) != 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (i & b) continue;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t send = upper ? u[i][w] : u[i | b][w];
        const uint32_t got = __shfl_xor_sync(0xffffffffu, send, b);
        if (upper) u[i][w] = got;
        else u[i | b][w] = got;
      }
    }
  }
}

// Bits [off, off + 64) of a mask row of `words` words; outside it 0.
__device__ __forceinline__ uint64_t mask_window(const unsigned int* row, int words, int off) {
  const int w = off >> 5, sh = off & 31;
  auto word = [&](int i) -> uint64_t { return i >= 0 && i < words ? row[i] : 0u; };
  uint64_t v = (word(w) | (word(w + 1) << 32)) >> sh;
  if (sh) v |= word(w + 2) << (64 - sh);
  return v;
}

// ----------------------------------------------------------------- kernel --
template <int DP, typename T, bool kPaged, bool kPair>
__global__ void __maxnreg__(96)
    serving_attention_kernel(const __grid_constant__ CUtensorMap tmQ, const __grid_constant__ CUtensorMap tmK,
                             const __grid_constant__ CUtensorMap tmV, const __grid_constant__ ServingArgs a) {
  using L = SvSmem<DP, kPair>;
  constexpr int kTileRows = (kPair ? 2 : 1) * kSvRows;
  constexpr int kStages = L::kStages;
  constexpr int kChunks = DP / 64;              // 64-column swizzle chunks
  constexpr int kParts = 2;                     // in which P is announced (4: 3% slower, 1: 5%)
  constexpr int kPSteps = 4 / kParts;           // P.V K-steps per part and half
  constexpr int kPPairs = 8 * kPSteps;          // packed P columns per part and half
  constexpr uint32_t kColO = 256;
  constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;

  extern __shared__ __align__(1024) uint8_t sv_smem[];
  uint8_t* smem = sv_smem;
  uint8_t* sQ = smem;
  uint8_t* sK = smem + L::kKOff;
  uint8_t* sV = smem + L::kVOff;
  float* xchg = reinterpret_cast<float*>(smem + L::kXOff);
  auto* ctl = reinterpret_cast<SvControl<kStages>*>(smem + L::kCtlOff);
  static_assert(sizeof(SvControl<kStages>) <= L::kBytes - L::kCtlOff, "control block");

  const uint32_t warp = warp_id();
  const uint32_t lane = lane_id();
  if (warp == 1) {
    tmem_alloc(&ctl->tmem, 512);
    tmem_relinquish();
  } else if (warp == 2 && lane == 0) {
    for (int i = 0; i < kSvTasks; ++i) {
      mbar_init(&ctl->task_full[i], 1);
      mbar_init(&ctl->task_empty[i], 19);  // every other warp
    }
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&ctl->k_full[s], 1);
      mbar_init(&ctl->k_empty[s], 1);
      mbar_init(&ctl->v_full[s], 1);
      mbar_init(&ctl->v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctl->q_full[t], 1);
      mbar_init(&ctl->q_empty[t], 1);
      mbar_init(&ctl->s_full[t], 1);
      mbar_init(&ctl->o_done[t], 1);
      for (int p = 0; p < kParts; ++p) mbar_init(&ctl->p_part[p][t], 8);  // one arrive per softmax warp
    }
    mbar_init(&ctl->drain, 1);
    mbar_init(&ctl->cancel, 1);
    for (int i = 0; i < 16; ++i) ctl->pair_abort[i >> 1][i & 1] = 0;
    for (int i = 0; i < 8; ++i) ctl->quad_abort[i >> 1][i & 1] = 0;
    fence_mbar_init();
  } else if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmQ);
    tma_prefetch_desc(&tmK);
    tma_prefetch_desc(&tmV);
  }
  // Nothing of an earlier kernel is read before it is complete; the join
  // kernel, whose blocks read the lengths as they start, may start after that.
  griddep_wait();
  if constexpr (kPaged) griddep_launch_dependents();
  // the scheduler finds its place meanwhile
  SvPromptLine<kPair> line;
  SvWalk<kTileRows> walk;
  bool more = true;
  [[maybe_unused]] long long quota = 1;
  if (warp == 19) {
    if constexpr (kPaged) {
      long long total;
      more = sv_share<kTileRows>(a, blockIdx.x, gridDim.x, walk, &quota, &total);
    } else {
      line.load(a);
    }
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;

  uint32_t n_task = 0;  // pieces taken so far
  auto wait_task = [&](uint64_t* full, uint32_t parity) { return mbar_wait(full, parity, kSiteProducerEmpty); };
  // The next piece for a worker warp; nullptr: no more work, or a wait gave up (*ok false).
  auto take_task = [&](bool* ok, auto wait) -> const SvTask* {
    const uint32_t slot = n_task % kSvTasks;
    *ok = __all_sync(0xffffffffu, wait(&ctl->task_full[slot], (n_task / kSvTasks) & 1));
    const SvTask* t = &ctl->task[slot];
    if (!*ok || t->loads < 0) return nullptr;
    ++n_task;
    return t;
  };
  // ... and done with it (its fields are not read again).
  auto drop_task = [&]() {
    __syncwarp();
    if (lane == 0) mbar_arrive(&ctl->task_empty[(n_task - 1) % kSvTasks]);
  };

  if (warp == 19) {
    // --------------------------------------------------------------- schedule
    bool ok = (smem_u32(smem) & 1023) == 0;
    uint32_t count = 0;            // pieces handed out
    uint32_t q_used[2] = {0, 0};   // loads of each Q tile
    uint32_t asked = 0;            // requests for further blocks
    uint32_t id = blockIdx.x;
    if constexpr (kPaged)
      if (lane == 0) a.cuts[2 * blockIdx.x].x = 0;
    while (ok) {
      SvPiece p;
      if constexpr (kPaged) {
        more = more && walk.next(a, blockIdx.x, p);
        if (more && p.part >= 0 && p.kb == 0 && lane == 0) {
          // starts here and is cut by the end of the share: for the join
          const long long last = (p.first + walk.blocks - 1) / quota;
          a.cuts[2 * blockIdx.x] = make_int4(static_cast<int>(last) - static_cast<int>(blockIdx.x) + 1, p.part, p.s.n,
                                             p.tile * (kTileRows / kSvRows) * a.tile_tokens);
          a.cuts[2 * blockIdx.x + 1] = make_int4(p.s.q0, p.hk, 0, 0);
        }
      } else {
        if (count > 0) {
          // the block that was asked for when the last piece was handed out
          ok = __all_sync(0xffffffffu, mbar_wait(&ctl->cancel, (asked - 1) & 1, kSiteProducerEmpty));
          if (!ok) break;
          more = answered_block(&ctl->cancelled, &id);
          fence_async_shared();  // read before the next answer is written
          __syncwarp();
        }
        p.kb = 0;
        p.part = -1;
        more = more && line.find(a, id, p);
        if (more) {
          if (lane == 0) {
            mbar_expect_tx(&ctl->cancel, 16);
            request_block(&ctl->cancelled, &ctl->cancel);
          }
          ++asked;
        }
      }
      const uint32_t slot = count % kSvTasks;
      if (count >= kSvTasks)
        ok = __all_sync(0xffffffffu, mbar_wait(&ctl->task_empty[slot], (count / kSvTasks - 1) & 1, kSiteProducerEmpty));
      if (!ok) break;
      SvTask* t = &ctl->task[slot];
      if (!more) {
        if (lane == 0) {
          t->loads = -1;
          mbar_arrive(&ctl->task_full[slot]);
        }
        break;
      }
      const int tok0 = p.tile * (kPair ? 2 : 1) * a.tile_tokens;
      int n[2], loads;
      if constexpr (kPair) {
        // blocks that some row of each tile sees
        const int ke = kPaged ? p.kb + p.loads : INT32_MAX;
        const bool chain = kPaged ? a.mask == nullptr : a.causal != 0;
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          const int first = tok0 + s * a.tile_tokens;
          int keys = 0;
          if (first < p.s.n)
            keys = chain ? max(min(p.s.m, p.s.sure + min(p.s.n, first + a.tile_tokens)), 0) : p.s.m;
          n[s] = max(min((keys + kSvKeys - 1) / kSvKeys, ke) - p.kb, 0);
        }
        loads = max(n[0], n[1]);
      } else {
        loads = p.loads;
        if constexpr (!kPaged) {
          const int keys = a.causal ? max(min(p.s.m, p.s.sure + min(p.s.n, tok0 + a.tile_tokens)), 0) : p.s.m;
          loads = (keys + kSvKeys - 1) / kSvKeys;
        }
        n[0] = (loads + 1) >> 1;
        n[1] = loads >> 1;
      }
      if (lane == 0) {
        t->q0 = p.s.q0;
        t->n = p.s.n;
        t->k0 = p.s.k0;
        t->m = p.s.m;
        t->sure = p.s.sure;
        t->b = p.b;
        t->hk = p.hk;
        t->tok0 = tok0;
        t->kb = p.kb;
        t->loads = loads;
        t->blocks[0] = n[0];
        t->blocks[1] = n[1];
        t->part = p.part;
        mbar_arrive(&ctl->task_full[slot]);
      }
      __syncwarp();
      ++count;
      // Q: tile_tokens x pack rows of each tile (the last rows of a tile that
      // pack does not divide, and rows past the sequence, are nobody's)
#pragma unroll
      for (int s = 0; s < (kPair ? 2 : 1); ++s) {
        if (!ok || (kPair ? n[s] : loads) == 0) continue;
        if (q_used[s] > 0)
          ok = __all_sync(0xffffffffu, mbar_wait(&ctl->q_empty[s], (q_used[s] - 1) & 1, kSiteFlashQ));
        if (!ok) continue;
        ++q_used[s];
        if (lane == 0) mbar_expect_tx(&ctl->q_full[s], a.tile_tokens * a.pack * 128 * kChunks);
        __syncwarp();
        for (int c = 0; c < kChunks; ++c)
          tma_load_3d_warp(smem_u32(sQ + s * L::kQ + c * 16384), &tmQ, smem_u32(&ctl->q_full[s]), c * 64,
                           p.hk * a.pack, p.s.q0 + tok0 + s * a.tile_tokens);
      }
    }
    // What was asked for arrives before the CTA ends; so do the Q tiles (the MMA
    // warp waits for them, or, if a wait gave up, this one does).
    if constexpr (!kPaged)
      if (!ok && asked > 0) mbar_wait(&ctl->cancel, (asked - 1) & 1, kSiteDrain);
    if (!ok)
      for (int s = 0; s < 2; ++s)
        if (q_used[s] > 0) mbar_wait(&ctl->q_full[s], (q_used[s] - 1) & 1, kSiteDrain);
    __syncwarp();
  } else if (warp == 0 || warp == 18) {
    // ------------------------------------------------------ key / value loads
    const bool is_v = warp == 18;
    const CUtensorMap* tm = is_v ? &tmV : &tmK;
    uint8_t* ring = is_v ? sV : sK;
    uint64_t* full = is_v ? ctl->v_full : ctl->k_full;
    uint64_t* empty = is_v ? ctl->v_empty : ctl->k_empty;
    int st = 0;
    uint32_t round = 0, issued = 0;
    bool ok = true;
    while (const SvTask* t = take_task(&ok, wait_task)) {
      const int loads = t->loads, kb = t->kb, m = t->m, k0 = t->k0, b = t->b;
      const int kv_head = t->hk / a.groups_per_kv;
      drop_task();
      const int* table = kPaged ? a.page_table + b * a.table_stride : nullptr;
      // lane x looks up the page of box x (box_rows keys), a block ahead
      auto lookup = [&](int j) -> int {
        int page = 0;
        if constexpr (kPaged) {
          const int in = static_cast<int>(lane) * a.box_rows;
          const int key = (kb + j) * kSvKeys + in;
          if (j < loads && in < kSvKeys && key < m) page = table[key / a.page_size];
        }
        return page;
      };
      int page = lookup(0), ahead = lookup(1);
      for (int j = 0; j < loads; ++j) {
        const int key0 = (kb + j) * kSvKeys;
        if (round > 0) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (round - 1) & 1, kSiteFlashFree));
        if (!ok) break;
        const uint32_t dst = smem_u32(ring + st * L::kKV), bar = smem_u32(&full[st]);
        if constexpr (kPaged) {
          const int boxes = (min(kSvKeys, m - key0) + a.box_rows - 1) / a.box_rows;
          if (page < 0 || page >= a.num_pages) {  // outside the tensor: TMA fills zeros
            record_bad_index();
            page = -1;
          }
          if (lane == 0) mbar_expect_tx(&full[st], static_cast<uint32_t>(boxes * a.box_rows * 128 * kChunks));
          __syncwarp();
          int in_page = key0 % a.page_size;
#pragma unroll 4
          for (int box = 0; box < boxes; ++box) {
            const int at = __shfl_sync(0xffffffffu, page, box);
#pragma unroll
            for (int c = 0; c < kChunks; ++c)
              tma_load_4d_warp(dst + c * 16384 + box * a.box_rows * 128, tm, bar, c * 64, in_page, kv_head, at);
            in_page += a.box_rows;
            if (in_page == a.page_size) in_page = 0;
          }
        } else {
          if (lane == 0) mbar_expect_tx(&full[st], L::kKV);
          __syncwarp();
#pragma unroll
          for (int c = 0; c < kChunks; ++c) tma_load_3d_warp(dst + c * 16384, tm, bar, c * 64, kv_head, k0 + key0);
        }
        ++issued;
        page = ahead;
        ahead = lookup(j + 2);
        if (++st == kStages) {
          st = 0;
          ++round;
        }
      }
      if (!ok) break;
    }
    if (!ok)  // a wait gave up: the loads in flight end before the CTA does
      for (uint32_t c = issued > kStages ? issued - kStages : 0; c < issued; ++c)
        mbar_wait(&full[c % kStages], (c / kStages) & 1, kSiteDrain);
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA
    // The whole warp runs the loop, converged; one elected lane issues.
    constexpr uint32_t idesc_s = make_idesc_f16(kSvRows, kSvKeys, false, false) | kFmt;
    constexpr uint32_t idesc_o = make_idesc_f16(kSvRows, DP, false, true) | kFmt;
    const uint64_t qd0 = make_sdesc(smem_u32(sQ), 16, 1024, kSw128);
    const uint64_t kd0 = make_sdesc(smem_u32(sK), 16, 1024, kSw128);
    const uint64_t vd0 = make_sdesc(smem_u32(sV), 16384, 1024, kSw128);
    uint32_t kc = 0, vc = 0;      // blocks taken from the rings
    uint32_t p_cnt[2] = {0, 0};   // P blocks taken of each stream
    uint32_t q_cnt[2] = {0, 0};
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
      ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, site));
    };
    // Values past the sequence's end may be anything: 0 times them must be 0.
    auto take_values = [&](int live) {
      const int st = vc % kStages;
      wait(&ctl->v_full[st], (vc / kStages) & 1, kSiteFlashKV);
      if (ok && live < kSvKeys) {
        const uint4 zero = {0, 0, 0, 0};
        for (int c = 0; c < kChunks; ++c)
          for (int x = live * 8 + static_cast<int>(lane); x < kSvKeys * 8; x += 32)
            *reinterpret_cast<uint4*>(sV + st * L::kKV + c * 16384 + x * 16) = zero;
        fence_async_shared();
        __syncwarp();
      }
    };
    // O_t += P_t . V, part by part as the softmax announces P
    auto issue_pv = [&](int t, bool fresh) {
      const uint64_t vd = vd0 + static_cast<uint64_t>(((vc % kStages) * L::kKV) >> 4);
      const uint32_t o_tmem = tmem + kColO + t * 128;
      const uint32_t p_tmem = tmem + t * 128;
#pragma unroll
      for (int p = 0; p < kParts; ++p) {
        wait(&ctl->p_part[p][t], p_cnt[t] & 1, kSiteFlashP);
        if (!ok) return;
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int q = 0; q < kPSteps; ++q) {
            const int k = 4 * h + p * kPSteps + q;
            umma_f16_ts_warp(o_tmem, p_tmem + k * 8, vd + static_cast<uint64_t>((k * 2048) >> 4), idesc_o,
                             !fresh || k != 0);
          }
      }
      ++p_cnt[t];
    };
    // S_t = Q . K^T
    auto issue_s = [&](int t) {
      tc_fence_after();
      const uint64_t qd = qd0 + static_cast<uint64_t>((kPair ? t * L::kQ : 0) >> 4);
      const uint64_t kd = kd0 + static_cast<uint64_t>(((kc % kStages) * L::kKV) >> 4);
#pragma unroll
      for (int k = 0; k < DP / 16; ++k) {
        const uint64_t off = static_cast<uint64_t>(((k >> 2) * 16384 + (k & 3) * 32) >> 4);
        umma_f16_ss_warp(tmem + t * 128, qd + off, kd + off, idesc_s, k != 0);
      }
      umma_commit_warp(&ctl->s_full[t]);
    };
    while (const SvTask* task = take_task(&ok, wait_task)) {
      const int loads = task->loads, n0 = task->blocks[0], n1 = task->blocks[1];
      const int tail = task->m - task->kb * kSvKeys;  // keys from this piece's first block on
      drop_task();
      if constexpr (kPair) {
        for (int j = 0; j <= loads && ok; ++j) {
          if (j < loads) wait(&ctl->k_full[kc % kStages], (kc / kStages) & 1, kSiteFlashKV);
          if (j >= 1) take_values(tail - (j - 1) * kSvKeys);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int n = t == 0 ? n0 : n1;
            if (ok && j >= 1 && j <= n) {
              issue_pv(t, j == 1);
              if (ok && j == n) umma_commit_warp(&ctl->o_done[t]);
            }
            if (ok && j < n) {
              if (j == 0) wait(&ctl->q_full[t], q_cnt[t]++ & 1, kSiteFlashQ);
              if (!ok) break;
              issue_s(t);
              if (j == n - 1) umma_commit_warp(&ctl->q_empty[t]);
            }
          }
          if (!ok) break;
          if (j < loads) {
            umma_commit_warp(&ctl->k_empty[kc % kStages]);
            ++kc;
          }
          if (j >= 1) {
            umma_commit_warp(&ctl->v_empty[vc % kStages]);
            ++vc;
          }
        }
      } else {
        if (loads == 0) continue;
        wait(&ctl->q_full[0], q_cnt[0]++ & 1, kSiteFlashQ);
        for (int j = 0; j < loads + 2 && ok; ++j) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if ((j & 1) != t) continue;
            if (j >= 2) {
              take_values(tail - (j - 2) * kSvKeys);
              if (ok) issue_pv(t, j == 2 + t);
              if (!ok) break;
              umma_commit_warp(&ctl->v_empty[vc % kStages]);
              ++vc;
              if (j >= loads) umma_commit_warp(&ctl->o_done[t]);
            }
            if (j < loads) {
              wait(&ctl->k_full[kc % kStages], (kc / kStages) & 1, kSiteFlashKV);
              if (!ok) break;
              issue_s(t);
              umma_commit_warp(&ctl->k_empty[kc % kStages]);
              if (j == loads - 1) umma_commit_warp(&ctl->q_empty[0]);
              ++kc;
            }
          }
        }
      }
      if (!ok) break;
    }
    umma_commit_warp(&ctl->drain);
    mbar_wait(&ctl->drain, 0, kSiteDrain);
    __syncwarp();
  } else {
    // --------------------------------------------------- softmax / output
    const int grp = (static_cast<int>(warp) - 2) >> 3;        // stream
    const int half = ((static_cast<int>(warp) - 2) >> 2) & 1;  // of a block's scores
    const int wq = static_cast<int>(warp & 3);                 // TMEM lane quarter
    const int r = wq * 32 + static_cast<int>(lane);            // row of the tile
    const int row_tok = r / a.pack;                            // its token and head within the tile
    const int row_head = r - row_tok * a.pack;
    const int pair_id = grp * 4 + wq;
    const uint32_t pair_bar = 1 + pair_id;  // 64 threads: both halves of these rows
    const uint32_t quad_bar = 9 + wq;       // 128 threads: both halves, both streams
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tS = tmem + lane_off + grp * 128 + half * 64;
    const uint32_t tP = tmem + lane_off + grp * 128 + half * 32;
    const float sl = a.scale_log2;
    uint32_t events = 0;  // barriers of the pair so far, the parity of its abort flags
    uint32_t s_cnt = 0;   // blocks of this stream so far
    uint32_t o_cnt[2] = {0, 0};
    bool alive = true;
    auto swap_slot = [&](uint32_t ev) {
      return xchg + ((L::kXBufs == 2 ? (ev & 1) * 2 : 0) + grp) * (2 * kSvRows);
    };
    // (the warps that meet at barriers go on or end together)
    auto wait_task_together = [&](uint64_t* full, uint32_t parity) {
      return mbar_wait_together<kPair ? 64 : 128>(full, parity, kSiteProducerEmpty, kPair ? pair_bar : quad_bar,
                                                  kWaitTimeoutNs);
    };
    bool ok = true;
    while (const SvTask* task = take_task(&ok, wait_task_together)) {
      const uint32_t piece_parity = n_task & 1;
      // ---- this piece's row
      const int tok = task->tok0 + (kPair ? grp * a.tile_tokens : 0) + row_tok;
      const bool live = row_tok < a.tile_tokens && tok < task->n;
      const bool tree = kPaged && a.mask != nullptr;
      int sees = task->m;  // keys 0 .. sees - 1 are visible (and the nodes of the mask row)
      if (tree) sees = task->sure;
      else if (kPaged || a.causal) sees = min(task->m, task->sure + tok + 1);
      if (!live) sees = 0;
      float m_use = -INFINITY;  // running maximum, exact to the rescale threshold
      float l = 0.0f;           // this half's share of the row sum
      const int nblk = task->blocks[grp];
      const int kv_first = task->kb * kSvKeys + (kPair ? 0 : grp * kSvKeys) + half * 64;
      const bool warp_live = __any_sync(0xffffffffu, live);
      for (int i = 0; i < nblk; ++i, ++s_cnt, ++events) {
        if (!mbar_wait(&ctl->s_full[grp], s_cnt & 1, kSiteFlashS)) ctl->pair_abort[pair_id][events & 1] = 1;
        if (!warp_live) {
          // no row here: nothing reads these lanes of P
          vote_barrier<64>(pair_bar, false);
          if (ctl->pair_abort[pair_id][events & 1]) {
            alive = false;
            break;
          }
          if (lane == 0)
            for (int p = 0; p < kParts; ++p) mbar_arrive(&ctl->p_part[p][grp]);
          continue;
        }
        tc_fence_after();
        const int kv0 = kv_first + i * (kPair ? kSvKeys : 2 * kSvKeys);
        float s[64];
        tmem_ld64(tS, s);
        float mx[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) mx[x] = -INFINITY;
        if (sees - kv0 >= 64) {
#pragma unroll
          for (int x = 0; x < 32; ++x) mx[x & 7] = fmax3(mx[x & 7], s[2 * x], s[2 * x + 1]);
        } else {
          const int nv = sees - kv0;
          uint64_t vis = nv <= 0 ? 0ull : (1ull << nv) - 1;
          if (tree && live) {
            const int node = kv0 - task->sure;  // of this half's first key
            const int nodes = task->m - task->sure;
            if (node > -64 && node < nodes) {
              uint64_t bits = mask_window(a.mask + (task->q0 + tok) * a.mask_stride, a.mask_words, node);
              if (nodes - node < 64) bits &= (1ull << (nodes - node)) - 1;
              vis |= bits;
            }
          }
#pragma unroll
          for (int x = 0; x < 64; ++x) {
            if (!((vis >> x) & 1)) s[x] = -INFINITY;
            mx[x & 7] = fmaxf(mx[x & 7], s[x]);
          }
        }
        const float pmax = fmaxf(fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])),
                                 fmaxf(fmaxf(mx[4], mx[5]), fmaxf(mx[6], mx[7])));
        // One vote of the two warps (which also orders both halves' S loads
        // before either's P stores); the maxima are exchanged only when some
        // row's grows.
        tc_fence_before();
        const bool any_grow = vote_barrier<64>(pair_bar, sl * pmax > m_use + 8.0f);
        tc_fence_after();
        if (ctl->pair_abort[pair_id][events & 1]) {
          alive = false;
          break;
        }
        bool grow = false;
        float m_new = m_use;
        if (any_grow) {
          float* xs = swap_slot(events);
          xs[half * kSvRows + r] = pmax;
          named_bar_sync(pair_bar, 64);
          const float rmax = sl * fmaxf(pmax, xs[(half ^ 1) * kSvRows + r]);
          if constexpr (L::kXBufs == 1) named_bar_sync(pair_bar, 64);
          grow = rmax > m_use + 8.0f;
          if (grow) m_new = rmax;
        }
        const float alpha = grow ? exp2f(m_use - m_new) : 1.0f;  // 0 on the first block with a visible key
        if (i > 0 && __any_sync(0xffffffffu, grow)) {
          const uint32_t tO = tmem + lane_off + kColO + grp * 128 + half * (DP / 2);
#pragma unroll 1
          for (int c = 0; c < DP / 16; ++c) {
            uint32_t o[8];
            tmem_ld8(tO + c * 8, o);
#pragma unroll
            for (int x = 0; x < 8; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
            tmem_st8(tO + c * 8, o);
          }
        }
        // a row that has seen nothing yet: every score is -inf, every weight 0
        const float m_sub = m_new == -INFINITY ? 0.0f : m_new;
        const uint64_t sl2 = f2_pack(sl, sl);
        const uint64_t nm2 = f2_pack(-m_sub, -m_sub);
        uint64_t sm2[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) sm2[x] = 0ull;
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          uint32_t pk[kPPairs];
#pragma unroll
          for (int y = 0; y < kPPairs; ++y) {
            const int x = p * kPPairs + y;
            float x0, x1;
            f2_unpack(f2_fma(f2_pack(s[2 * x], s[2 * x + 1]), sl2, nm2), x0, x1);
            const float p0 = ex2_mufu(x0), p1 = ex2_mufu(x1);
            sm2[x & 3] = f2_add(sm2[x & 3], f2_pack(p0, p1));
            // (rounded to the element type: a 16-bit product takes 16-bit operands; the sums keep fp32)
            pk[y] = pack2<T>(p0, p1);
          }
          tmem_st_p(tP + p * kPPairs, pk);
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&ctl->p_part[p][grp]);
        }
        float sv[8];
#pragma unroll
        for (int x = 0; x < 4; ++x) f2_unpack(sm2[x], sv[2 * x], sv[2 * x + 1]);
        l = l * alpha + (((sv[0] + sv[1]) + (sv[2] + sv[3])) + ((sv[4] + sv[5]) + (sv[6] + sv[7])));
        m_use = m_new;
      }
      // ---- output.  With the pair form each half of a stream has half of
      // the row's columns; with the single form the row's four threads have a
      // quarter each, of the sum of both streams.
      if (kPair && !alive) break;
      float w0, w1 = 0.0f;  // of O_0 and O_1 (pair form: w0 of this stream's)
      float l_row, m_row;
      const int part = task->part;
      const bool whole = !kPaged || part < 0;
      if constexpr (kPair) {
        float* xs = swap_slot(events);
        xs[half * kSvRows + r] = l;
        if (nblk > 0 && !mbar_wait(&ctl->o_done[grp], o_cnt[grp] & 1, kSiteFlashPV))
          ctl->pair_abort[pair_id][events & 1] = 1;
        if (nblk > 0) ++o_cnt[grp];
        named_bar_sync(pair_bar, 64);
        l_row = l + xs[(half ^ 1) * kSvRows + r];
        if (ctl->pair_abort[pair_id][events & 1]) {
          alive = false;
          break;
        }
        ++events;
        m_row = m_use;
        w0 = !whole ? 1.0f : l_row != 0.0f ? 1.0f / l_row : 0.0f;
        if (nblk == 0) w0 = 0.0f;
      } else {
        if (!alive) ctl->quad_abort[wq][piece_parity] = 1;
        // both streams of this row: m and the two halves' sums
        float* xs = xchg;
        for (int t = 0; t < 2; ++t) {
          const int n = task->blocks[t];
          if (n > 0 && !mbar_wait(&ctl->o_done[t], o_cnt[t] & 1, kSiteFlashPV)) ctl->quad_abort[wq][piece_parity] = 1;
          if (n > 0) ++o_cnt[t];
        }
        named_bar_sync(quad_bar, 128);  // the last block's exchange has been read
        xs[(grp * 2 + half) * kSvRows + r] = l;
        named_bar_sync(quad_bar, 128);
        const float l0 = xs[0 * kSvRows + r] + xs[1 * kSvRows + r];
        const float l1 = xs[2 * kSvRows + r] + xs[3 * kSvRows + r];
        named_bar_sync(quad_bar, 128);
        if (half == 0) xs[grp * kSvRows + r] = m_use;
        named_bar_sync(quad_bar, 128);
        const float m0 = xs[0 * kSvRows + r], m1 = xs[1 * kSvRows + r];
        named_bar_sync(quad_bar, 128);
        if (ctl->quad_abort[wq][piece_parity]) {
          alive = false;
          break;
        }
        m_row = fmaxf(m0, m1);
        const float m_sub = m_row == -INFINITY ? 0.0f : m_row;
        w0 = exp2f(m0 - m_sub);  // 0 for a stream that saw nothing
        w1 = exp2f(m1 - m_sub);
        l_row = l0 * w0 + l1 * w1;
        if (whole) {
          const float inv = l_row != 0.0f ? 1.0f / l_row : 0.0f;
          w0 *= inv;
          w1 *= inv;
        }
      }
      tc_fence_after();
      if (warp_live) {
        constexpr int kCols = kPair ? DP / 2 : DP / 4;
        const int c0 = kPair ? half * kCols : (2 * grp + half) * kCols;
        const bool on0 = task->blocks[kPair ? grp : 0] > 0;
        const bool on1 = !kPair && task->blocks[1] > 0;
        const int head = task->hk * a.pack + row_head;
        const long long qrow = task->q0 + tok;
        // parts: [unit of 4 columns][row][4], m, l
        const int prow = (kPair ? grp * kSvRows : 0) + r;
        float* slot = whole ? nullptr : a.parts + static_cast<size_t>(part) * kTileRows * (DP + 2);
        // the rows of this lane's four neighbours, for which it stores one unit of each
        T* out[4];
        bool put[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const long long to = __shfl_sync(0xffffffffu, qrow * a.o_st[0] + head * a.o_st[1], (lane & ~3u) + x);
          put[x] = __shfl_sync(0xffffffffu, static_cast<int>(live), (lane & ~3u) + x) != 0;
          out[x] = static_cast<T*>(a.o) + to;
        }
        constexpr int kStep = 32 < kCols ? 32 : kCols;  // 32 or 16 columns at a time
#pragma unroll 1
        for (int c = c0; c < c0 + kCols; c += kStep) {
          float o[kStep];
#pragma unroll
          for (int x = 0; x < kStep; ++x) o[x] = 0.0f;
          if (on0) {
            const uint32_t src = tmem + lane_off + kColO + (kPair ? grp : 0) * 128 + c;
#pragma unroll
            for (int x = 0; x < kStep; x += 8) {
              uint32_t e[8];
              tmem_ld8(src + x, e);
#pragma unroll
              for (int y = 0; y < 8; ++y) o[x + y] = w0 != 0.0f ? w0 * __uint_as_float(e[y]) : 0.0f;
            }
          }
          if (on1) {
            const uint32_t src = tmem + lane_off + kColO + 128 + c;
#pragma unroll
            for (int x = 0; x < kStep; x += 8) {
              uint32_t e[8];
              tmem_ld8(src + x, e);
#pragma unroll
              for (int y = 0; y < 8; ++y) o[x + y] += w1 != 0.0f ? w1 * __uint_as_float(e[y]) : 0.0f;
            }
          }
          if (slot != nullptr) {
            if (live)
#pragma unroll
              for (int x = 0; x < kStep; x += 4)
                *reinterpret_cast<float4*>(slot + (static_cast<size_t>((c + x) / 4) * kTileRows + prow) * 4) =
                    make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
          } else {
            uint32_t u[4][4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
              for (int w = 0; w < 4; ++w)
                u[x][w] = x * 8 < kStep ? pack2<T>(o[(x * 8 + 2 * w) % kStep], o[(x * 8 + 2 * w + 1) % kStep]) : 0u;
            exchange_units(u);
            // u[x] is now unit lane & 3 of neighbour x's row: 64 bytes in a row per four lanes
            const int col = c + static_cast<int>(lane & 3) * 8;
            const bool in = static_cast<int>(lane & 3) * 8 < kStep && col < a.head_dim;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if (in && put[x])
                *reinterpret_cast<uint4*>(out[x] + col) = make_uint4(u[x][0], u[x][1], u[x][2], u[x][3]);
          }
        }
        if (live && half == 0 && (kPair || grp == 0)) {
          if (slot != nullptr) {
            slot[static_cast<size_t>(kTileRows) * DP + prow] = m_row;
            slot[static_cast<size_t>(kTileRows) * (DP + 1) + prow] = l_row;
          } else if (a.lse != nullptr) {
            a.lse[qrow * a.q_heads + head] = (m_row + log2f(l_row)) * 0.6931471805599453f;
          }
        }
      }
      tc_fence_before();  // O has been read before the next P is announced,
      if constexpr (!kPair) named_bar_sync(quad_bar, 128);  // by the other stream's warps too
      drop_task();
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds up the parts of the item that starts in share c = blockIdx.x and goes
// on past its end, in order.
//   m = max m_p,  o = sum 2^(m_p - m) O_p / sum 2^(m_p - m) l_p
// Few-row form, whose parts lie row by row: a warp per row.  (Its blocks find
// their cut item while the parts are still being computed.)
template <int DP, typename T, int kTileRows>
__global__ void __launch_bounds__(kSvJoinThreads) attention_join_kernel(const __grid_constant__ ServingArgs a) {
  __shared__ int from, parts, slot0, first, tokens, q0, hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    SvWalk<kTileRows> w;
    long long quota, total;
    const bool work = sv_share<kTileRows>(a, blockIdx.x, gridDim.x, w, &quota, &total);
    if (lane == 0) {
      parts = 0;
      SvPiece p;
      while (work && w.next(a, blockIdx.x, p)) {
        if (p.part < 0 || p.kb != 0) continue;  // whole, or the end of an earlier share's item
        // starts here and is cut by the end of the share
        const long long last = (p.first + w.blocks - 1) / quota;
        from = blockIdx.x;
        parts = static_cast<int>(last) - blockIdx.x + 1;
        slot0 = p.part;
        first = p.tile * kTileRows;
        tokens = p.s.n;
        q0 = p.s.q0;
        hk = p.hk;
      }
    }
  }
  __syncthreads();
  griddep_wait();  // the parts
  griddep_launch_dependents();
  if (parts == 0) return;
  constexpr size_t kSlot = static_cast<size_t>(kTileRows) * (DP + 2);
  auto part = [&](int i) { return a.parts + (i == 0 ? slot0 : 2 * (from + i)) * kSlot; };
  constexpr size_t kM = static_cast<size_t>(kTileRows) * DP, kL = static_cast<size_t>(kTileRows) * (DP + 1);
  // row r of the item -> its token and head within the group; false if it is nobody's
  auto row_of = [&](int r, int* tok, int* head) {
    const int row = first + r;
    *tok = row / a.group;
    *head = row - *tok * a.group;
    return *tok < tokens;
  };
  // Eight parts at a time, all of whose loads are under way together.
  auto join_row = [&](int r, int unit0, int unit_step) {
    int tok, head;
    if (!row_of(r, &tok, &head)) return;
    const long long qrow = q0 + tok;
    const int qh = hk * a.group + head;
    for (int unit = unit0; unit * 4 < a.head_dim; unit += unit_step) {
      float o[4] = {}, m = -INFINITY, l = 0.0f;
      for (int i0 = 0; i0 < parts; i0 += 8) {
        float pm[8], pl[8];
        float4 pv[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const bool on = i0 + i < parts;
          const float* p = part(on ? i0 + i : i0);
          pm[i] = on ? p[kM + r] : -INFINITY;
          pl[i] = p[kL + r];
          pv[i] = *reinterpret_cast<const float4*>(p + static_cast<size_t>(r) * DP + unit * 4);
        }
        float top = m;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, pm[i]);
        const float sub = top == -INFINITY ? 0.0f : top;
        const float keep = exp2f(m - sub);
        m = top;
        l *= keep;
#pragma unroll
        for (int x = 0; x < 4; ++x) o[x] *= keep;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float w = exp2f(pm[i] - sub);
          if (w != 0.0f) {  // (a part that saw nothing of the row holds anything)
            l += w * pl[i];
            o[0] += w * pv[i].x;
            o[1] += w * pv[i].y;
            o[2] += w * pv[i].z;
            o[3] += w * pv[i].w;
          }
        }
      }
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
      uint2 v;
      v.x = pack2<T>(o[0] * inv, o[1] * inv);
      v.y = pack2<T>(o[2] * inv, o[3] * inv);
      *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + qrow * a.o_st[0] + qh * a.o_st[1] + unit * 4) = v;
      if (a.lse != nullptr && unit == 0) a.lse[qrow * a.q_heads + qh] = (m + log2f(l)) * 0.6931471805599453f;
    }
  };
  for (int r = blockIdx.y * (kSvJoinThreads / 32) + warp; r < kTileRows; r += gridDim.y * (kSvJoinThreads / 32))
    join_row(r, lane, 32);
}

// The same for the row forms, whose parts lie by four columns, rows along the
// lanes: a thread per (row, 16 columns).  No register of an SM is free for
// these blocks before its CTA of the attention ends, so they do not look for
// their item but read it from `cuts`.  Nearly all items are cut once or twice:
// the loads of two parts (or of four, half the columns at a time) are under
// way together.  The join of 16 drafted trees (275 parts of up to 133 KB) takes
// 10.8 us alone; eight parts at a time, four columns a thread, took 21.
template <int DP, typename T, int kTileRows>
__global__ void __launch_bounds__(kSvJoinThreads) attention_join_rows_kernel(const __grid_constant__ ServingArgs a) {
  griddep_wait();  // the parts
  griddep_launch_dependents();
  const int4 cut = a.cuts[2 * blockIdx.x];
  const int parts = cut.x;
  if (parts == 0) return;
  const int4 seq = a.cuts[2 * blockIdx.x + 1];
  constexpr size_t kSlot = static_cast<size_t>(kTileRows) * (DP + 2);
  constexpr size_t kM = static_cast<size_t>(kTileRows) * DP, kL = static_cast<size_t>(kTileRows) * (DP + 1);
  constexpr int kPer = kSvJoinThreads / kTileRows;  // threads of a row within a block
  const int r = threadIdx.x % kTileRows;
  const int c0 = (blockIdx.y * kPer + threadIdx.x / kTileRows) * 16;
  const int in = r % kSvRows, t = in / a.pack;
  const int tok = cut.w + r / kSvRows * a.tile_tokens + t;
  if (t >= a.tile_tokens || tok >= cut.z || c0 >= a.head_dim) return;
  const long long qrow = seq.x + tok;
  const int qh = seq.y * a.pack + in - t * a.pack;
  auto part = [&](int i) { return a.parts + (i == 0 ? cut.y : 2 * (static_cast<int>(blockIdx.x) + i)) * kSlot; };
  T* out = static_cast<T*>(a.o) + qrow * a.o_st[0] + qh * a.o_st[1];
  float m = -INFINITY;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) m = fmaxf(m, part(i)[kM + r]);
  const float sub = m == -INFINITY ? 0.0f : m;
  // kBatch parts and 8 / kBatch units of four columns at a time
  auto join = [&](auto batch) {
    constexpr int kBatch = decltype(batch)::value, kUnits = 8 / kBatch;
#pragma unroll 1
    for (int c = c0; c < c0 + 16 && c < a.head_dim; c += 4 * kUnits) {
      float o[4 * kUnits] = {}, l = 0.0f;
#pragma unroll 1
      for (int i0 = 0; i0 < parts; i0 += kBatch) {
        float pm[kBatch], pl[kBatch];
        float4 pv[kBatch][kUnits];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const bool on = i0 + i < parts;
          const float* p = part(on ? i0 + i : i0);
          pm[i] = on ? p[kM + r] : -INFINITY;
          pl[i] = p[kL + r];
#pragma unroll
          for (int u = 0; u < kUnits; ++u)
            pv[i][u] = *reinterpret_cast<const float4*>(p + (static_cast<size_t>(c / 4 + u) * kTileRows + r) * 4);
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          const float w = exp2f(pm[i] - sub);
          if (w != 0.0f) {  // (a part that saw nothing of the row holds anything)
            l += w * pl[i];
#pragma unroll
            for (int u = 0; u < kUnits; ++u) {
              o[4 * u] += w * pv[i][u].x;
              o[4 * u + 1] += w * pv[i][u].y;
              o[4 * u + 2] += w * pv[i][u].z;
              o[4 * u + 3] += w * pv[i][u].w;
            }
          }
        }
      }
      const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
      for (int u = 0; u < kUnits; u += 2) {
        if (c + 4 * u >= a.head_dim) continue;
        uint4 v;
        v.x = pack2<T>(o[4 * u] * inv, o[4 * u + 1] * inv);
        v.y = pack2<T>(o[4 * u + 2] * inv, o[4 * u + 3] * inv);
        v.z = pack2<T>(o[4 * u + 4] * inv, o[4 * u + 5] * inv);
        v.w = pack2<T>(o[4 * u + 6] * inv, o[4 * u + 7] * inv);
        *reinterpret_cast<uint4*>(out + c + 4 * u) = v;
      }
      if (a.lse != nullptr && c == 0) a.lse[qrow * a.q_heads + qh] = (m + log2f(l)) * 0.6931471805599453f;
    }
  };
  if (parts == 2) join(std::integral_constant<int, 2>{});
  else join(std::integral_constant<int, 4>{});
}

}  // namespace akili
