// serving_attention.cuh — attention of packed queries over packed keys
// (prompts) or over a paged cache (new tokens, drafted trees), on tcgen05:
//
//   o_i = sum_j softmax_j(scale q_i.k_j) v_j   over the keys j that i sees
//
// Rows.  The G = q_heads / kv_heads query heads of a key head share its keys,
// so the rows of a (sequence, key head) are its tokens times G: row r is
// token r / G, head r % G of the group.  Short sequences and single tokens
// fill the 128-row tiles of the tensor core that way, keys are loaded once
// for the group, and a causal tile spans few tokens, so that its diagonal
// wastes little.
//
// One CTA per SM, 576 threads, two streams of scores, each with its own S/P
// and O accumulators in tensor memory (S_t and P_t at columns 128 t, O_t at
// 256 + 128 t), so that the tensor core works on one stream while the
// softmax of the other runs:
//   pair form   stream t is the 128-row tile t of 256 rows; both read every
//               key block.  For prompts and large trees.
//   single form both streams are the same 128 rows, stream t reads the key
//               blocks of parity t, and the two are merged at the end.  For
//               single tokens and small trees, which are bound by reading the
//               cache.
// Warps:
//   warp 0       TMA: key and value blocks of 128 keys into two rings, by one
//                box per block (packed) or one per page part (paged).
//   warp 1       TMEM owner and MMA issuer: per step O_t += P_t V of the
//                stream's previous block, then S_t = Q_t K^T of its next one
//                (over the columns of that P_t; the MMAs run in order).
//   warps 2..9   softmax of stream 0, warps 10..17 of stream 1: two threads
//                per row with 64 of a block's 128 scores each.  They swap
//                their block maxima through shared memory behind a barrier of
//                their two warps, keep the running maximum (rescaling O_t in
//                TMEM only when it grows by more than 2^8: a stale maximum
//                cancels in O / l) and write P = exp2(scale log2e s - m) over
//                S_t in parts, each announced to the MMA warp on its own.
//
// Work.  Prompts: one CTA per (256 rows, key head), the tiles with the most
// keys first.  Cache: the key blocks of all (sequence, key head, row tile)
// items form one line that is cut into equal shares, one per CTA, so uneven
// lengths and few long sequences fill the GPU alike; an item that is cut
// leaves its parts (O, m, l in fp32) in the workspace and
// attention_join_kernel adds them up in order.
#pragma once
#include <type_traits>

#include "cache.cuh"
#include "flash.cuh"
#include "rope.cuh"
#include "sm100.cuh"

namespace akili {

constexpr int kSvRows = 128;  // rows of a tile
constexpr int kSvKeys = 128;  // keys of a block
constexpr int kSvThreads = 64 + 512;
constexpr int kSvJoinThreads = 256;
constexpr int kSvJoinSplit = 4;  // blocks that share the rows of a cut item

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
  int q_heads, kv_heads, group, head_dim, batch, total_q, total_k, causal;
  int num_pages, page_size, max_pages, mask_words;
  int box_rows;     // paged keys: rows of a TMA box, a divisor of page_size
  int chunk_heads;  // packed keys: key heads that are scheduled together
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

// A run of key blocks of one (sequence, key head, row tile).
struct SvPiece {
  SvSeq s;
  int b, hk;
  int row0, rows;  // first row of the tile(s), rows of the (sequence, key head)
  int kb;          // first key block
  int n[2];        // blocks of each stream
  int loads;       // blocks loaded
  int part;        // slot of the workspace, or -1: the whole item
};

// Keys that some row of [row0, row0 + 128) may see.
template <bool kPaged>
__device__ __forceinline__ int sv_key_end(const ServingArgs& a, const SvSeq& s, int row0, int rows) {
  if (row0 >= rows) return 0;
  const bool chain = kPaged ? a.mask == nullptr : a.causal != 0;
  if (!chain) return s.m;
  const int last = (min(rows, row0 + kSvRows) - 1) / a.group;
  return max(min(s.m, s.sure + last + 1), 0);
}

template <bool kPaged, bool kPair>
__device__ __forceinline__ void sv_streams(const ServingArgs& a, SvPiece& p, int ke) {
  if constexpr (kPair) {
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int end = (sv_key_end<kPaged>(a, p.s, p.row0 + t * kSvRows, p.rows) + kSvKeys - 1) / kSvKeys;
      p.n[t] = max(min(end, ke) - p.kb, 0);
    }
    p.loads = max(p.n[0], p.n[1]);
  } else {
    p.loads = ke - p.kb;
    p.n[0] = (p.loads + 1) >> 1;
    p.n[1] = p.loads >> 1;
  }
}

// A CTA's share of the line of key blocks; every role walks it by itself.
// kTileRows: rows of an item (16 to 256).
template <int kTileRows>
struct SvWalk {
  long long pos, begin, end, off;  // off: position within sequence b
  int b;
  SvSeq s;
  int rows, tiles, blocks;
  long long size;

  __device__ __forceinline__ void load(const ServingArgs& a) {
    bool clamped;
    s = sv_sequence<true>(a, b, &clamped);
    rows = s.n * a.group;
    tiles = (rows + kTileRows - 1) / kTileRows;
    blocks = (s.m + kSvKeys - 1) / kSvKeys;
    size = static_cast<long long>(a.kv_heads) * tiles * blocks;
  }
  __device__ __forceinline__ bool next(const ServingArgs& a, int cta, SvPiece& p) {
    if (pos >= end) return false;
    while (off >= size) {
      off -= size;
      if (++b >= a.batch) return false;
      load(a);
    }
    const long long item = off / blocks;
    const int kb = static_cast<int>(off - item * blocks);
    const int take = static_cast<int>(min(static_cast<long long>(blocks - kb), end - pos));
    p.s = s;
    p.b = b;
    p.hk = static_cast<int>(item / tiles);
    p.row0 = static_cast<int>(item - static_cast<long long>(p.hk) * tiles) * kTileRows;
    p.rows = rows;
    p.kb = kb;
    p.part = take == blocks ? -1 : 2 * cta + (pos == begin ? 0 : 1);
    sv_streams<true, kTileRows == 2 * kSvRows>(a, p, kb + take);
    pos += take;
    off += take;
    return true;
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

// Blocks of sequence b on the line (0 past the batch).
template <int kTileRows>
__device__ __forceinline__ long long sv_line_blocks(const ServingArgs& a, int b, bool record) {
  if (b >= a.batch) return 0;
  SvWalk<kTileRows> w;
  w.b = b;
  w.load(a);
  if (record) {
    bool clamped;
    sv_sequence<true>(a, b, &clamped);
    if (clamped) record_bad_index();
  }
  return w.size;
}

// The share of CTA `cta` of `ctas` (one warp): false if it is empty.
template <int kTileRows>
__device__ __forceinline__ bool sv_share(const ServingArgs& a, int cta, int ctas, SvWalk<kTileRows>& w,
                                         long long* quota_out, long long* total_out) {
  const int lane = threadIdx.x & 31;
  long long total = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) total += sv_line_blocks<kTileRows>(a, b0 + lane, cta == 0);
  total = warp_sum(total);
  const long long quota = (total + ctas - 1) / ctas;
  *quota_out = quota;
  *total_out = total;
  w.begin = w.pos = cta * quota;
  w.end = min(w.begin + quota, total);
  if (w.begin >= total) return false;
  long long before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const long long mine = sv_line_blocks<kTileRows>(a, b0 + lane, false);
    const long long upto = before + warp_scan(mine);
    const unsigned hit = __ballot_sync(0xffffffffu, upto > w.begin);
    if (hit) {
      const int at = __ffs(hit) - 1;
      w.b = b0 + at;
      w.off = w.begin - __shfl_sync(0xffffffffu, upto - mine, at);
      w.load(a);
      return true;
    }
    before = __shfl_sync(0xffffffffu, upto, 31);
  }
  return false;
}

// Prompts: block `id` of the grid -> (sequence, key head, 256-row tile), one
// warp; false past the last.  chunk_heads key heads of all sequences are taken
// together (their keys and values fit in L2 then), within them the tiles
// level by level from the last (the one with the most keys under a causal
// mask) to the first, so that the longest start earliest.
__device__ __forceinline__ int sv_levels(const ServingArgs& a, int b) {
  if (b >= a.batch) return 0;
  bool clamped;
  return (sv_sequence<false>(a, b, &clamped).n * a.group + 2 * kSvRows - 1) / (2 * kSvRows);
}
__device__ __forceinline__ bool sv_prompt_tile(const ServingArgs& a, long long id, int* b_out, int* hk, int* level) {
  const int lane = threadIdx.x & 31;
  auto at_least = [&](int l) {  // tiles of level l and above
    long long c = 0;
    for (int b0 = 0; b0 < a.batch; b0 += 32) c += max(sv_levels(a, b0 + lane) - l, 0);
    return warp_sum(c);
  };
  int top = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 32) top = max(top, sv_levels(a, b0 + lane));
  top = __reduce_max_sync(0xffffffffu, top);
  const long long tiles = at_least(0);
  if (id >= tiles * a.kv_heads) return false;
  const long long chunk = id / (tiles * a.chunk_heads);
  const long long rem = id - chunk * tiles * a.chunk_heads;
  const int heads = min(a.chunk_heads, a.kv_heads - static_cast<int>(chunk) * a.chunk_heads);
  const long long x = rem / heads;
  *hk = static_cast<int>(chunk) * a.chunk_heads + static_cast<int>(rem - x * heads);
  int lo = 0, hi = top - 1;  // the last level with more than x tiles at or above it
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (at_least(mid) > x) lo = mid;
    else hi = mid - 1;
  }
  *level = lo;
  long long left = x - at_least(lo + 1);
  for (int b0 = 0; b0 < a.batch; b0 += 32) {
    const unsigned on = __ballot_sync(0xffffffffu, sv_levels(a, b0 + lane) > lo);
    const int c = __popc(on);
    if (left < c) {
      *b_out = b0 + __fns(on, 0, static_cast<int>(left) + 1);
      return true;
    }
    left -= c;
  }
  return false;
}

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

template <int kStages>
struct SvControl {
  uint64_t q_full[2];  // pair form: of each tile; single form: the first
  uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
  uint64_t s_full[2], o_done[2];
  uint64_t p_part[4][2];
  uint64_t drain;
  uint32_t tmem;
  int work;                   // 0: nothing to do
  int b, hk, level;           // prompts
  int pad;
  long long begin, end, off;  // cache
  // a wait that gave up, for the threads that the next barrier joins: [pair of warps][parity], [quad][parity]
  volatile int pair_abort[8][2];
  volatile int quad_abort[4][2];
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
    serving_attention_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                             const __grid_constant__ ServingArgs a) {
  using L = SvSmem<DP, kPair>;
  constexpr int kTileRows = (kPair ? 2 : 1) * kSvRows;
  constexpr int kStages = L::kStages;
  constexpr int kChunks = DP / 64;              // 64-column swizzle chunks
  constexpr int kParts = DP >= 128 ? 4 : 2;     // parts in which P is announced
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
  static_assert(sizeof(SvControl<kStages>) <= 1024, "control block");

  const uint32_t warp = warp_id();
  const uint32_t lane = lane_id();
  const int cta = blockIdx.x;
  if constexpr (kPaged) griddep_launch_dependents();

  if (warp == 0) {
    bool work;
    if constexpr (kPaged) {
      SvWalk<kTileRows> w;
      long long quota, total;
      work = sv_share<kTileRows>(a, cta, gridDim.x, w, &quota, &total);
      if (lane == 0 && work) {
        ctl->b = w.b;
        ctl->begin = w.begin;
        ctl->end = w.end;
        ctl->off = w.off;
      }
    } else {
      int b = 0, hk = 0, level = 0;
      work = sv_prompt_tile(a, cta, &b, &hk, &level);
      if (lane == 0) {
        ctl->b = b;
        ctl->hk = hk;
        ctl->level = level;
      }
    }
    if (lane == 0) {
      ctl->work = work && (smem_u32(smem) & 1023) == 0;
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
    }
  } else if (warp == 1) {
    tmem_alloc(&ctl->tmem, 512);
    tmem_relinquish();
  } else if (warp == 2 && lane == 0) {
    for (int t = 0; t < 2; ++t) mbar_init(&ctl->q_full[t], kPair ? 8 : 16);  // one arrive per softmax warp
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&ctl->k_full[s], 1);
      mbar_init(&ctl->k_empty[s], 1);
      mbar_init(&ctl->v_full[s], 1);
      mbar_init(&ctl->v_empty[s], 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctl->s_full[t], 1);
      mbar_init(&ctl->o_done[t], 1);
      for (int p = 0; p < kParts; ++p) mbar_init(&ctl->p_part[p][t], 8);  // one arrive per softmax warp
    }
    mbar_init(&ctl->drain, 1);
    for (int i = 0; i < 16; ++i) ctl->pair_abort[i >> 1][i & 1] = 0;
    for (int i = 0; i < 8; ++i) ctl->quad_abort[i >> 1][i & 1] = 0;
    fence_mbar_init();
  }
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;
  const bool work = ctl->work != 0;

  // The pieces of this CTA: one tile (prompts) or a share of the line (cache).
  SvWalk<kTileRows> walk;
  int pieces = 0;
  if constexpr (kPaged) {
    if (work) {
      walk.begin = walk.pos = ctl->begin;
      walk.end = ctl->end;
      walk.off = ctl->off;
      walk.b = ctl->b;
      walk.load(a);
    }
  }
  auto next = [&](SvPiece& p) -> bool {
    if (!work) return false;
    if constexpr (kPaged) {
      return walk.next(a, cta, p);
    } else {
      if (pieces++) return false;
      bool clamped;
      p.b = ctl->b;
      p.hk = ctl->hk;
      p.s = sv_sequence<false>(a, p.b, &clamped);
      p.rows = p.s.n * a.group;
      p.row0 = ctl->level * (2 * kSvRows);
      p.kb = 0;
      p.part = -1;
      sv_streams<false, kPair>(a, p, INT32_MAX);
      return true;
    }
  };

  SvPiece pc;
  if (warp == 0) {
    // ------------------------------------------------------------ loads
    uint32_t count = 0;  // blocks issued to either ring
    bool ok = true;
    while (ok && next(pc)) {
      for (int j = 0; j < pc.loads && ok; ++j, ++count) {
        const int st = count % kStages;
        const uint32_t ph = (count / kStages) & 1;
        const int key0 = (pc.kb + j) * kSvKeys;
        uint32_t bytes = L::kKV;
        int page = 0, boxes = 0;
        const bool mine = lane == 0;
        if constexpr (kPaged) {
          // lane b looks up the page of box b (box_rows keys)
          boxes = (min(kSvKeys, pc.s.m - key0) + a.box_rows - 1) / a.box_rows;
          bytes = static_cast<uint32_t>(boxes * a.box_rows * 128 * kChunks);
          if (static_cast<int>(lane) < boxes) {
            const int key = key0 + static_cast<int>(lane) * a.box_rows;
            page = a.page_table[pc.b * a.table_stride + key / a.page_size];
            if (page < 0 || page >= a.num_pages) {  // outside the tensor: TMA fills zeros
              record_bad_index();
              page = -1;
            }
          }
        }
        auto load = [&](const CUtensorMap& tm, uint8_t* ring, uint64_t* full, uint64_t* empty) {
          if (count >= kStages) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], ph ^ 1, kSiteFlashFree));
          if (!ok) return;
          if (lane == 0) mbar_expect_tx(&full[st], bytes);
          __syncwarp();
          if constexpr (kPaged) {
            const uint32_t dst = smem_u32(ring + st * L::kKV), bar = smem_u32(&full[st]);
            int in_page = key0 % a.page_size;
#pragma unroll 4
            for (int box = 0; box < boxes; ++box) {
              const int at = __shfl_sync(0xffffffffu, page, box);
              for (int c = 0; c < kChunks; ++c)
                tma_load_4d_warp(dst + c * 16384 + box * a.box_rows * 128, &tm, bar, c * 64, in_page, pc.hk, at);
              in_page += a.box_rows;
              if (in_page == a.page_size) in_page = 0;
            }
          } else {
            if (mine)
              for (int c = 0; c < kChunks; ++c)
                tma_load_3d(ring + st * L::kKV + c * 16384, &tm, &full[st], c * 64, pc.hk, pc.s.k0 + key0);
          }
        };
        load(tmK, sK, ctl->k_full, ctl->k_empty);
        if (ok) load(tmV, sV, ctl->v_full, ctl->v_empty);
      }
    }
    if (!ok) {
      // a wait gave up: the loads in flight end before the CTA does
      for (uint32_t c = count > kStages ? count - kStages : 0; c < count; ++c) {
        mbar_wait(&ctl->k_full[c % kStages], (c / kStages) & 1, kSiteDrain);
        mbar_wait(&ctl->v_full[c % kStages], (c / kStages) & 1, kSiteDrain);
      }
    }
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
    auto take_values = [&](int block) {
      const int st = vc % kStages;
      wait(&ctl->v_full[st], (vc / kStages) & 1, kSiteFlashKV);
      const int live = pc.s.m - block * kSvKeys;
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
    while (ok && next(pc)) {
      // (a tile without blocks in this piece is not loaded: its warps go on to the next piece)
      if (!kPair || pc.n[0] > 0) wait(&ctl->q_full[0], q_cnt[0]++ & 1, kSiteFlashQ);
      if (kPair && pc.n[1] > 0) wait(&ctl->q_full[1], q_cnt[1]++ & 1, kSiteFlashQ);
      if constexpr (kPair) {
        for (int j = 0; j <= pc.loads && ok; ++j) {
          if (j < pc.loads) wait(&ctl->k_full[kc % kStages], (kc / kStages) & 1, kSiteFlashKV);
          if (j >= 1) take_values(pc.kb + j - 1);
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (ok && j >= 1 && j <= pc.n[t]) {
              issue_pv(t, j == 1);
              if (ok && j == pc.n[t]) umma_commit_warp(&ctl->o_done[t]);
            }
            if (ok && j < pc.n[t]) issue_s(t);
          }
          if (!ok) break;
          if (j < pc.loads) {
            umma_commit_warp(&ctl->k_empty[kc % kStages]);
            ++kc;
          }
          if (j >= 1) {
            umma_commit_warp(&ctl->v_empty[vc % kStages]);
            ++vc;
          }
        }
      } else {
        for (int j = 0; j < pc.loads + 2 && ok; ++j) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if ((j & 1) != t) continue;
            if (j >= 2) {
              take_values(pc.kb + j - 2);
              if (ok) issue_pv(t, j == 2 + t);
              if (!ok) break;
              umma_commit_warp(&ctl->v_empty[vc % kStages]);
              ++vc;
              if (j >= pc.loads) umma_commit_warp(&ctl->o_done[t]);
            }
            if (j < pc.loads) {
              wait(&ctl->k_full[kc % kStages], (kc / kStages) & 1, kSiteFlashKV);
              if (!ok) break;
              issue_s(t);
              umma_commit_warp(&ctl->k_empty[kc % kStages]);
              ++kc;
            }
          }
        }
      }
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
    uint32_t n_piece = 0;
    bool alive = true;
    auto swap_slot = [&](uint32_t ev) {
      return xchg + ((L::kXBufs == 2 ? (ev & 1) * 2 : 0) + grp) * (2 * kSvRows);
    };
    while (alive && next(pc)) {
      // ---- this piece's row
      const int row = pc.row0 + (kPair ? grp * kSvRows : 0) + r;
      const bool live = row < pc.rows;
      const int tok = live ? row / a.group : 0;
      const int head = pc.hk * a.group + (live ? row - tok * a.group : 0);
      const long long qrow = pc.s.q0 + tok;
      const bool tree = kPaged && a.mask != nullptr;
      int sees = pc.s.m;  // keys 0 .. sees - 1 are visible (and the nodes of the mask row)
      if (tree) sees = pc.s.sure;
      else if (kPaged || a.causal) sees = min(pc.s.m, pc.s.sure + tok + 1);
      if (!live) sees = 0;
      // ---- Q into shared memory (K-major, 128-byte swizzle), zero past the rows and the head
      if (!kPair || pc.n[grp] > 0) {
        constexpr int kCols = kPair ? DP / 2 : DP / 4;  // of this thread
        const int c0 = kPair ? half * kCols : (2 * grp + half) * kCols;
        const T* src = static_cast<const T*>(a.q) + qrow * a.q_st[0] + head * a.q_st[1];
        uint4 v[kCols / 8];
#pragma unroll
        for (int x = 0; x < kCols / 8; ++x) {
          v[x] = uint4{0, 0, 0, 0};
          if (live && c0 + x * 8 < a.head_dim) v[x] = *reinterpret_cast<const uint4*>(src + c0 + x * 8);
        }
        uint8_t* dst = sQ + (kPair ? grp * L::kQ : 0) + r * 128;
#pragma unroll
        for (int x = 0; x < kCols / 8; ++x) {
          const int c = (c0 + x * 8) / 8;  // 16-byte column
          *reinterpret_cast<uint4*>(dst + (c >> 3) * 16384 + (((c & 7) ^ (r & 7)) << 4)) = v[x];
        }
        fence_async_shared();
        tc_fence_before();  // the last piece's O has been read
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->q_full[kPair ? grp : 0]);
      }
      float m_use = -INFINITY;
      float m_true = -INFINITY;  // exact running maximum (m_use may lag it by the rescale threshold)
      float l = 0.0f;            // this half's share of the row sum
      const int nblk = pc.n[grp];
      const bool warp_live = __any_sync(0xffffffffu, live);
      for (int i = 0; i < nblk; ++i, ++s_cnt, ++events) {
        if (!mbar_wait(&ctl->s_full[grp], s_cnt & 1, kSiteFlashS)) ctl->pair_abort[pair_id][events & 1] = 1;
        if (!warp_live) {
          // no row here: nothing reads these lanes of P
          named_bar_sync(pair_bar, 64);
          if constexpr (L::kXBufs == 1) named_bar_sync(pair_bar, 64);
          if (ctl->pair_abort[pair_id][events & 1]) {
            alive = false;
            break;
          }
          if (lane == 0)
            for (int p = 0; p < kParts; ++p) mbar_arrive(&ctl->p_part[p][grp]);
          continue;
        }
        tc_fence_after();
        const int kv0 = (pc.kb + (kPair ? i : 2 * i + grp)) * kSvKeys + half * 64;
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
            const int node = kv0 - pc.s.sure;  // of this half's first key
            const int nodes = pc.s.m - pc.s.sure;
            if (node > -64 && node < nodes) {
              uint64_t bits = mask_window(a.mask + qrow * a.mask_stride, a.mask_words, node);
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
        float* xs = swap_slot(events);
        xs[half * kSvRows + r] = pmax;
        tc_fence_before();
        named_bar_sync(pair_bar, 64);
        tc_fence_after();
        const float other = xs[(half ^ 1) * kSvRows + r];
        if constexpr (L::kXBufs == 1) named_bar_sync(pair_bar, 64);
        if (ctl->pair_abort[pair_id][events & 1]) {
          alive = false;
          break;
        }
        const float rmax = sl * fmaxf(pmax, other);
        m_true = fmaxf(m_true, rmax);
        const bool grow = rmax > m_use + 8.0f;
        const float m_new = grow ? rmax : m_use;
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
      float* slot = nullptr;  // [kRows][DP] O, [kRows] m, [kRows] l
      if (kPaged && pc.part >= 0) slot = a.parts + static_cast<size_t>(pc.part) * kTileRows * (DP + 2);
      const int prow = (kPair ? grp * kSvRows : 0) + r;
      T* out = static_cast<T*>(a.o) + qrow * a.o_st[0] + head * a.o_st[1];
      float w0 = 0.0f, w1 = 0.0f;  // of O_0 and O_1 (pair form: w0 of this stream's)
      float l_row, m_row;
      if constexpr (kPair) {
        if (!alive) break;
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
        w0 = slot != nullptr ? 1.0f : l_row > 0.0f || l_row != l_row ? 1.0f / l_row : 0.0f;
        if (nblk == 0) w0 = 0.0f;
      } else {
        if (!alive) ctl->quad_abort[wq][n_piece & 1] = 1;
        // both streams of this row: m and the two halves' sums
        float* xs = xchg;
        for (int t = 0; t < 2; ++t) {
          if (pc.n[t] > 0 && !mbar_wait(&ctl->o_done[t], o_cnt[t] & 1, kSiteFlashPV))
            ctl->quad_abort[wq][n_piece & 1] = 1;
          if (pc.n[t] > 0) ++o_cnt[t];
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
        if (ctl->quad_abort[wq][n_piece & 1]) {
          alive = false;
          break;
        }
        m_row = fmaxf(m0, m1);
        const float m_sub = m_row == -INFINITY ? 0.0f : m_row;
        w0 = exp2f(m0 - m_sub);  // 0 for a stream that saw nothing
        w1 = exp2f(m1 - m_sub);
        l_row = l0 * w0 + l1 * w1;
        if (slot == nullptr) {
          const float inv = l_row > 0.0f || l_row != l_row ? 1.0f / l_row : 0.0f;
          w0 *= inv;
          w1 *= inv;
        }
      }
      ++n_piece;
      tc_fence_after();
      if (warp_live) {
        constexpr int kCols = kPair ? DP / 2 : DP / 4;
        const int c0 = kPair ? half * kCols : (2 * grp + half) * kCols;
        constexpr int kStep = kCols < 32 ? kCols : 32;
#pragma unroll 1
        for (int c = c0; c < c0 + kCols; c += kStep) {
          float o[kStep];
#pragma unroll
          for (int x = 0; x < kStep; ++x) o[x] = 0.0f;
#pragma unroll
          for (int t = 0; t < (kPair ? 1 : 2); ++t) {
            const int u = kPair ? grp : t;
            if (pc.n[u] == 0) continue;  // nothing was accumulated there
            const float w = t == 0 ? w0 : w1;
#pragma unroll
            for (int x = 0; x < kStep; x += 8) {
              uint32_t e[8];
              tmem_ld8(tmem + lane_off + kColO + u * 128 + c + x, e);
#pragma unroll
              for (int y = 0; y < 8; ++y) o[x + y] += w != 0.0f ? w * __uint_as_float(e[y]) : 0.0f;
            }
          }
          if (!live) continue;
          if (slot != nullptr) {
#pragma unroll
            for (int x = 0; x < kStep; x += 4)
              *reinterpret_cast<float4*>(slot + static_cast<size_t>(prow) * DP + c + x) =
                  make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
          } else {
#pragma unroll
            for (int x = 0; x < kStep; x += 8)
              if (c + x < a.head_dim) {
                uint4 v;
                v.x = pack2<T>(o[x], o[x + 1]);
                v.y = pack2<T>(o[x + 2], o[x + 3]);
                v.z = pack2<T>(o[x + 4], o[x + 5]);
                v.w = pack2<T>(o[x + 6], o[x + 7]);
                *reinterpret_cast<uint4*>(out + c + x) = v;
              }
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
    }
  }

  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Adds up the parts of the item that starts in share c = blockIdx.x and goes
// on past its end, in order: a warp per row, four values of the head per lane.
//   m = max m_p,  o = sum 2^(m_p - m) O_p / sum 2^(m_p - m) l_p
template <int DP, typename T, int kTileRows>
__global__ void __launch_bounds__(kSvJoinThreads) attention_join_kernel(const __grid_constant__ ServingArgs a) {
  __shared__ int from, parts, slot0, row0, rows, q0, hk;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (warp == 0) {
    SvWalk<kTileRows> w;
    long long quota, total;
    const bool work = sv_share<kTileRows>(a, blockIdx.x, gridDim.x, w, &quota, &total);
    if (lane == 0) {
      parts = 0;
      SvPiece p;
      while (work) {
        const long long start = w.pos;
        if (!w.next(a, blockIdx.x, p)) break;
        if (p.part < 0 || p.kb != 0) continue;  // whole, or the end of an earlier share's item
        // starts here and is cut by the end of the share
        const long long last = (start + w.blocks - 1) / quota;
        from = blockIdx.x;
        parts = static_cast<int>(last) - blockIdx.x + 1;
        slot0 = p.part;
        row0 = p.row0;
        rows = p.rows;
        q0 = p.s.q0;
        hk = p.hk;
      }
    }
  }
  __syncthreads();
  griddep_wait();  // the parts
  if (parts == 0) return;
  const int n = min(kTileRows, rows - row0);
  constexpr size_t kSlot = static_cast<size_t>(kTileRows) * (DP + 2);
  auto part = [&](int i) { return a.parts + (i == 0 ? slot0 : 2 * (from + i)) * kSlot; };
  for (int r = blockIdx.y * (kSvJoinThreads / 32) + warp; r < n; r += gridDim.y * (kSvJoinThreads / 32)) {
    float m = -INFINITY;
    for (int i = lane; i < parts; i += 32) m = fmaxf(m, part(i)[static_cast<size_t>(kTileRows) * DP + r]);
#pragma unroll
    for (int x = 16; x; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
    const float m_sub = m == -INFINITY ? 0.0f : m;
    float o[4] = {}, l = 0.0f;
    const int d = lane * 4;
    const bool on = d < a.head_dim;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
      const float* p = part(i);
      const float w = exp2f(p[static_cast<size_t>(kTileRows) * DP + r] - m_sub);
      l += w * p[static_cast<size_t>(kTileRows) * (DP + 1) + r];
      if (on && w != 0.0f) {
        const float4 v = *reinterpret_cast<const float4*>(p + static_cast<size_t>(r) * DP + d);
        o[0] += w * v.x;
        o[1] += w * v.y;
        o[2] += w * v.z;
        o[3] += w * v.w;
      }
    }
    const int row = row0 + r;
    const int tok = row / a.group;
    const int head = hk * a.group + row - tok * a.group;
    const long long qrow = q0 + tok;
    const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;
    if (on) {
      uint2 v;
      v.x = pack2<T>(o[0] * inv, o[1] * inv);
      v.y = pack2<T>(o[2] * inv, o[3] * inv);
      *reinterpret_cast<uint2*>(static_cast<T*>(a.o) + qrow * a.o_st[0] + head * a.o_st[1] + d) = v;
    }
    if (a.lse != nullptr && lane == 0) a.lse[qrow * a.q_heads + head] = (m + log2f(l)) * 0.6931471805599453f;
  }
}

}  // namespace akili
