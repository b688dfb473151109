// decode_attention.cuh — the few-row form of the attention over a paged cache
// (serving_attention.cuh): single tokens and small trees, up to N = 16, 32 or
// 64 rows (tokens times grouped heads) per key head.
//
// Reading the cache is all the time such a call has, so the kernel must never
// be what the loads wait for.  With the rows as the M side of the tensor core
// (the row forms) four or eight rows still cost a 128-row softmax on one SM
// quarter and every (sequence, key head) drained the pipeline: 1.2 us a block
// and 6 us an item, against the 1.5 us a block takes to arrive.  Here the keys
// are the M side:
//   S^T = K Q^T        [128 keys x N]   A = K tile, B = Q, both K-major
//   P^T = 2^(c S^T - m) one thread per key, all N rows: 128 threads on all
//                      four quarters, N exponentials each
//   O^T += V^T P^T     [DP x N]         A = V tile (MN-major), B = P^T from
//                      shared memory (key by key, MN-major), rounded to the
//                      element type, as a 16-bit product takes it; the row
//                      sums keep fp32
// A row's maximum is over the 128 threads, but it is only needed where some
// score passes the running maximum by more than 2^8 (a stale maximum cancels
// in O / l): one barrier per block carries that vote, and the reduction and
// the rescaling of O run only then.  Row sums stay per thread until the end.
// What belongs to a row (maximum, factors, address, its visible keys as bit
// words of a block) is worked out by one thread and read by all from shared
// memory; with every thread doing so for itself a short item of 64 rows took
// 36000 cycles.
//
// Warps: 0 key loads, 1 value loads (each issues its own ring's TMA boxes, one
// per page part), 2 TMEM owner and MMA issuer, 3 loads the next item's Q, 4..7
// softmax and output.  Q, S, P and O have two buffers each, so an item's first
// scores are computed while the last one is still being written out.
//
// Measured: 32 contexts of 77 to 16383 tokens, one new token each, 32/8 heads
// of 128, bf16: 171 us, 6.4 TB/s, 0.98 of the copy rate (the row form 242 us);
// one context of 4001 tokens, 32 heads, fp16: 17 us from L2, 20 from HBM, of
// which 10 are its 65 MB and the rest start, first loads and join.
#pragma once
#include "serving_attention.cuh"

namespace akili {

constexpr int kDcThreads = 256;

template <int DP, int N>
struct DcSmem {
  static constexpr int kKV = kSvKeys * DP * 2;  // one key or value block
  static constexpr int kQ = N * DP * 2;
  static constexpr int kP = kSvKeys * N * 2;
  // what is left of 227 KB; values are held longer than keys
  static constexpr int kKStages = DP == 64 ? 5 : N == 64 ? 2 : 3;
  static constexpr int kVStages = DP == 64 ? 5 : 3;
  static constexpr int kVOff = kKStages * kKV;
  // (with DP = 64 the MMA's M = 128 reads 16 KB past a value block, within
  // this memory: rows of O^T that nobody uses)
  static constexpr int kQOff = kVOff + kVStages * kKV;
  static constexpr int kPOff = kQOff + 2 * kQ;
  static constexpr int kXOff = DP == 64 && 2 * (kQ + kP) < 16384 ? kQOff + 16384 : kPOff + 2 * kP;
  // by row: [4 warps] exchange, [4 x 32 keys] visible bits, maximum, factor
  static constexpr int kCtlOff = kXOff + 10 * N * 4;
  static constexpr int kBytes = kCtlOff + 512;
  static_assert(kBytes <= 232448, "227 KB of shared memory per CTA");
};

struct DcControl {
  uint64_t k_full[5], k_empty[5], v_full[5], v_empty[5];
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], pv_done[2], o_full[2], o_empty[2];
  uint64_t drain;
  uint32_t tmem;
  volatile int abort[2];  // a wait that gave up before the barrier of this parity
};

// Reduces v[n] over the warp's lanes by halving: after it lane L holds the
// result of row (L * N / 32) + i in v[i] (N >= 32), or of row L / (32 / N).
template <int N, typename Op>
__device__ __forceinline__ void lane_reduce(float (&v)[N], Op op) {
  const uint32_t lane = lane_id();
  int count = N;
#pragma unroll
  for (int b = 16; b >= 1; b >>= 1) {
    if (count > 1) {
      const bool upper = (lane & b) != 0;
#pragma unroll
      for (int i = 0; i < N / 2; ++i) {
        if (i < count / 2) {
          const float send = upper ? v[i] : v[i + count / 2];
          const float keep = upper ? v[i + count / 2] : v[i];
          v[i] = op(keep, __shfl_xor_sync(0xffffffffu, send, b));
        }
      }
      count /= 2;
    } else {
      v[0] = op(v[0], __shfl_xor_sync(0xffffffffu, v[0], b));
    }
  }
}

template <int N>
__device__ __forceinline__ void tmem_ld_n(uint32_t taddr, float (&v)[N]) {
  if constexpr (N == 64) {
    tmem_ld64(taddr, v);
  } else if constexpr (N == 32) {
    tmem_ld32(taddr, v);
  } else {
#pragma unroll
    for (int c = 0; c < N; c += 8) {
      uint32_t e[8];
      tmem_ld8(taddr + c, e);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c + i] = __uint_as_float(e[i]);
    }
  }
}

template <int DP, typename T, int N>
__global__ void __launch_bounds__(kDcThreads, 1)
    decode_attention_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                            const __grid_constant__ ServingArgs a) {
  using L = DcSmem<DP, N>;
  constexpr int kChunks = DP / 64;
  constexpr int kKStages = L::kKStages, kVStages = L::kVStages;
  constexpr uint32_t kColO = 2 * N;  // S at 0 and N, O at 2N and 3N
  constexpr uint32_t kTmemCols = 4 * N;
  constexpr uint32_t kFmt = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
  constexpr uint32_t kPSwizzle = N == 16 ? kSw32 : N == 32 ? kSw64 : kSw128;
  static_assert(N == 16 || N == 32 || N == 64, "rows per item");

  extern __shared__ __align__(1024) uint8_t sv_smem[];
  uint8_t* smem = sv_smem;
  auto* ctl = reinterpret_cast<DcControl*>(smem + L::kCtlOff);
  static_assert(sizeof(DcControl) <= 512, "control block");
  float* xchg = reinterpret_cast<float*>(smem + L::kXOff);
  uint32_t* visible = reinterpret_cast<uint32_t*>(xchg + 4 * N);
  float* row_max = xchg + 8 * N;
  float* factor = xchg + 9 * N;
  const uint32_t warp = warp_id();
  const uint32_t lane = lane_id();

  if (warp == 3) {
    if (lane == 0) {
      tma_prefetch_desc(&tmK);
      tma_prefetch_desc(&tmV);
      for (int s = 0; s < kKStages; ++s) {
        mbar_init(&ctl->k_full[s], 1);
        mbar_init(&ctl->k_empty[s], 1);
      }
      for (int s = 0; s < kVStages; ++s) {
        mbar_init(&ctl->v_full[s], 1);
        mbar_init(&ctl->v_empty[s], 1);
      }
      for (int i = 0; i < 2; ++i) {
        mbar_init(&ctl->q_full[i], 1);
        mbar_init(&ctl->q_empty[i], 1);
        mbar_init(&ctl->s_full[i], 1);
        mbar_init(&ctl->p_full[i], 4);  // one arrive per softmax warp
        mbar_init(&ctl->pv_done[i], 1);
        mbar_init(&ctl->o_full[i], 1);
        mbar_init(&ctl->o_empty[i], 4);
        ctl->abort[i] = 0;
      }
      mbar_init(&ctl->drain, 1);
      fence_mbar_init();
    }
    __syncwarp();
  } else if (warp == 2) {
    tmem_alloc(&ctl->tmem, kTmemCols);
    tmem_relinquish();
  }
  // Nothing of an earlier kernel is read before it is complete; the join
  // kernel, whose blocks read the lengths as they start, may start after that.
  griddep_wait();
  griddep_launch_dependents();
  // Every warp finds the CTA's share by itself and the loaders look up their
  // first pages before the barrier: the first load leaves that much earlier
  // (5500 -> 4500 cycles after the start).
  SvWalk<N> walk;
  SvPiece pc;
  long long quota, total;
  const bool work = sv_share<N>(a, blockIdx.x, gridDim.x, walk, &quota, &total) && (smem_u32(smem) & 1023) == 0;
  auto next = [&]() { return work && walk.next(a, blockIdx.x, pc); };
  // lane b looks up the page of box b (box_rows keys) of block j of the piece
  auto lookup = [&](int j) -> int {
    const int in = static_cast<int>(lane) * a.box_rows;
    const int key = (pc.kb + j) * kSvKeys + in;
    return j < pc.loads && in < kSvKeys && key < pc.s.m ? a.page_table[pc.b * a.table_stride + key / a.page_size] : 0;
  };
  bool have = next();
  int page = have && warp < 2 ? lookup(0) : 0;
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ctl->tmem;

  if (warp < 2) {
    // ------------------------------------------------------ key / value loads
    const bool is_v = warp == 1;
    const CUtensorMap* tm = is_v ? &tmV : &tmK;
    uint8_t* ring = smem + (is_v ? L::kVOff : 0);
    uint64_t* full = is_v ? ctl->v_full : ctl->k_full;
    uint64_t* empty = is_v ? ctl->v_empty : ctl->k_empty;
    const int stages = is_v ? kVStages : kKStages;
    int st = 0;
    uint32_t round = 0, issued = 0;
    bool ok = true;
    for (bool first = true; ok && have; have = next(), first = false) {
      if (!first) page = lookup(0);
      int ahead = lookup(1);
      for (int j = 0; j < pc.loads; ++j) {
        const int key0 = (pc.kb + j) * kSvKeys;
        const int boxes = (min(kSvKeys, pc.s.m - key0) + a.box_rows - 1) / a.box_rows;
        if (round > 0) ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], (round - 1) & 1, kSiteFlashFree));
        if (!ok) break;
        if (page < 0 || page >= a.num_pages) {  // outside the tensor: TMA fills zeros
          record_bad_index();
          page = -1;
        }
        if (lane == 0) mbar_expect_tx(&full[st], static_cast<uint32_t>(boxes * a.box_rows * 128 * kChunks));
        __syncwarp();
        const uint32_t dst = smem_u32(ring + st * L::kKV), bar = smem_u32(&full[st]);
        int in_page = key0 % a.page_size;
#pragma unroll 4
        for (int box = 0; box < boxes; ++box) {
          const int at = __shfl_sync(0xffffffffu, page, box);
#pragma unroll
          for (int c = 0; c < kChunks; ++c)
            tma_load_4d_warp(dst + c * 16384 + box * a.box_rows * 128, tm, bar, c * 64, in_page, pc.hk, at);
          in_page += a.box_rows;
          if (in_page == a.page_size) in_page = 0;
        }
        ++issued;
        page = ahead;
        ahead = lookup(j + 2);
        if (++st == stages) {
          st = 0;
          ++round;
        }
      }
    }
    if (!ok)  // a wait gave up: the loads in flight end before the CTA does
      for (uint32_t c = issued > static_cast<uint32_t>(stages) ? issued - stages : 0; c < issued; ++c)
        mbar_wait(&full[c % stages], (c / stages) & 1, kSiteDrain);
    __syncwarp();
  } else if (warp == 2) {
    // ------------------------------------------------------------------- MMA
    constexpr uint32_t idesc_s = make_idesc_f16(kSvKeys, N, false, false) | kFmt;
    constexpr uint32_t idesc_o = make_idesc_f16(128, N, true, true) | kFmt;
    const uint64_t kd0 = make_sdesc(smem_u32(smem), 16, 1024, kSw128);
    const uint64_t vd0 = make_sdesc(smem_u32(smem + L::kVOff), 16384, 1024, kSw128);
    const uint64_t qd0 = make_sdesc(smem_u32(smem + L::kQOff), 16, 1024, kSw128);
    const uint64_t pd0 = make_sdesc(smem_u32(smem + L::kPOff), kSvKeys * N * 2, 16 * N, kPSwizzle);
    int ks = 0, vs = 0;
    uint32_t kr = 0, vr = 0;  // rounds of the rings
    uint32_t g = 0;           // blocks whose S was issued
    uint32_t item = 0;
    bool ok = true;
    auto wait = [&](uint64_t* bar, uint32_t parity, uint32_t site) {
      ok = ok && __all_sync(0xffffffffu, mbar_wait(bar, parity, site));
    };
    // block g - 1, whose O^T += V^T P^T is issued after S of block g
    int held_live = 0;         // its keys inside the sequence (may exceed 128)
    uint32_t held_item = 0;
    bool held = false, held_first = false, held_last = false;
    auto issue_pv = [&]() {
      const uint32_t pb = (g - 1) & 1;
      wait(&ctl->v_full[vs], vr & 1, kSiteFlashKV);
      if (held_first && held_item >= 2) wait(&ctl->o_empty[held_item & 1], ((held_item >> 1) - 1) & 1, kSiteFlashFree);
      if (!ok) return;
      if (held_live < kSvKeys) {
        // values past the sequence's end may be anything: 0 times them must be 0
        uint8_t* v = smem + L::kVOff + vs * L::kKV;
        const uint4 zero = {0, 0, 0, 0};
        for (int c = 0; c < kChunks; ++c)
          for (int x = held_live * 8 + static_cast<int>(lane); x < kSvKeys * 8; x += 32)
            *reinterpret_cast<uint4*>(v + c * 16384 + x * 16) = zero;
        fence_async_shared();
        __syncwarp();
      }
      wait(&ctl->p_full[pb], ((g - 1) >> 1) & 1, kSiteFlashP);
      if (!ok) return;
      tc_fence_after();
      const uint64_t vd = vd0 + static_cast<uint64_t>((vs * L::kKV) >> 4);
      const uint64_t pd = pd0 + static_cast<uint64_t>((pb * L::kP) >> 4);
      const uint32_t o = tmem + kColO + (held_item & 1) * N;
#pragma unroll
      for (int k = 0; k < kSvKeys / 16; ++k)
        umma_f16_ss_warp(o, vd + static_cast<uint64_t>((k * 2048) >> 4), pd + static_cast<uint64_t>((k * 32 * N) >> 4),
                         idesc_o, !held_first || k != 0);
      umma_commit_warp(&ctl->pv_done[pb]);
      umma_commit_warp(&ctl->v_empty[vs]);
      if (held_last) umma_commit_warp(&ctl->o_full[held_item & 1]);
      if (++vs == kVStages) {
        vs = 0;
        ++vr;
      }
    };
    for (; ok && have; have = next()) {
      for (int j = 0; j < pc.loads && ok; ++j) {
        // The product of the block before goes first where its successor's keys
        // are still on their way.
        if (held && !__all_sync(0xffffffffu, mbar_try_wait(smem_u32(&ctl->k_full[ks]), kr & 1))) {
          issue_pv();
          held = false;
          if (!ok) break;
        }
        if (j == 0) wait(&ctl->q_full[item & 1], (item >> 1) & 1, kSiteFlashQ);
        wait(&ctl->k_full[ks], kr & 1, kSiteFlashKV);
        if (!ok) break;
        // (S of block g - 2 was read before its P was announced, which issue_pv has waited for)
        tc_fence_after();
        const uint64_t kd = kd0 + static_cast<uint64_t>((ks * L::kKV) >> 4);
        const uint64_t qd = qd0 + static_cast<uint64_t>(((item & 1) * L::kQ) >> 4);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          umma_f16_ss_warp(tmem + (g & 1) * N, kd + static_cast<uint64_t>(((k >> 2) * 16384 + (k & 3) * 32) >> 4),
                           qd + static_cast<uint64_t>(((k >> 2) * (N * 128) + (k & 3) * 32) >> 4), idesc_s, k != 0);
        umma_commit_warp(&ctl->s_full[g & 1]);
        umma_commit_warp(&ctl->k_empty[ks]);
        if (j == pc.loads - 1) umma_commit_warp(&ctl->q_empty[item & 1]);
        if (++ks == kKStages) {
          ks = 0;
          ++kr;
        }
        if (held) issue_pv();
        ++g;
        held = true;
        held_first = j == 0;
        held_last = j == pc.loads - 1;
        held_item = item;
        held_live = pc.s.m - (pc.kb + j) * kSvKeys;
      }
      ++item;
    }
    if (ok && held) issue_pv();
    umma_commit_warp(&ctl->drain);
    mbar_wait(&ctl->drain, 0, kSiteDrain);
    __syncwarp();
  } else if (warp == 3) {
    // --------------------------------------------------------------- Q loads
    // rows x 16-byte columns over the lanes, K-major with the 128-byte swizzle
    uint32_t item = 0;
    bool ok = true;
    for (; ok && have; ++item, have = next()) {
      if (item >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&ctl->q_empty[item & 1], ((item >> 1) - 1) & 1, kSiteFlashFree));
      if (!ok) break;
      uint8_t* dst = smem + L::kQOff + (item & 1) * L::kQ;
      constexpr int kUnits = N * DP / 8;  // 16-byte units
#pragma unroll 4
      for (int x = lane; x < kUnits; x += 32) {
        const int n = x / (DP / 8), c = x % (DP / 8);
        const int row = pc.tile * N + n;
        uint4 v = {0, 0, 0, 0};
        if (row < pc.s.n * a.group && c * 8 < a.head_dim) {
          const int tok = row / a.group;
          const int head = pc.hk * a.group + row - tok * a.group;
          v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + (pc.s.q0 + tok) * a.q_st[0] +
                                              head * a.q_st[1] + c * 8);
        }
        *reinterpret_cast<uint4*>(dst + (c >> 3) * (N * 128) + n * 128 + (((c & 7) ^ (n & 7)) << 4)) = v;
      }
      fence_async_shared();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->q_full[item & 1]);
    }
    __syncwarp();
  } else {
    // ------------------------------------------------------ softmax / output
    const int wq = static_cast<int>(warp & 3);        // TMEM lane quarter
    const int t = wq * 32 + static_cast<int>(lane);   // key of the block; later: column of the head
    const uint32_t tbase = tmem + (static_cast<uint32_t>(wq * 32) << 16);
    constexpr uint32_t kBar = 1;
    const float sl = a.scale_log2;
    const bool tree = a.mask != nullptr;
    uint32_t g = 0, item = 0;
    bool alive = true;
    float l[N];
    // lane_reduce's results -> the exchange
    auto share = [&](const float (&v)[N]) {
      if constexpr (N >= 32) {
#pragma unroll
        for (int i = 0; i < N / 32; ++i) xchg[wq * N + lane * (N / 32) + i] = v[i];
      } else {
        if (lane % (32 / N) == 0) xchg[wq * N + lane / (32 / N)] = v[0];
      }
    };
    for (; alive && have; ++item, have = next()) {
#pragma unroll
      for (int n = 0; n < N; ++n) l[n] = 0.0f;
      const int row0 = pc.tile * N;
      const int nrows = min(N, pc.s.n * a.group - row0);
      // keys that every row sees
      const int common = tree ? pc.s.sure : min(pc.s.m, pc.s.sure + row0 / a.group + 1);
      for (int j = 0; j < pc.loads; ++j, ++g) {
        const int key0 = (pc.kb + j) * kSvKeys;
        if (!mbar_wait(&ctl->s_full[g & 1], (g >> 1) & 1, kSiteFlashS)) ctl->abort[g & 1] = 1;
        tc_fence_after();
        float s[N];
        tmem_ld_n<N>(tbase + (g & 1) * N, s);
        if (key0 + kSvKeys > common) {
          // the keys each row sees, 32 to a word
          for (int x = t; x < 4 * N; x += 128) {
            const int n = x % N, first = key0 + 32 * (x / N);
            uint32_t word = 0;
            if (n < nrows) {
              const int tok = (row0 + n) / a.group;
              const int nv = (tree ? pc.s.sure : min(pc.s.m, pc.s.sure + tok + 1)) - first;
              word = nv <= 0 ? 0u : nv >= 32 ? ~0u : (1u << nv) - 1;
              const int node = first - pc.s.sure, nodes = pc.s.m - pc.s.sure;
              if (tree && node > -32 && node < nodes) {
                uint32_t bits = static_cast<uint32_t>(mask_window(a.mask + (pc.s.q0 + tok) * a.mask_stride, a.mask_words, node));
                if (nodes - node < 32) bits &= (1u << (nodes - node)) - 1;
                word |= bits;
              }
            }
            visible[x] = word;
          }
          named_bar_sync(kBar, 128);
#pragma unroll
          for (int n = 0; n < N; n += 4) {
            const uint4 w = *reinterpret_cast<const uint4*>(visible + wq * N + n);
            if (!((w.x >> lane) & 1)) s[n] = -INFINITY;
            if (!((w.y >> lane) & 1)) s[n + 1] = -INFINITY;
            if (!((w.z >> lane) & 1)) s[n + 2] = -INFINITY;
            if (!((w.w >> lane) & 1)) s[n + 3] = -INFINITY;
          }
        }
        // the P buffer's last reader, block g - 2
        if (g >= 2 && !mbar_wait(&ctl->pv_done[g & 1], ((g >> 1) - 1) & 1, kSiteFlashPV)) ctl->abort[g & 1] = 1;
        bool grow = true;  // an item's first block brings the maxima
        if (j > 0) {
          float over = -INFINITY;
#pragma unroll
          for (int n = 0; n < N; n += 4) {
            const float4 m = *reinterpret_cast<const float4*>(row_max + n);
            over = fmaxf(over, fmaxf(fmaxf(fmaf(s[n], sl, -m.x), fmaf(s[n + 1], sl, -m.y)),
                                     fmaxf(fmaf(s[n + 2], sl, -m.z), fmaf(s[n + 3], sl, -m.w))));
          }
          grow = vote_barrier<128>(kBar, over > 8.0f);
          if (ctl->abort[g & 1]) {
            alive = false;
            break;
          }
        }
        if (grow) {
          {
            float mx[N];
#pragma unroll
            for (int n = 0; n < N; ++n) mx[n] = s[n];
            lane_reduce<N>(mx, [](float x, float y) { return fmaxf(x, y); });
            share(mx);
          }
          named_bar_sync(kBar, 128);
          if (t < N) {
            // "nothing seen" is the lowest finite value: any finite score passes it
            const float old = j > 0 ? row_max[t] : -3.4028235e38f;
            const float top = sl * fmaxf(fmaxf(xchg[t], xchg[N + t]), fmaxf(xchg[2 * N + t], xchg[3 * N + t]));
            const float now = top > old + 8.0f ? top : old;
            row_max[t] = now;
            factor[t] = exp2f(old - now);
          }
          // O holds the blocks up to g - 1 once their products are done
          if (j > 0 && !mbar_wait(&ctl->pv_done[(g - 1) & 1], ((g - 1) >> 1) & 1, kSiteFlashPV)) ctl->abort[g & 1] = 1;
          named_bar_sync(kBar, 128);
          if (ctl->abort[g & 1]) {
            alive = false;
            break;
          }
          if (j > 0) {
            tc_fence_after();
            const uint32_t to = tbase + kColO + (item & 1) * N;
#pragma unroll
            for (int c = 0; c < N; c += 8) {
              float f[8];
              *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(factor + c);
              *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(factor + c + 4);
              uint32_t e[8];
              tmem_ld8(to + c, e);
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                l[c + i] *= f[i];
                e[i] = __float_as_uint(__uint_as_float(e[i]) * f[i]);
              }
              tmem_st8(to + c, e);
            }
          }
        }
        uint8_t* prow = smem + L::kPOff + (g & 1) * L::kP + t * (2 * N);
#pragma unroll
        for (int u = 0; u < N / 8; ++u) {
          float m[8];
          *reinterpret_cast<float4*>(m) = *reinterpret_cast<const float4*>(row_max + u * 8);
          *reinterpret_cast<float4*>(m + 4) = *reinterpret_cast<const float4*>(row_max + u * 8 + 4);
          uint32_t e[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = u * 8 + 2 * i;
            const float p0 = ex2_mufu(fmaf(s[n], sl, -m[2 * i])), p1 = ex2_mufu(fmaf(s[n + 1], sl, -m[2 * i + 1]));
            l[n] += p0;
            l[n + 1] += p1;
            e[i] = pack2<T>(p0, p1);
          }
          const int x = N == 16 ? u ^ ((t >> 2) & 1) : N == 32 ? u ^ ((t >> 1) & 3) : u ^ (t & 7);
          *reinterpret_cast<uint4*>(prow + x * 16) = make_uint4(e[0], e[1], e[2], e[3]);
        }
        fence_async_shared();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->p_full[g & 1]);
      }
      // ---- output
      if (!alive) break;
      lane_reduce<N>(l, [](float x, float y) { return x + y; });
      share(l);
      if (!mbar_wait(&ctl->o_full[item & 1], (item >> 1) & 1, kSiteFlashPV)) ctl->abort[g & 1] = 1;
      named_bar_sync(kBar, 128);
      if (ctl->abort[g & 1]) {
        alive = false;
        break;
      }
      float* slot = pc.part < 0 ? nullptr : a.parts + static_cast<size_t>(pc.part) * N * (DP + 2);
      if (t < nrows) {
        const float sum = (xchg[t] + xchg[N + t]) + (xchg[2 * N + t] + xchg[3 * N + t]);
        const float m = sum != 0.0f ? row_max[t] : -INFINITY;
        factor[t] = sum != 0.0f ? 1.0f / sum : 0.0f;
        if (slot != nullptr) {
          slot[N * DP + t] = m;
          slot[N * (DP + 1) + t] = sum;
        } else if (a.lse != nullptr) {
          const int tok = (row0 + t) / a.group;
          a.lse[(pc.s.q0 + tok) * static_cast<long long>(a.q_heads) + pc.hk * a.group + row0 + t - tok * a.group] =
              (m + log2f(sum)) * 0.6931471805599453f;
        }
      }
      tc_fence_after();
      float o[N];
      tmem_ld_n<N>(tbase + kColO + (item & 1) * N, o);
      tc_fence_before();
      named_bar_sync(kBar, 128);
      if (lane == 0) mbar_arrive(&ctl->o_empty[item & 1]);
      if (slot != nullptr) {
        if (t < DP) {
#pragma unroll
          for (int n = 0; n < N; ++n)
            if (n < nrows) slot[n * DP + t] = o[n];
        }
      } else if (t < a.head_dim) {
        int rem = row0 % a.group;
        T* out = static_cast<T*>(a.o) + (pc.s.q0 + row0 / a.group) * a.o_st[0] + (pc.hk * a.group + rem) * a.o_st[1] + t;
        const long long next_tok = a.o_st[0] - (a.group - 1) * a.o_st[1];  // from a token's last head to the next one's first
#pragma unroll
        for (int n = 0; n < N; ++n) {
          if (n < nrows) {
            const float f = factor[n];
            *out = from_f32<T>(f != 0.0f ? o[n] * f : 0.0f);
            if (++rem == a.group) {
              rem = 0;
              out += next_tok;
            } else {
              out += a.o_st[1];
            }
          }
        }
      }
    }
  }

  __syncthreads();
  if (warp == 2) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

}  // namespace akili
