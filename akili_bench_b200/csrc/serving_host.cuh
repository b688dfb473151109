// serving_host.cuh — the entries of include/akili_serving.h: argument checks
// and launches.  Included by akili.cu (shares its device, scratch and
// tensor-map helpers).
#pragma once
#include "../../include/akili_serving.h"
#include "cache.cuh"
#include "decode_attention.cuh"
#include "rope.cuh"
#include "serving_attention.cuh"

namespace {

int serving_elem_bytes(uint32_t dtype) {
  return dtype == AKILI_DTYPE_F32 ? 4 : dtype == AKILI_DTYPE_F16 || dtype == AKILI_DTYPE_BF16 ? 2 : 0;
}

int check_aligned(std::initializer_list<uint64_t> ps, uint64_t bytes) {
  for (uint64_t p : ps)
    if (p == 0) return AKILI_E_NULL_ARG;
  for (uint64_t p : ps)
    if (p % bytes) return AKILI_E_ALIGN;
  return AKILI_OK;
}

template <size_t n>
bool all_multiples(const int64_t (&st)[n], int64_t of) {
  for (int64_t s : st)
    if (s % of) return false;
  return true;
}

// Whether an output's entries can lie apart: those of an axis with stride 0
// would be written one over the other, in any order.
template <size_t n>
bool apart(const int64_t (&stride)[n], const uint64_t (&extent)[n]) {
  for (size_t i = 0; i < n; ++i)
    if (extent[i] > 1 && stride[i] == 0) return false;
  return true;
}

// The serving kernels are programmatic dependents of whatever runs before
// them: a decode step is a chain of them, each a few microseconds long, and
// one may be dispatched and set up while the one before drains.  Each waits
// for its predecessor to complete before it touches memory.
template <typename... Params, typename... Args>
int launch_dependent(void (*kern)(Params...), dim3 grid, int threads, int smem, cudaStream_t st, const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = pdl_enabled() ? 1 : 0;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, args...) != cudaSuccess) {
    g_launches.fetch_add(1, std::memory_order_relaxed);
    cudaGetLastError();
    return AKILI_E_LAUNCH;
  }
  return launch_status();
}

// ------------------------------------------------------------------- rope --
// Blocks that share a token's heads, at most `most`: with few tokens as many as fill the GPU.
constexpr int rope_shares(int tokens, int most, int sms) {
  const int64_t want = (4ll * sms + tokens - 1) / tokens;
  return static_cast<int>(std::min<int64_t>({most, want, 65535}));
}
static_assert(rope_shares(1, 9, 148) == 9 && rope_shares(100, 9, 148) == 6 && rope_shares(INT32_MAX, 9, 148) == 1);

template <typename T, int VEC, bool kAppend>
int launch_rope(const DevInfo& di, const RopeArgs& r, cudaStream_t st) {
  const int units = r.rot_dim / 2 / VEC + (r.head_dim - r.rot_dim + 2 * VEC - 1) / (2 * VEC);
  const int hl = kRopeThreads / std::min(units, kRopeThreads);
  const int heads = r.q_heads + r.k_heads * (kAppend ? 2 : 1);
  const dim3 grid(r.tokens, rope_shares(r.tokens, (heads + hl - 1) / hl, di.sms));
  return launch_dependent(rope_kernel<T, VEC, kAppend>, grid, kRopeThreads, 0, st, r);
}

template <typename T, bool kAppend>
int launch_rope_vec(const DevInfo& di, const RopeArgs& r, bool vec, cudaStream_t st) {
  return vec ? launch_rope<T, 16 / sizeof(T), kAppend>(di, r, st) : launch_rope<T, 1, kAppend>(di, r, st);
}

int run_rope(const akili_rope_arg_t* a, bool append, cudaStream_t st) {
  if (!a) return AKILI_E_NULL_ARG;
  const int es = serving_elem_bytes(a->dtype);
  if (!es) return AKILI_E_DTYPE;
  if (a->flags & ~(AKILI_ROPE_INTERLEAVED | AKILI_ROPE_INVERSE)) return AKILI_E_UNSUPPORTED;
  if (a->rot_dim == 0 || a->rot_dim % 2 || a->rot_dim > a->head_dim || a->max_positions == 0) return AKILI_E_SHAPE;
  if (a->tokens > INT32_MAX || a->head_dim > 65536 || a->q_heads > 65536 || a->k_heads > 65536 ||
      a->max_positions > INT32_MAX)
    return AKILI_E_SHAPE;
  if (append && (a->page_size == 0 || a->page_size > INT32_MAX || a->num_pages > INT32_MAX)) return AKILI_E_SHAPE;
  if (a->tokens == 0 || (a->q_heads == 0 && a->k_heads == 0)) return AKILI_OK;
  int rc;
  if ((rc = check_aligned({a->positions_addr, a->table_addr}, 4))) return rc;
  if (a->q_heads && (rc = check_aligned({a->q_addr, a->q_out_addr}, es))) return rc;
  if (a->k_heads && (rc = check_aligned({a->k_addr}, es))) return rc;
  if (a->k_heads && !append && (rc = check_aligned({a->k_out_addr}, es))) return rc;
  if (a->k_heads && append && (rc = check_aligned({a->v_addr, a->k_pages_addr, a->v_pages_addr}, es))) return rc;
  if (append && a->k_out_addr % es) return AKILI_E_ALIGN;
  if (append && (rc = check_aligned({a->slots_addr}, 8))) return rc;
  if (a->q_heads && !apart(a->q_out_stride, {a->tokens, a->q_heads})) return AKILI_E_SHAPE;
  if (a->k_heads && (!append || a->k_out_addr) && !apart(a->k_out_stride, {a->tokens, a->k_heads}))
    return AKILI_E_SHAPE;
  if (a->k_heads && append && (!apart(a->k_page_stride, {a->num_pages, a->page_size, a->k_heads}) ||
                               !apart(a->v_page_stride, {a->num_pages, a->page_size, a->k_heads})))
    return AKILI_E_SHAPE;
  DevInfo di;
  if ((rc = device_info(&di))) return rc;
  RopeArgs r{};
  r.q = P(a->q_addr); r.k = P(a->k_addr); r.v = P(a->v_addr);
  r.q_out = W(a->q_out_addr);
  r.k_out = W(append ? a->k_pages_addr : a->k_out_addr);
  r.v_out = W(a->v_pages_addr);
  r.k_copy = append ? W(a->k_out_addr) : nullptr;
  r.positions = static_cast<const int*>(P(a->positions_addr));
  r.table = F(a->table_addr);
  r.slots = static_cast<const long long*>(P(a->slots_addr));
  r.tokens = a->tokens; r.q_heads = a->q_heads; r.k_heads = a->k_heads;
  r.head_dim = a->head_dim; r.rot_dim = a->rot_dim; r.max_positions = a->max_positions;
  r.num_pages = a->num_pages; r.page_size = a->page_size;
  r.interleaved = (a->flags & AKILI_ROPE_INTERLEAVED) != 0;
  r.sin_sign = (a->flags & AKILI_ROPE_INVERSE) ? -1.0f : 1.0f;
  for (int i = 0; i < 2; ++i) {
    r.q_st[i] = a->q_stride[i]; r.k_st[i] = a->k_stride[i]; r.qo_st[i] = a->q_out_stride[i];
    r.v_st[i] = a->v_stride[i];
    r.ko_st[i + 1] = r.kc_st[i] = a->k_out_stride[i];
  }
  if (append)
    for (int i = 0; i < 3; ++i) { r.ko_st[i] = a->k_page_stride[i]; r.vo_st[i] = a->v_page_stride[i]; }
  // 16-byte accesses where every vector of every head starts on 16 bytes
  const int64_t n = 16 / es;
  bool vec = a->table_addr % 16 == 0 && (a->rot_dim / 2) % n == 0 && (a->head_dim - a->rot_dim) % n == 0;
  if (a->q_heads)
    vec = vec && (a->q_addr | a->q_out_addr) % 16 == 0 && all_multiples(a->q_stride, n) &&
          all_multiples(a->q_out_stride, n);
  if (a->k_heads) {
    vec = vec && a->k_addr % 16 == 0 && all_multiples(a->k_stride, n);
    if (append)
      vec = vec && (a->v_addr | a->k_pages_addr | a->v_pages_addr) % 16 == 0 && all_multiples(a->v_stride, n) &&
            all_multiples(a->k_page_stride, n) && all_multiples(a->v_page_stride, n) &&
            (!a->k_out_addr || (a->k_out_addr % 16 == 0 && all_multiples(a->k_out_stride, n)));
    else
      vec = vec && a->k_out_addr % 16 == 0 && all_multiples(a->k_out_stride, n);
  }
  if (a->dtype == AKILI_DTYPE_F32)
    return append ? launch_rope_vec<float, true>(di, r, vec, st) : launch_rope_vec<float, false>(di, r, vec, st);
  if (a->dtype == AKILI_DTYPE_F16)
    return append ? launch_rope_vec<__half, true>(di, r, vec, st) : launch_rope_vec<__half, false>(di, r, vec, st);
  return append ? launch_rope_vec<__nv_bfloat16, true>(di, r, vec, st)
                : launch_rope_vec<__nv_bfloat16, false>(di, r, vec, st);
}

int run_rope_table(const akili_rope_table_arg_t* a, cudaStream_t st) {
  if (!a) return AKILI_E_NULL_ARG;
  if (a->scaling > AKILI_ROPE_SCALE_RAMP || a->reserved) return AKILI_E_UNSUPPORTED;
  if (a->max_positions == 0 || a->max_positions > INT32_MAX || a->rot_dim == 0 || a->rot_dim % 2 ||
      a->rot_dim > kRopeMaxRot)
    return AKILI_E_SHAPE;
  const auto positive = [](double x) { return x > 0.0 && std::isfinite(x); };
  if (!positive(a->base) || !(a->amplitude >= 0.0) || !std::isfinite(a->amplitude)) return AKILI_E_UNSUPPORTED;
  if (a->scaling != AKILI_ROPE_SCALE_NONE && !positive(a->factor)) return AKILI_E_UNSUPPORTED;
  if (a->scaling == AKILI_ROPE_SCALE_BASE && a->rot_dim == 2) return AKILI_E_UNSUPPORTED;
  if (a->scaling >= AKILI_ROPE_SCALE_BANDS &&
      (!positive(a->original_positions) || !positive(a->low) || !positive(a->high) || a->high <= a->low))
    return AKILI_E_UNSUPPORTED;
  if (a->scaling == AKILI_ROPE_SCALE_RAMP && a->base <= 1.0) return AKILI_E_UNSUPPORTED;
  int rc;
  if ((rc = check_aligned({a->table_addr}, 4))) return rc;
  DevInfo di;
  if ((rc = device_info(&di))) return rc;
  RopeTableArgs t{};
  const int half = a->rot_dim / 2;
  const double r = a->rot_dim, two_pi = 6.283185307179586;
  double base = a->base;
  if (a->scaling == AKILI_ROPE_SCALE_BASE) base *= std::pow(a->factor, r / (r - 2.0));
  // RAMP: the pair that turns n times within original_positions is
  // i(n) = r ln(original / (2 pi n)) / (2 ln base)
  double lo = 0.0, hi = 0.0;
  if (a->scaling == AKILI_ROPE_SCALE_RAMP) {
    const auto pair_of = [&](double turns) {
      return r * std::log(a->original_positions / (two_pi * turns)) / (2.0 * std::log(base));
    };
    lo = std::max(std::floor(pair_of(a->high)), 0.0);
    hi = std::min(std::ceil(pair_of(a->low)), r - 1.0);
    if (hi <= lo) hi = lo + 0.001;
  }
  for (int i = 0; i < half; ++i) {
    double f = std::pow(base, -2.0 * i / r);
    if (a->scaling == AKILI_ROPE_SCALE_LINEAR) f /= a->factor;
    if (a->scaling == AKILI_ROPE_SCALE_BANDS) {
      const double turns = a->original_positions * f / two_pi;  // original / wavelength
      const double keep = std::min(std::max((turns - a->low) / (a->high - a->low), 0.0), 1.0);
      f = keep * f + (1.0 - keep) * f / a->factor;
    }
    if (a->scaling == AKILI_ROPE_SCALE_RAMP) {
      const double slow = std::min(std::max((i - lo) / (hi - lo), 0.0), 1.0);
      f = slow * f / a->factor + (1.0 - slow) * f;
    }
    t.freq[i] = f;
  }
  t.amplitude = a->amplitude != 0.0 ? a->amplitude
                : a->scaling == AKILI_ROPE_SCALE_RAMP && a->factor > 1.0 ? 0.1 * std::log(a->factor) + 1.0
                                                                         : 1.0;
  t.table = static_cast<float*>(W(a->table_addr));
  t.max_positions = a->max_positions;
  t.rot_dim = a->rot_dim;
  return launch_dependent(rope_table_kernel,
                          dim3(grid_for(di, static_cast<size_t>(a->max_positions) * half, 256, 8)), 256, 0, st, t);
}

// ------------------------------------------------------------------ cache --
int run_tree_mask(const akili_tree_mask_arg_t* a, cudaStream_t st) {
  if (!a) return AKILI_E_NULL_ARG;
  if (a->reserved) return AKILI_E_UNSUPPORTED;
  if (a->total_q > INT32_MAX - 128 || a->batch > INT32_MAX || a->mask_words == 0 || a->mask_words > 65536)
    return AKILI_E_SHAPE;
  if (a->total_q == 0) return AKILI_OK;
  if (a->batch == 0) return AKILI_E_SHAPE;
  int rc;
  if ((rc = check_aligned({a->parents_addr, a->cu_q_addr, a->mask_addr}, 4))) return rc;
  DevInfo di;
  if ((rc = device_info(&di))) return rc;
  return launch_dependent(tree_mask_kernel, dim3((a->total_q + 127) / 128), 128, 0, st,
                          static_cast<const int*>(P(a->parents_addr)), static_cast<const int*>(P(a->cu_q_addr)),
                          static_cast<unsigned int*>(W(a->mask_addr)), static_cast<int>(a->batch),
                          static_cast<int>(a->total_q), static_cast<int>(a->mask_words));
}

// Whether the int32s of `a` [rows, cols] share memory with the n at `p`.
bool ints_overlap(uint64_t a, uint64_t rows, uint64_t cols, int64_t row_stride, uint64_t p, uint64_t n) {
  if (a == 0 || p == 0) return false;
  for (uint64_t r = 0; r < rows; ++r) {
    const uint64_t row = a + 4 * static_cast<int64_t>(r) * row_stride;
    if (row < p + 4 * n && p < row + 4 * cols) return true;
  }
  return false;
}

template <typename U>
int launch_accept(AcceptArgs g, const akili_cache_accept_arg_t* a, cudaStream_t st) {
  g.vecs = static_cast<int>(a->head_dim * a->elem_bytes / sizeof(U));
  const int64_t cols = 2ll * a->kv_heads * g.vecs;
  const int share = static_cast<int>(std::min<int64_t>((cols + kAcceptThreads - 1) / kAcceptThreads, 1024));
  return launch_dependent(cache_accept_kernel<U>, dim3(share, a->batch, a->layers), kAcceptThreads, 0, st, g);
}

int run_cache_accept(const akili_cache_accept_arg_t* a, cudaStream_t st) {
  if (!a) return AKILI_E_NULL_ARG;
  if (a->reserved) return AKILI_E_UNSUPPORTED;
  if (a->elem_bytes != 1 && a->elem_bytes != 2 && a->elem_bytes != 4) return AKILI_E_DTYPE;
  if (a->page_size == 0 || a->kv_heads == 0 || a->head_dim == 0 || a->layers == 0 || a->max_pages == 0)
    return AKILI_E_SHAPE;
  if (a->layers > 65535 || a->batch > 65535 || a->kv_heads > 65536 || a->head_dim > 8192 ||
      a->page_size > INT32_MAX || a->num_pages > INT32_MAX || a->max_pages > INT32_MAX || a->max_accepted > INT32_MAX)
    return AKILI_E_SHAPE;
  if (a->batch == 0) return AKILI_OK;
  int rc;
  if ((rc = check_aligned({a->k_pages_addr, a->v_pages_addr}, a->elem_bytes))) return rc;
  if ((rc = check_aligned({a->page_table_addr, a->context_lens_addr, a->n_accepted_addr}, 4))) return rc;
  if (a->max_accepted && (rc = check_aligned({a->accepted_addr}, 4))) return rc;
  if (a->new_lens_addr % 4) return AKILI_E_ALIGN;
  if (!apart(a->k_page_stride, {a->layers, a->num_pages, a->page_size, a->kv_heads}) ||
      !apart(a->v_page_stride, {a->layers, a->num_pages, a->page_size, a->kv_heads}))
    return AKILI_E_SHAPE;
  // one block writes a sequence's new length while others still read what the moves go by
  const uint64_t out = a->new_lens_addr, n = a->batch;
  if (ints_overlap(a->context_lens_addr, 1, n, 0, out, n) || ints_overlap(a->n_accepted_addr, 1, n, 0, out, n) ||
      ints_overlap(a->accepted_addr, n, a->max_accepted, a->accepted_stride, out, n) ||
      ints_overlap(a->page_table_addr, n, a->max_pages, a->page_table_stride, out, n))
    return AKILI_E_UNSUPPORTED;
  DevInfo di;
  if ((rc = device_info(&di))) return rc;
  AcceptArgs g{};
  g.k = static_cast<char*>(W(a->k_pages_addr));
  g.v = static_cast<char*>(W(a->v_pages_addr));
  g.page_table = static_cast<const int*>(P(a->page_table_addr));
  g.context_lens = static_cast<const int*>(P(a->context_lens_addr));
  g.accepted = static_cast<const int*>(P(a->accepted_addr));
  g.n_accepted = static_cast<const int*>(P(a->n_accepted_addr));
  g.new_lens = static_cast<int*>(W(a->new_lens_addr));
  g.kv_heads = a->kv_heads; g.num_pages = a->num_pages; g.page_size = a->page_size;
  g.max_pages = a->max_pages; g.max_accepted = a->max_accepted;
  uint64_t bits = a->k_pages_addr | a->v_pages_addr | (a->head_dim * a->elem_bytes);
  for (int i = 0; i < 4; ++i) {
    g.k_st[i] = a->k_page_stride[i] * a->elem_bytes;
    g.v_st[i] = a->v_page_stride[i] * a->elem_bytes;
    bits |= static_cast<uint64_t>(g.k_st[i] | g.v_st[i]);
  }
  g.table_stride = a->page_table_stride;
  g.acc_stride = a->accepted_stride;
  // 16-byte moves where every head row starts on 16 bytes, else element by element
  if (bits % 16 == 0) return launch_accept<uint4>(g, a, st);
  if (a->elem_bytes == 4) return launch_accept<uint32_t>(g, a, st);
  if (a->elem_bytes == 2) return launch_accept<uint16_t>(g, a, st);
  return launch_accept<uint8_t>(g, a, st);
}

// -------------------------------------------------------------- attention --
// Keys and values of the key heads that are scheduled together: half of L2.
constexpr uint64_t kPromptChunkBytes = 64ull << 20;

int check_heads(uint32_t dtype, uint32_t hq, uint32_t hk, uint32_t d, float scale) {
  if (dtype != AKILI_DTYPE_F16 && dtype != AKILI_DTYPE_BF16) return AKILI_E_DTYPE;
  if (hq == 0 || hk == 0 || hq % hk || d == 0 || d % 8) return AKILI_E_SHAPE;
  if (d > 128 || hq > 65535) return AKILI_E_UNSUPPORTED;
  if (!(scale >= 0.0f) || !std::isfinite(scale)) return AKILI_E_UNSUPPORTED;
  return AKILI_OK;
}

// The tile loads need positive strides (a broadcast axis has 0); the stride of
// an axis of one entry is never used.
template <size_t n>
bool loadable(const int64_t (&stride)[n], const uint64_t (&extent)[n]) {
  for (size_t i = 0; i < n; ++i)
    if (extent[i] > 1 && stride[i] <= 0) return false;
  return true;
}

float scale_log2_of(float scale, uint32_t d) {
  return (scale != 0.0f ? scale : 1.0f / std::sqrt(static_cast<float>(d))) * 1.4426950408889634f;
}

// [d3][d2][d1][d0] tensor of 16-bit values with these strides (elements), box
// [box3][box2][box1][64], 128-byte swizzle.  The stride of an axis of one entry is never used.
bool map_heads(CUtensorMap* m, const void* ptr, uint32_t dtype, int rank, const uint64_t (&dim)[4],
               const int64_t (&stride)[3], const uint32_t (&box)[3]) {
  EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  cuuint64_t dims[4], strides[3];
  cuuint32_t boxes[4] = {64, box[0], box[1], box[2]}, es[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) dims[i] = dim[i];
  for (int i = 0; i + 1 < rank; ++i) strides[i] = dim[i + 1] == 1 ? (dim[0] * 2 + 15) / 16 * 16 : stride[i] * 2;
  return enc(m, dtype == AKILI_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank,
             const_cast<void*>(ptr), dims, strides, boxes, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// The attribute that grants a kernel its shared memory, once per device; `done`
// belongs to one kernel.
struct SmemGrant {
  std::mutex mu;
  std::map<int, bool> done;
  int operator()(const void* kern, int bytes) {
    int dev = 0;
    cudaGetDevice(&dev);
    std::lock_guard<std::mutex> lock(mu);
    if (done[dev]) return AKILI_OK;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
      cudaGetLastError();
      return AKILI_E_LAUNCH;
    }
    done[dev] = true;
    return AKILI_OK;
  }
};

// Packing of a token's heads into the rows of a 128-row tile.
void pack_heads(ServingArgs& g) {
  g.pack = g.group;
  while (g.pack > kSvRows || g.group % g.pack) --g.pack;
  g.head_groups = g.q_heads / g.pack;
  g.groups_per_kv = g.group / g.pack;
  g.tile_tokens = kSvRows / g.pack;
}

// A tile's queries: tile_tokens tokens x pack heads x 64 columns.
bool map_queries(CUtensorMap* m, const ServingArgs& g, uint32_t dtype, const int64_t (&q_stride)[2]) {
  return map_heads(m, g.q, dtype, 3,
                   {static_cast<uint64_t>(g.head_dim), static_cast<uint64_t>(g.q_heads),
                    static_cast<uint64_t>(g.total_q), 1},
                   {q_stride[1], q_stride[0], 0},
                   {static_cast<uint32_t>(g.pack), static_cast<uint32_t>(g.tile_tokens), 1});
}

template <int DP, typename T, bool kPair>
int launch_prompt_form(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const ServingArgs& g,
                       int blocks, cudaStream_t st) {
  auto kern = serving_attention_kernel<DP, T, false, kPair>;
  constexpr int smem = SvSmem<DP, kPair>::kBytes;
  static SmemGrant grant;
  if (const int rc = grant(reinterpret_cast<const void*>(kern), smem)) return rc;
  return launch_dependent(kern, dim3(blocks), kSvThreads, smem, st, tq, tk, tv, g);
}

// Two tiles a CTA, or one where even that many CTAs run at once: one tile
// reads the keys twice as often, but has half the work one after another
// (440 + 2698 tokens, 4 heads: 50 -> 31 us; 24 short sequences in two waves of
// single tiles: 12.4 -> 13.4).
template <int DP, typename T>
int launch_prompt(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const ServingArgs& g, int sms,
                  cudaStream_t st) {
  const auto blocks = [&](int tiles) {  // at most one tile (pair) of a sequence is not full
    return (static_cast<int64_t>(g.total_q) / (tiles * g.tile_tokens) + g.batch) * g.head_groups;
  };
  if (blocks(1) > INT32_MAX) return AKILI_E_SHAPE;
  return blocks(1) > sms ? launch_prompt_form<DP, T, true>(tq, tk, tv, g, static_cast<int>(blocks(2)), st)
                         : launch_prompt_form<DP, T, false>(tq, tk, tv, g, static_cast<int>(blocks(1)), st);
}

// The attention over a cache with items of kTileRows rows, then the join of
// its cut items.
template <int DP, typename T, int kTileRows>
int launch_cache(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const ServingArgs& g, int blocks,
                 cudaStream_t st) {
  static SmemGrant grant;
  int rc;
  if constexpr (kTileRows >= kSvRows) {
    constexpr bool kPair = kTileRows > kSvRows;
    auto kern = serving_attention_kernel<DP, T, true, kPair>;
    constexpr int smem = SvSmem<DP, kPair>::kBytes;
    if ((rc = grant(reinterpret_cast<const void*>(kern), smem))) return rc;
    rc = launch_dependent(kern, dim3(blocks), kSvThreads, smem, st, tq, tk, tv, g);
  } else {
    auto kern = decode_attention_kernel<DP, T, kTileRows>;
    constexpr int smem = DcSmem<DP, kTileRows>::kBytes;
    if ((rc = grant(reinterpret_cast<const void*>(kern), smem))) return rc;
    rc = launch_dependent(kern, dim3(blocks), kDcThreads, smem, st, tk, tv, g);
  }
  if (rc) return rc;
  const dim3 join(blocks, kSvJoinSplit<kTileRows, DP>);
  if constexpr (kTileRows >= kSvRows)
    return launch_dependent(attention_join_rows_kernel<DP, T, kTileRows>, join, kSvJoinThreads, 0, st, g);
  else
    return launch_dependent(attention_join_kernel<DP, T, kTileRows>, join, kSvJoinThreads, 0, st, g);
}

template <int DP, typename T>
int launch_cache_rows(int rows, const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv,
                      const ServingArgs& g, int blocks, cudaStream_t st) {
  switch (rows) {
    case 16: return launch_cache<DP, T, 16>(tq, tk, tv, g, blocks, st);
    case 32: return launch_cache<DP, T, 32>(tq, tk, tv, g, blocks, st);
    case 64: return launch_cache<DP, T, 64>(tq, tk, tv, g, blocks, st);
    case 128: return launch_cache<DP, T, 128>(tq, tk, tv, g, blocks, st);
    default: return launch_cache<DP, T, 256>(tq, tk, tv, g, blocks, st);
  }
}

int run_prompt_attention(const akili_prompt_attention_arg_t* a, cudaStream_t st) {
  if (!a) return AKILI_E_NULL_ARG;
  int rc;
  if ((rc = check_heads(a->dtype, a->q_heads, a->kv_heads, a->head_dim, a->softmax_scale))) return rc;
  if (a->causal > 1 || a->reserved) return AKILI_E_UNSUPPORTED;
  if (a->total_q > (1u << 30) || a->total_k > (1u << 30) || a->batch > (1u << 20)) return AKILI_E_SHAPE;
  if (a->batch == 0 && a->total_q) return AKILI_E_SHAPE;
  if (a->total_q == 0) return AKILI_OK;
  if ((rc = check_ptrs({a->q_addr, a->o_addr}))) return rc;
  if (a->total_k && (rc = check_ptrs({a->k_addr, a->v_addr}))) return rc;
  if ((rc = check_aligned({a->cu_q_addr, a->cu_k_addr}, 4))) return rc;
  if (a->lse_addr % 4) return AKILI_E_ALIGN;
  if (!all_multiples(a->q_stride, 8) || !all_multiples(a->k_stride, 8) || !all_multiples(a->v_stride, 8) ||
      !all_multiples(a->o_stride, 8))
    return AKILI_E_ALIGN;
  if (!loadable(a->q_stride, {a->total_q, a->q_heads}) || !loadable(a->k_stride, {a->total_k, a->kv_heads}) ||
      !loadable(a->v_stride, {a->total_k, a->kv_heads}) || !loadable(a->o_stride, {a->total_q, a->q_heads}))
    return AKILI_E_SHAPE;
  DevInfo di;
  if ((rc = device_info(&di))) return rc;
  const uint64_t group = a->q_heads / a->kv_heads;
  if (a->total_q * group > (1u << 30)) return AKILI_E_SHAPE;
  ServingArgs g{};
  g.q = P(a->q_addr); g.o = W(a->o_addr);
  g.lse = static_cast<float*>(W(a->lse_addr));
  g.cu_q = static_cast<const int*>(P(a->cu_q_addr));
  g.cu_k = static_cast<const int*>(P(a->cu_k_addr));
  g.q_heads = a->q_heads; g.kv_heads = a->kv_heads; g.group = static_cast<int>(group);
  g.head_dim = a->head_dim; g.batch = a->batch;
  g.total_q = a->total_q; g.total_k = a->total_k; g.causal = a->causal;
  pack_heads(g);
  g.scale_log2 = scale_log2_of(a->softmax_scale, a->head_dim);
  for (int i = 0; i < 2; ++i) { g.q_st[i] = a->q_stride[i]; g.o_st[i] = a->o_stride[i]; }
  const uint64_t per_head = static_cast<uint64_t>(a->total_k) * a->head_dim * 4;  // bytes of K and V
  g.chunk_heads = static_cast<int>(std::min<uint64_t>(
      std::max<uint64_t>(kPromptChunkBytes / std::max<uint64_t>(per_head, 1), 1) * g.groups_per_kv, g.head_groups));
  // without any key the maps are never used; they are made over q then
  const bool keys = a->total_k > 0;
  const uint64_t dim[4] = {a->head_dim, keys ? a->kv_heads : 1, keys ? a->total_k : 1, 1};
  CUtensorMap tq, tk, tv;
  if (!map_heads(&tk, P(keys ? a->k_addr : a->q_addr), a->dtype, 3, dim, {a->k_stride[1], a->k_stride[0], 0},
                 {1, kSvKeys, 1}) ||
      !map_heads(&tv, P(keys ? a->v_addr : a->q_addr), a->dtype, 3, dim, {a->v_stride[1], a->v_stride[0], 0},
                 {1, kSvKeys, 1}) ||
      !map_queries(&tq, g, a->dtype, a->q_stride))
    return AKILI_E_LAUNCH;
  const int n = di.sms;
  if (a->dtype == AKILI_DTYPE_BF16)
    return g.head_dim <= 64 ? launch_prompt<64, __nv_bfloat16>(tq, tk, tv, g, n, st)
                            : launch_prompt<128, __nv_bfloat16>(tq, tk, tv, g, n, st);
  return g.head_dim <= 64 ? launch_prompt<64, __half>(tq, tk, tv, g, n, st) : launch_prompt<128, __half>(tq, tk, tv, g, n, st);
}

int check_tree(const akili_tree_attention_arg_t* a) {
  if (!a) return AKILI_E_NULL_ARG;
  int rc;
  if ((rc = check_heads(a->dtype, a->q_heads, a->kv_heads, a->head_dim, a->softmax_scale))) return rc;
  if (a->reserved) return AKILI_E_UNSUPPORTED;
  if (a->page_size == 0 || a->page_size % 8 || a->page_size > (1u << 20) || a->max_pages == 0 || a->num_pages == 0)
    return AKILI_E_SHAPE;
  if (a->total_q > (1u << 30) || a->batch > (1u << 20) || a->num_pages > INT32_MAX || a->max_pages > INT32_MAX ||
      static_cast<uint64_t>(a->max_pages) * a->page_size > (1u << 30) || a->mask_words > 65536)
    return AKILI_E_SHAPE;
  if (a->batch == 0 && a->total_q) return AKILI_E_SHAPE;
  if (static_cast<uint64_t>(a->total_q) * (a->q_heads / a->kv_heads) > (1u << 30)) return AKILI_E_SHAPE;
  return AKILI_OK;
}

// Rows of an item (tokens times grouped heads of one key head): the smallest
// form that holds the mean of the sequences.  The host does not know the
// single lengths; a longer sequence takes several items.
int tree_tile_rows(const akili_tree_attention_arg_t* a) {
  const uint64_t rows = static_cast<uint64_t>(a->total_q) * (a->q_heads / a->kv_heads);
  int form = 16;
  while (form < 2 * kSvRows && rows > static_cast<uint64_t>(form) * a->batch) form *= 2;
  return form;
}

// Two parts (O, m, l) for each share of the line of key blocks, then (row
// forms) what the join has to know of each share.
size_t tree_parts_bytes(const DevInfo& di, const akili_tree_attention_arg_t* a) {
  return 2ull * di.sms * tree_tile_rows(a) * ((a->head_dim <= 64 ? 64 : 128) + 2) * sizeof(float);
}
size_t tree_workspace_bytes(const DevInfo& di, const akili_tree_attention_arg_t* a) {
  return tree_parts_bytes(di, a) + (tree_tile_rows(a) >= kSvRows ? 2 * di.sms * sizeof(int4) : 0);
}

int run_tree_attention(const akili_tree_attention_arg_t* a, cudaStream_t st) {
  int rc;
  if ((rc = check_tree(a))) return rc;
  if (a->total_q == 0) return AKILI_OK;
  if ((rc = check_ptrs({a->q_addr, a->k_pages_addr, a->v_pages_addr, a->o_addr}))) return rc;
  if ((rc = check_aligned({a->page_table_addr, a->context_lens_addr, a->cu_q_addr}, 4))) return rc;
  if (a->lse_addr % 4 || a->mask_addr % 4) return AKILI_E_ALIGN;
  if (a->mask_addr && a->mask_words == 0) return AKILI_E_SHAPE;
  if (!all_multiples(a->q_stride, 8) || !all_multiples(a->o_stride, 8) || !all_multiples(a->k_page_stride, 8) ||
      !all_multiples(a->v_page_stride, 8))
    return AKILI_E_ALIGN;
  if (!loadable(a->q_stride, {a->total_q, a->q_heads}) ||
      !loadable(a->k_page_stride, {a->num_pages, a->page_size, a->kv_heads}) ||
      !loadable(a->v_page_stride, {a->num_pages, a->page_size, a->kv_heads}) ||
      !loadable(a->o_stride, {a->total_q, a->q_heads}))
    return AKILI_E_SHAPE;
  DevInfo di;
  if ((rc = device_info(&di))) return rc;
  Mode md;
  md.workspace = W(a->workspace);
  md.workspace_bytes = a->workspace ? a->workspace_bytes : 0;
  char* parts = nullptr;
  if ((rc = acquire_scratch(md, tree_workspace_bytes(di, a), st, &parts))) return rc;
  ServingArgs g{};
  g.q = P(a->q_addr); g.o = W(a->o_addr);
  g.lse = static_cast<float*>(W(a->lse_addr));
  g.cu_q = static_cast<const int*>(P(a->cu_q_addr));
  g.ctx = static_cast<const int*>(P(a->context_lens_addr));
  g.page_table = static_cast<const int*>(P(a->page_table_addr));
  g.mask = static_cast<const unsigned int*>(P(a->mask_addr));
  g.parts = reinterpret_cast<float*>(parts);
  g.cuts = reinterpret_cast<int4*>(parts + tree_parts_bytes(di, a));
  g.q_heads = a->q_heads; g.kv_heads = a->kv_heads; g.group = static_cast<int>(a->q_heads / a->kv_heads);
  g.head_dim = a->head_dim; g.batch = a->batch; g.total_q = a->total_q;
  g.num_pages = a->num_pages; g.page_size = a->page_size; g.max_pages = a->max_pages; g.mask_words = a->mask_words;
  g.box_rows = 8;
  while (g.box_rows < kSvKeys && a->page_size % (2 * g.box_rows) == 0) g.box_rows *= 2;
  g.scale_log2 = scale_log2_of(a->softmax_scale, a->head_dim);
  for (int i = 0; i < 2; ++i) { g.q_st[i] = a->q_stride[i]; g.o_st[i] = a->o_stride[i]; }
  g.table_stride = a->page_table_stride;
  g.mask_stride = a->mask_stride;
  const int rows = tree_tile_rows(a);
  if (rows >= kSvRows) {
    pack_heads(g);
  } else {  // the few-row form takes a group's heads whole
    g.pack = g.group;
    g.head_groups = g.kv_heads;
    g.groups_per_kv = 1;
    g.tile_tokens = 1;
  }
  const uint64_t dim[4] = {a->head_dim, a->page_size, a->kv_heads, a->num_pages};
  CUtensorMap tq = {}, tk, tv;
  if (!map_heads(&tk, P(a->k_pages_addr), a->dtype, 4, dim,
                 {a->k_page_stride[1], a->k_page_stride[2], a->k_page_stride[0]}, {static_cast<uint32_t>(g.box_rows), 1, 1}) ||
      !map_heads(&tv, P(a->v_pages_addr), a->dtype, 4, dim,
                 {a->v_page_stride[1], a->v_page_stride[2], a->v_page_stride[0]}, {static_cast<uint32_t>(g.box_rows), 1, 1}) ||
      (rows >= kSvRows && !map_queries(&tq, g, a->dtype, a->q_stride)))
    return AKILI_E_LAUNCH;
  if (a->dtype == AKILI_DTYPE_BF16)
    return g.head_dim <= 64 ? launch_cache_rows<64, __nv_bfloat16>(rows, tq, tk, tv, g, di.sms, st)
                            : launch_cache_rows<128, __nv_bfloat16>(rows, tq, tk, tv, g, di.sms, st);
  return g.head_dim <= 64 ? launch_cache_rows<64, __half>(rows, tq, tk, tv, g, di.sms, st)
                          : launch_cache_rows<128, __half>(rows, tq, tk, tv, g, di.sms, st);
}

}  // namespace

extern "C" {

int akili_rope(const akili_rope_arg_t* a, akili_stream_t s) { return run_rope(a, false, S(s)); }
int akili_rope_append(const akili_rope_arg_t* a, akili_stream_t s) { return run_rope(a, true, S(s)); }
int akili_rope_table(const akili_rope_table_arg_t* a, akili_stream_t s) { return run_rope_table(a, S(s)); }
int akili_prompt_attention(const akili_prompt_attention_arg_t* a, akili_stream_t s) {
  return run_prompt_attention(a, S(s));
}
int akili_tree_attention(const akili_tree_attention_arg_t* a, akili_stream_t s) { return run_tree_attention(a, S(s)); }
int akili_tree_attention_workspace(const akili_tree_attention_arg_t* a, uint64_t* bytes) {
  if (!bytes) return AKILI_E_NULL_ARG;
  const int rc = check_tree(a);
  if (rc) return rc;
  DevInfo di;
  if (const int no = device_info(&di)) return no;
  *bytes = tree_workspace_bytes(di, a);
  return AKILI_OK;
}
int akili_tree_mask(const akili_tree_mask_arg_t* a, akili_stream_t s) { return run_tree_mask(a, S(s)); }
int akili_cache_accept(const akili_cache_accept_arg_t* a, akili_stream_t s) { return run_cache_accept(a, S(s)); }

}  // extern "C"
