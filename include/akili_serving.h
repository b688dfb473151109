/*
 * akili_serving.h — the serving operators of the B200 backend: what a
 * transformer layer needs next to the projections of akili.h to answer
 * prompts and to decode with a paged key/value cache.
 *
 *   akili_rope              rotary positions of queries and keys
 *   akili_rope_append       the same, the rotated keys and the values written
 *                           into the pages of a cache
 *   akili_rope_table        the cos/sin table both read, with the usual
 *                           scalings for contexts longer than the trained one
 *   akili_prompt_attention  causal attention over packed prompts of different
 *                           lengths, grouped heads
 *   akili_tree_attention    attention of new tokens (one per sequence, a
 *                           chunk, or a tree of drafted tokens) over the cache
 *   akili_tree_mask         the ancestor bits of drafted trees from parents
 *   akili_cache_accept      compaction: the accepted branch's cache entries
 *                           move to the end of the sure context
 *
 * Calls are asynchronous on `stream` and return AKILI_OK or an AKILI_E_*
 * code, like those of akili.h; arguments are checked before any CUDA call.
 * The caller owns every buffer.  Strides are in elements; the innermost
 * (head_dim) axis is contiguous; what is written has no stride of 0 along an
 * axis of more than one entry.  Lengths, indices and masks live on the
 * device and are not read by the host: one that is out of range makes no
 * access outside the buffers: lengths are clamped to what the buffers hold,
 * entries are skipped, and where an entry's comment says so
 * AKILI_STATUS_BAD_INDEX is recorded for akili_device_status().
 */
#ifndef AKILI_SERVING_H_
#define AKILI_SERVING_H_

#include "akili.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A third element type, for the entries of this header only. */
#define AKILI_DTYPE_BF16 2u

#define AKILI_STATUS_BAD_INDEX 0x2001u

/* ---- rotary positions ---------------------------------------------------- */
#define AKILI_ROPE_INTERLEAVED 1u /* pairs (2i, 2i+1); default (i, i + rot_dim/2) */
#define AKILI_ROPE_INVERSE     2u /* rotate by -angle: the gradient of the rotation */

/* y1 = x1 cos - x2 sin, y2 = x2 cos + x1 sin over the first rot_dim values of
 * every head of every token, computed in fp32 and rounded once; the rest of
 * the head is copied.  cos | sin = table[positions[token]].
 * q [tokens, q_heads, head_dim], k [tokens, k_heads, head_dim]; either head
 * count may be 0.  An output may be its input (in place); other overlaps are
 * not allowed.  A token whose position is outside [0, max_positions) is
 * skipped and recorded. */
typedef struct {
  uint32_t dtype; /* of q, k, v, the outputs and the pages: F32, F16 or BF16 */
  uint32_t flags; /* AKILI_ROPE_* */
  uint32_t tokens, q_heads, k_heads, head_dim;
  uint32_t rot_dim;       /* even, 0 < rot_dim <= head_dim */
  uint32_t max_positions; /* rows of the table */
  uint64_t q_addr, k_addr, q_out_addr;
  uint64_t k_out_addr;     /* akili_rope_append: optional, the rotated k once more (for a prompt's own attention) */
  uint64_t positions_addr; /* int32 [tokens] */
  uint64_t table_addr;     /* fp32 [max_positions, rot_dim]: rot_dim/2 cosines, then the sines */
  int64_t  q_stride[2], k_stride[2], q_out_stride[2], k_out_stride[2]; /* token, head */
  /* akili_rope_append only: v [tokens, k_heads, head_dim] and the rotated k go
   * to row slots[token] = page * page_size + offset of the pages
   * [num_pages, page_size, k_heads, head_dim].  A slot of -1 marks padding:
   * nothing is written for its k and v (nor for one outside the pages, which
   * is recorded).  Slots are distinct. */
  uint64_t v_addr, slots_addr; /* slots: int64 [tokens] */
  uint64_t k_pages_addr, v_pages_addr;
  uint32_t num_pages, page_size;
  int64_t  v_stride[2];                        /* token, head */
  int64_t  k_page_stride[3], v_page_stride[3]; /* page, token, head */
} akili_rope_arg_t;

int akili_rope(const akili_rope_arg_t* arg, akili_stream_t stream);
int akili_rope_append(const akili_rope_arg_t* arg, akili_stream_t stream);

/* table[p][i] = amplitude * cos(p f_i), table[p][rot_dim/2 + i] = amplitude *
 * sin(p f_i), evaluated in fp64 and rounded to fp32; f_i = base^(-2i/rot_dim)
 * changed by `scaling`:
 *   NONE    as is
 *   LINEAR  f_i / factor (position interpolation)
 *   BASE    base * factor^(rot_dim / (rot_dim - 2)) in place of base (NTK-aware)
 *   BANDS   by wavelength w = 2 pi / f_i: f_i / factor where
 *           w > original_positions / low, f_i where w < original_positions /
 *           high, a linear blend in original_positions / w between
 *   RAMP    by rotations within original_positions (YaRN): f_i where the pair
 *           turns more than `high` times, f_i / factor where it turns less
 *           than `low` times, a linear ramp in i between (its ends rounded
 *           outward to whole i)
 * amplitude 0 means 1, and 0.1 ln(factor) + 1 for RAMP with factor > 1. */
#define AKILI_ROPE_SCALE_NONE   0u
#define AKILI_ROPE_SCALE_LINEAR 1u
#define AKILI_ROPE_SCALE_BASE   2u
#define AKILI_ROPE_SCALE_BANDS  3u
#define AKILI_ROPE_SCALE_RAMP   4u
typedef struct {
  uint32_t max_positions, rot_dim; /* rot_dim even, at most 256 */
  uint32_t scaling;
  uint32_t reserved; /* 0 */
  double   base, factor, original_positions, low, high, amplitude;
  uint64_t table_addr; /* fp32 [max_positions, rot_dim] */
} akili_rope_table_arg_t;

int akili_rope_table(const akili_rope_table_arg_t* arg, akili_stream_t stream);

/* ---- attention over packed prompts --------------------------------------- */
/* Sequence b has the query rows cu_q[b] .. cu_q[b+1]-1 and the key rows
 * cu_k[b] .. cu_k[b+1]-1.  With n queries and m keys, query i sees key j when
 * j < m and, with causal = 1, j <= i + m - n (the last query sees every key).
 *   o_i = sum_j softmax_j(softmax_scale q_i.k_j) v_j
 * over the visible keys; a row that sees none gives 0 (and lse -inf).  Query
 * head h reads key head h / (q_heads / kv_heads).  q, o [total_q, q_heads,
 * head_dim], k, v [total_k, kv_heads, head_dim].  Scores, maxima, sums and the
 * output accumulate in fp32; the weights are rounded to the element type for
 * their product with v.  Keys a row does not see may hold anything; a value
 * row that some query of its 128-query tile does not see has to be finite
 * (rows outside the sequence may hold anything). */
typedef struct {
  uint32_t dtype; /* F16 or BF16 */
  uint32_t q_heads, kv_heads, head_dim; /* q_heads % kv_heads == 0; head_dim % 8 == 0, <= 128 */
  uint32_t batch, total_q, total_k;
  uint32_t causal;        /* 0 or 1 */
  float    softmax_scale; /* 0: head_dim^-0.5 (the smallest positive float: equal weights) */
  uint32_t reserved;      /* 0 */
  uint64_t q_addr, k_addr, v_addr, o_addr;
  uint64_t lse_addr;              /* optional fp32 [total_q, q_heads]: log of the row's sum of exponentials */
  uint64_t cu_q_addr, cu_k_addr;  /* int32 [batch + 1], ascending from 0 */
  int64_t  q_stride[2], k_stride[2], v_stride[2], o_stride[2]; /* token, head; multiples of 8, positive */
} akili_prompt_attention_arg_t;

int akili_prompt_attention(const akili_prompt_attention_arg_t* arg, akili_stream_t stream);

/* ---- attention of new tokens over a paged cache --------------------------- */
/* Sequence b has the new tokens (query rows) cu_q[b] .. cu_q[b+1]-1, n of
 * them, whose keys and values are already in the cache behind its
 * context_lens[b] sure tokens: entry j of the sequence is row j % page_size of
 * page page_table[b][j / page_size].  Every new token sees the whole context,
 * and the new token j when bit j % 32 of word j / 32 of its mask row is set
 * (mask_addr 0: when j is not after it, as for a single token or a chunk of a
 * prompt).  Otherwise as akili_prompt_attention.  Pages or page rows past a
 * sequence's end may hold anything; table entries past it are not read.  A page
 * index outside [0, num_pages) reads as a page of zeros; a sequence is clamped
 * to max_pages * page_size entries; both are recorded.
 * Without a workspace the call uses the scratch of its stream.  A graph that
 * was captured so keeps that memory for good, and its replays have to be
 * ordered with the stream's other calls; with a workspace of its own it is
 * independent of them. */
typedef struct {
  uint32_t dtype; /* F16 or BF16 */
  uint32_t q_heads, kv_heads, head_dim;
  uint32_t batch, total_q;
  uint32_t num_pages, page_size; /* page_size a multiple of 8 */
  uint32_t max_pages;            /* columns of the page table */
  uint32_t mask_words;           /* 32-bit words of a mask row (0 without a mask) */
  float    softmax_scale;        /* 0: head_dim^-0.5 */
  uint32_t reserved;             /* 0 */
  uint64_t q_addr, k_pages_addr, v_pages_addr, o_addr;
  uint64_t lse_addr;          /* optional fp32 [total_q, q_heads] */
  uint64_t page_table_addr;   /* int32 [batch, max_pages] */
  uint64_t context_lens_addr; /* int32 [batch] */
  uint64_t cu_q_addr;         /* int32 [batch + 1], ascending from 0 */
  uint64_t mask_addr;         /* optional int32 [total_q, mask_words] */
  uint64_t workspace, workspace_bytes; /* optional; akili_tree_attention_workspace() bytes, 256-byte aligned */
  int64_t  q_stride[2], o_stride[2];           /* token, head; multiples of 8, positive */
  int64_t  k_page_stride[3], v_page_stride[3]; /* page, token, head; multiples of 8, positive */
  int64_t  page_table_stride, mask_stride;     /* row strides */
} akili_tree_attention_arg_t;

int akili_tree_attention(const akili_tree_attention_arg_t* arg, akili_stream_t stream);
/* Bytes of workspace that any call with these head counts and sizes uses on
 * the current device (it does not depend on the lengths). */
int akili_tree_attention_workspace(const akili_tree_attention_arg_t* arg, uint64_t* bytes);

/* mask row of node i of sequence b: the bits of i and of its ancestors.
 * parents [total_q] holds, for each node, its parent's index within its
 * sequence, smaller than its own, or -1 (anything else ends the walk and is
 * recorded, as is a node past the mask's words). */
typedef struct {
  uint32_t batch, total_q, mask_words, reserved;
  uint64_t parents_addr; /* int32 [total_q] */
  uint64_t cu_q_addr;    /* int32 [batch + 1] */
  uint64_t mask_addr;    /* int32 [total_q, mask_words], contiguous */
} akili_tree_mask_arg_t;

int akili_tree_mask(const akili_tree_mask_arg_t* arg, akili_stream_t stream);

/* ---- compaction after a draft was verified -------------------------------- */
/* In every layer, the cache entry context_lens[b] + accepted[b][i] of sequence
 * b moves to context_lens[b] + i, for i < n_accepted[b]; accepted[b] ascends
 * (so accepted[b][i] >= i; an entry that does not, or that lies outside the
 * pages, is skipped and recorded).  new_lens[b] = context_lens[b] + n_accepted[b].
 * Pages are [layers, num_pages, page_size, kv_heads, head_dim]; sequences do
 * not share the pages that are written. */
typedef struct {
  uint32_t elem_bytes; /* bytes of an element: 1, 2 or 4 */
  uint32_t layers, batch, kv_heads, head_dim;
  uint32_t num_pages, page_size, max_pages;
  uint32_t max_accepted; /* columns of accepted */
  uint32_t reserved;     /* 0 */
  uint64_t k_pages_addr, v_pages_addr;
  uint64_t page_table_addr;   /* int32 [batch, max_pages] */
  uint64_t context_lens_addr; /* int32 [batch] */
  uint64_t accepted_addr;     /* int32 [batch, max_accepted] */
  uint64_t n_accepted_addr;   /* int32 [batch] */
  uint64_t new_lens_addr;     /* optional int32 [batch]; shares no memory with the four above */
  int64_t  k_page_stride[4], v_page_stride[4]; /* layer, page, token, head */
  int64_t  page_table_stride, accepted_stride;
} akili_cache_accept_arg_t;

int akili_cache_accept(const akili_cache_accept_arg_t* arg, akili_stream_t stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* AKILI_SERVING_H_ */
