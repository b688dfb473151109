// serving_attention.cuh — attention of packed queries over packed keys or
// over a paged cache:
//
//   o_i = sum_j softmax_j(scale q_i.k_j) v_j   over the keys j that i sees
#pragma once
#include "cache.cuh"
#include "rope.cuh"
#include "sm100.cuh"

namespace akili {

struct ServingArgs {
  const void *q, *k, *v;
  void* o;
  float* lse;
  const int* cu_q;
  const int* cu_k;       // packed keys
  const int* ctx;        // paged keys
  const int* page_table;
  const unsigned int* mask;
  int q_heads, kv_heads, head_dim, batch, total_q, total_k, causal;
  int num_pages, page_size, max_pages, mask_words;
  float scale_log2;
  long long q_st[2], o_st[2], k_st[3], v_st[3];  // packed: k_st = 0, token, head
  long long table_stride, mask_stride;
};

// One warp per (token, head): a key at a time, the running maximum and sum of
// the softmax in every lane, four values of the head per lane.
template <typename T, bool kPaged>
__global__ void __launch_bounds__(128) attention_rows_kernel(const ServingArgs a) {
  const long long w = blockIdx.x * 4ll + (threadIdx.x >> 5);
  if (w >= static_cast<long long>(a.total_q) * a.q_heads) return;
  const int t = static_cast<int>(w / a.q_heads), h = static_cast<int>(w % a.q_heads);
  if (t < a.cu_q[0] || t >= a.cu_q[a.batch]) return;
  const int lane = threadIdx.x & 31;
  const int b = find_sequence(a.cu_q, a.batch, t);
  const int n = min(a.cu_q[b + 1], a.total_q) - a.cu_q[b];
  const int i = t - a.cu_q[b];
  const int hk = h / (a.q_heads / a.kv_heads);
  const int d = lane * 4;
  const bool on = d < a.head_dim;
  int m, sure, k0 = 0;
  if constexpr (kPaged) {
    sure = max(a.ctx[b], 0);
    m = sure + n;
    if (static_cast<long long>(m) > static_cast<long long>(a.max_pages) * a.page_size) {
      m = a.max_pages * a.page_size;
      record_bad_index();
    }
  } else {
    k0 = max(a.cu_k[b], 0);
    m = max(min(a.cu_k[b + 1], a.total_k) - k0, 0);
    sure = m - n;
  }
  const int last = (kPaged ? a.mask != nullptr : !a.causal) ? m : min(m, sure + i + 1);
  float q[4] = {}, o[4] = {};
  const T* qp = static_cast<const T*>(a.q) + t * a.q_st[0] + h * a.q_st[1];
  if (on)
    for (int x = 0; x < 4; ++x) q[x] = to_f32(qp[d + x]);
  float top = -INFINITY, total = 0.0f;
  for (int j = 0; j < last; ++j) {
    long long ko, vo;
    if constexpr (kPaged) {
      if (a.mask != nullptr && j >= sure) {
        const int node = j - sure;
        if (node / 32 >= a.mask_words || !((a.mask[t * a.mask_stride + node / 32] >> (node % 32)) & 1)) continue;
      }
      const int page = a.page_table[b * a.table_stride + j / a.page_size];
      if (page < 0 || page >= a.num_pages) {  // reads as zeros
        record_bad_index();
        const float next = fmaxf(top, 0.0f), keep = exp2f(top - next);
        total = total * keep + exp2f(-next);
        for (int x = 0; x < 4; ++x) o[x] *= keep;
        top = next;
        continue;
      }
      ko = page * a.k_st[0] + (j % a.page_size) * a.k_st[1];
      vo = page * a.v_st[0] + (j % a.page_size) * a.v_st[1];
    } else {
      ko = (k0 + j) * a.k_st[1];
      vo = (k0 + j) * a.v_st[1];
    }
    const T* kp = static_cast<const T*>(a.k) + ko + hk * a.k_st[2];
    const T* vp = static_cast<const T*>(a.v) + vo + hk * a.v_st[2];
    float s = 0.0f, v[4] = {};
    if (on)
      for (int x = 0; x < 4; ++x) {
        s += q[x] * to_f32(kp[d + x]);
        v[x] = to_f32(vp[d + x]);
      }
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.scale_log2;
    const float next = fmaxf(top, s);
    const float shift = next == -INFINITY ? 0.0f : next;
    const float keep = exp2f(top - shift), p = exp2f(s - shift);
    total = total * keep + p;
    for (int x = 0; x < 4; ++x) o[x] = o[x] * keep + p * v[x];
    top = next;
  }
  T* op = static_cast<T*>(a.o) + t * a.o_st[0] + h * a.o_st[1];
  const float inv = total == 0.0f ? 0.0f : 1.0f / total;
  if (on)
    for (int x = 0; x < 4; ++x) op[d + x] = from_f32<T>(o[x] * inv);
  if (a.lse != nullptr && lane == 0)
    a.lse[static_cast<long long>(t) * a.q_heads + h] = (top + log2f(total)) * 0.6931471805599453f;
}

}  // namespace akili
