// cache.cuh — bookkeeping of the paged key/value cache around a verified
// draft: the ancestor bits of drafted trees and the compaction of the
// accepted branch.
#pragma once
#include <cuda_runtime.h>

#include "rope.cuh"
#include "sm100.cuh"

namespace akili {

// Sequence that owns packed row t: the last b with cu[b] <= t (t < cu[batch]).
__device__ __forceinline__ int find_sequence(const int* cu, int batch, int t) {
  int lo = 0, hi = batch - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu[mid] <= t) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// One thread per node walks up to its root.  A parent is smaller than its
// child, so the walk ends; one that is not ends it and is recorded.  Bound by
// the dependent loads of the longest branch: 16 trees of 16 to 64 nodes 3.5 us,
// 16 chains of 64 nodes 8.3 us.
__global__ void __launch_bounds__(128) tree_mask_kernel(const int* parents, const int* cu_q, unsigned int* mask,
                                                        int batch, int total, int words) {
  griddep_wait();
  griddep_launch_dependents();
  const int t = blockIdx.x * 128 + threadIdx.x;
  if (t >= total) return;
  unsigned int* row = mask + static_cast<long long>(t) * words;
  for (int w = 0; w < words; ++w) row[w] = 0;
  if (t < cu_q[0] || t >= cu_q[batch]) return;
  const int base = cu_q[find_sequence(cu_q, batch, t)];
  if (base < 0) {
    record_bad_index();
    return;
  }
  int j = t - base;
  while (j >= 0) {
    if (j < 32 * words) row[j / 32] |= 1u << (j & 31);
    else record_bad_index();
    const int p = parents[base + j];
    if (p >= j || p < -1) {
      record_bad_index();
      break;
    }
    j = p;
  }
}

struct AcceptArgs {
  char *k, *v;
  const int *page_table, *context_lens, *accepted, *n_accepted;
  int* new_lens;
  int kv_heads, num_pages, page_size, max_pages, max_accepted;
  int vecs;                             // accesses per head row
  long long k_st[4], v_st[4];           // layer, page, token, head, in bytes
  long long table_stride, acc_stride;
};

constexpr int kAcceptThreads = 128;
constexpr int kAcceptRows = 128;  // moves whose offsets are held at a time

// One block per (layer, sequence, share of the row).  Entry i's destination
// ctx + i is never the source of a later entry (accepted[j] >= j > i), and
// entries are taken in ascending order by the thread that owns the column, so
// moving in place needs no copy of the branch: a source is always read before
// the entry whose destination it is, or in the same batch, whose loads all
// come before its stores.  Bound by its chain of latencies (lengths, indices,
// pages, values): 16 sequences, 87 entries, 32 layers of 8 heads of 128 take
// 5.9 us, 22 MB.
template <typename U>
__global__ void __launch_bounds__(kAcceptThreads) cache_accept_kernel(const AcceptArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int layer = blockIdx.z;
  const int b = blockIdx.y;
  const int ctx = a.context_lens[b];
  int n = a.n_accepted[b];
  const bool teller = blockIdx.x == 0 && layer == 0 && threadIdx.x == 0;
  if (ctx < 0 || n < 0 || n > a.max_accepted) {
    if (teller) record_bad_index();
    if (ctx < 0) n = 0;
    n = min(max(n, 0), a.max_accepted);
  }
  if (a.new_lens != nullptr && teller) a.new_lens[b] = ctx + n;
  // [row]: byte offsets (without head and column) of source and destination, or -1
  __shared__ long long k_src[kAcceptRows], k_dst[kAcceptRows], v_src[kAcceptRows], v_dst[kAcceptRows];
  const int* table = a.page_table + b * a.table_stride;
  const int* acc = a.accepted + b * a.acc_stride;
  const long long cap = static_cast<long long>(a.max_pages) * a.page_size;
  const int cols = a.kv_heads * a.vecs;
  for (int i0 = 0; i0 < n; i0 += kAcceptRows) {
    __syncthreads();
    const int m = min(kAcceptRows, n - i0);
    for (int r = threadIdx.x; r < m; r += kAcceptThreads) {
      const int i = i0 + r;
      const int x = acc[i];
      const long long s = static_cast<long long>(ctx) + x, d = static_cast<long long>(ctx) + i;
      k_src[r] = -1;
      bool ok = x >= i && (i == 0 || x > acc[i - 1]) && s < cap;
      if (ok) {
        // (below 2^32: the sum of two ints)
        const uint32_t us = static_cast<uint32_t>(s), ud = static_cast<uint32_t>(d), size = a.page_size;
        const int ps = table[us / size], pd = table[ud / size];
        ok = ps >= 0 && ps < a.num_pages && pd >= 0 && pd < a.num_pages;
        if (ok && s != d) {
          const long long os = us % size, od = ud % size;
          k_src[r] = ps * a.k_st[1] + os * a.k_st[2];
          k_dst[r] = pd * a.k_st[1] + od * a.k_st[2];
          v_src[r] = ps * a.v_st[1] + os * a.v_st[2];
          v_dst[r] = pd * a.v_st[1] + od * a.v_st[2];
        }
      }
      if (!ok && blockIdx.x == 0 && layer == 0) record_bad_index();
    }
    __syncthreads();
    for (int e = blockIdx.x * kAcceptThreads + threadIdx.x; e < 2 * cols; e += gridDim.x * kAcceptThreads) {
      const bool is_v = e >= cols;
      const int c = is_v ? e - cols : e;
      const int h = c / a.vecs, x = c - h * a.vecs;
      char* base = is_v ? a.v + layer * a.v_st[0] + h * a.v_st[3] : a.k + layer * a.k_st[0] + h * a.k_st[3];
      base += static_cast<long long>(x) * sizeof(U);
      const long long* src = is_v ? v_src : k_src;
      const long long* dst = is_v ? v_dst : k_dst;
      constexpr int kBatch = 8;
      for (int r = 0; r < m; r += kBatch) {
        U held[kBatch];
        bool live[kBatch];
#pragma unroll
        for (int q = 0; q < kBatch; ++q) {
          live[q] = r + q < m && k_src[r + q] >= 0;
          if (live[q]) held[q] = *reinterpret_cast<const U*>(base + src[r + q]);
        }
#pragma unroll
        for (int q = 0; q < kBatch; ++q)
          if (live[q]) *reinterpret_cast<U*>(base + dst[r + q]) = held[q];
      }
    }
  }
}

}  // namespace akili
