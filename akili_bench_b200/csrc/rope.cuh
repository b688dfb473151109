// rope.cuh — rotary positions of queries and keys, in place, out of place or
// with the rotated keys and the values written into the pages of a cache.
//
//   y1 = x1 cos(p f_i) - x2 sin(p f_i),   y2 = x2 cos(p f_i) + x1 sin(p f_i)
//
// for the pair i of the first rot_dim values of each head, p the token's
// position; (x1, x2) are the values i and i + rot_dim/2, or 2i and 2i + 1
// (interleaved).  The inverse rotation (sin negated) is the transpose, so it
// is the gradient.
//
// Nothing is reused but the token's table row, so the kernel is bound by HBM
// bandwidth: every value is read and written once.  One block per token (and
// per share of its heads when there are few tokens); a thread keeps the
// cosines and sines of its VEC pairs in registers and walks over the heads, so
// the table is read once per token and thread, from L2.
//
// Measured: 8192 tokens, 32 + 8 heads of 128, fp16: 30.2 us, 5.7 TB/s (an
// elementwise product of the same bytes: 27.5 us; the copy rate would be
// 26.3).  Blocks of 128 threads measured 32 us (24 against 22 for the append),
// of 256 threads 46, of one warp 31 (and 16 against 11 for 2049 tokens in fp32);
// two heads a thread, persistent blocks with the next position read ahead, and
// whole rows through shared memory by bulk copies 31 to 36 us.
// 7 tokens: 2.2 us.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/akili_serving.h"
#include "sm100.cuh"

namespace akili {

constexpr int kRopeThreads = 64;

static_assert(kStatusBadIndex == AKILI_STATUS_BAD_INDEX, "status code of a skipped index");

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// VEC values moved as one access (16 bytes, or one value).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) ValueVec {
  T v[VEC];
};

// Two values at a time.
__device__ __forceinline__ float2 to_f32x2(const float* x) { return make_float2(x[0], x[1]); }
__device__ __forceinline__ float2 to_f32x2(const __half* x) { return __half22float2(*reinterpret_cast<const __half2*>(x)); }
__device__ __forceinline__ float2 to_f32x2(const __nv_bfloat16* x) {
  return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(x));
}
__device__ __forceinline__ void from_f32x2(float* y, float a, float b) {
  y[0] = a;
  y[1] = b;
}
__device__ __forceinline__ void from_f32x2(__half* y, float a, float b) {
  *reinterpret_cast<__half2*>(y) = __floats2half2_rn(a, b);
}
__device__ __forceinline__ void from_f32x2(__nv_bfloat16* y, float a, float b) {
  *reinterpret_cast<__nv_bfloat162*>(y) = __floats2bfloat162_rn(a, b);
}

struct RopeArgs {
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;  // append: k_out, v_out are the pages
  void* k_copy;                 // append: optional, the rotated k by token
  const int* positions;
  const float* table;
  const long long* slots;  // append only
  int tokens, q_heads, k_heads, head_dim, rot_dim, max_positions;
  int num_pages, page_size;
  int interleaved;
  float sin_sign;
  long long q_st[2], k_st[2], v_st[2], qo_st[2];
  long long ko_st[3], vo_st[3];  // page, token, head (akili_rope: 0, token, head)
  long long kc_st[2];
};

// Threads of a block: `hl` head lanes of `ul` consecutive units each.  A unit
// is VEC pairs (2 VEC values) of the rotated part or 2 VEC values of the rest.
template <typename T, int VEC, bool kAppend>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a) {
  using V = ValueVec<T, VEC>;
  griddep_wait();
  griddep_launch_dependents();
  const int t = blockIdx.x;
  const int p = a.positions[t];
  if (p < 0 || p >= a.max_positions) {
    if (threadIdx.x == 0) record_bad_index();
    return;
  }
  long long slot = t;
  bool store_kv = true;
  if constexpr (kAppend) {
    slot = a.slots[t];
    store_kv = slot >= 0 && slot < static_cast<long long>(a.num_pages) * a.page_size;
    if (!store_kv && slot != -1 && threadIdx.x == 0) record_bad_index();
  }
  const int half = a.rot_dim / 2;
  const int turn_units = half / VEC;
  const int rest = a.head_dim - a.rot_dim;
  const int units = turn_units + (rest + 2 * VEC - 1) / (2 * VEC);
  const int ul = min(units, kRopeThreads);
  const int hl = kRopeThreads / ul;
  const int lane_u = threadIdx.x % ul;
  const int lane_h = threadIdx.x / ul;
  if (lane_h >= hl) return;
  const int heads = a.q_heads + a.k_heads + (kAppend ? a.k_heads : 0);
  const float* row = a.table + static_cast<long long>(p) * a.rot_dim;
  long long page = 0, in_page = t;
  if constexpr (kAppend) {
    if (store_kv) {
      page = slot / a.page_size;
      in_page = slot - page * a.page_size;
    }
  }
  for (int u = lane_u; u < units; u += ul) {
    const bool turn = u < turn_units;
    float c[VEC], s[VEC];
    if (turn) {
      if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
          *reinterpret_cast<float4*>(c + i) = *reinterpret_cast<const float4*>(row + u * VEC + i);
          *reinterpret_cast<float4*>(s + i) = *reinterpret_cast<const float4*>(row + half + u * VEC + i);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          c[i] = row[u * VEC + i];
          s[i] = row[half + u * VEC + i];
        }
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) s[i] *= a.sin_sign;
    }
    // offsets of the unit's two vectors within a head
    int o0, o1;
    if (turn) {
      o0 = a.interleaved ? 2 * u * VEC : u * VEC;
      o1 = a.interleaved ? o0 + VEC : half + u * VEC;
    } else {
      o0 = a.rot_dim + (u - turn_units) * 2 * VEC;
      o1 = o0 + VEC < a.head_dim ? o0 + VEC : o0;
    }
    for (int h = blockIdx.y * hl + lane_h; h < heads; h += gridDim.y * hl) {
      const T* src;
      T* dst;
      T* copy = nullptr;
      bool rotate = turn;
      if (h < a.q_heads) {
        src = static_cast<const T*>(a.q) + t * a.q_st[0] + h * a.q_st[1];
        dst = static_cast<T*>(a.q_out) + t * a.qo_st[0] + h * a.qo_st[1];
      } else {
        int hk = h - a.q_heads;
        if (!kAppend || hk < a.k_heads) {
          src = static_cast<const T*>(a.k) + t * a.k_st[0] + hk * a.k_st[1];
          dst = static_cast<T*>(a.k_out) + page * a.ko_st[0] + in_page * a.ko_st[1] + hk * a.ko_st[2];
          if (kAppend && a.k_copy != nullptr) copy = static_cast<T*>(a.k_copy) + t * a.kc_st[0] + hk * a.kc_st[1];
        } else {
          hk -= a.k_heads;
          src = static_cast<const T*>(a.v) + t * a.v_st[0] + hk * a.v_st[1];
          dst = static_cast<T*>(a.v_out) + page * a.vo_st[0] + in_page * a.vo_st[1] + hk * a.vo_st[2];
          rotate = false;
        }
      }
      V x0 = *reinterpret_cast<const V*>(src + o0);
      V x1 = *reinterpret_cast<const V*>(src + o1);
      if (rotate) {
        if constexpr (VEC == 1) {
          const float y1 = to_f32(x0.v[0]), y2 = to_f32(x1.v[0]);
          x0.v[0] = from_f32<T>(y1 * c[0] - y2 * s[0]);
          x1.v[0] = from_f32<T>(y2 * c[0] + y1 * s[0]);
        } else if (a.interleaved) {
          // x0 and x1 hold the pairs (0, 1), (2, 3), ... of 2 VEC values in a row
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) {
            const float2 y = to_f32x2(x0.v + 2 * i), z = to_f32x2(x1.v + 2 * i);
            from_f32x2(x0.v + 2 * i, y.x * c[i] - y.y * s[i], y.y * c[i] + y.x * s[i]);
            from_f32x2(x1.v + 2 * i, z.x * c[VEC / 2 + i] - z.y * s[VEC / 2 + i],
                       z.y * c[VEC / 2 + i] + z.x * s[VEC / 2 + i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < VEC; i += 2) {
            const float2 y = to_f32x2(x0.v + i), z = to_f32x2(x1.v + i);
            from_f32x2(x0.v + i, y.x * c[i] - z.x * s[i], y.y * c[i + 1] - z.y * s[i + 1]);
            from_f32x2(x1.v + i, z.x * c[i] + y.x * s[i], z.y * c[i + 1] + y.y * s[i + 1]);
          }
        }
      }
      if (h < a.q_heads || store_kv) {
        *reinterpret_cast<V*>(dst + o0) = x0;
        *reinterpret_cast<V*>(dst + o1) = x1;
      }
      if (copy != nullptr) {
        *reinterpret_cast<V*>(copy + o0) = x0;
        *reinterpret_cast<V*>(copy + o1) = x1;
      }
    }
  }
}

constexpr int kRopeMaxRot = 256;
struct RopeTableArgs {
  double freq[kRopeMaxRot / 2];
  double amplitude;
  float* table;
  int max_positions, rot_dim;
};

// cos | sin of p f_i in fp64: an fp32 product p f_i would be wrong by 4e-3 at
// p = 131072.  Built once per model; 64 pairs x 131072 positions take 66 us.
__global__ void __launch_bounds__(256) rope_table_kernel(const __grid_constant__ RopeTableArgs a) {
  griddep_wait();
  griddep_launch_dependents();
  const int half = a.rot_dim / 2;
  const long long n = static_cast<long long>(a.max_positions) * half;
  for (long long e = blockIdx.x * 256ll + threadIdx.x; e < n; e += gridDim.x * 256ll) {
    const long long p = e / half;
    const int i = static_cast<int>(e - p * half);
    double s, c;
    sincos(static_cast<double>(p) * a.freq[i], &s, &c);
    a.table[p * a.rot_dim + i] = static_cast<float>(a.amplitude * c);
    a.table[p * a.rot_dim + half + i] = static_cast<float>(a.amplitude * s);
  }
}

}  // namespace akili
