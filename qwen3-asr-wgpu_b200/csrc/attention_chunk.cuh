// GQA attention of chunks of new tokens over the paged cache.
//
// Request i brings n_i query rows whose last stands at position kv_len[i] - 1; row j (position
// p = kv_len[i] - n_i + j) attends the positions 0..p of its slot:
//   s_t = scale * q . k_t,   o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m)
// with the running maximum m and sum of an online softmax, so K and V are passed over once.
#pragma once
#include <cuda_bf16.h>
#include "device_common.cuh"
#include "gemm_tc.cuh"  // griddep_*

namespace qasr {

constexpr int CHUNK_DIM = 128;
constexpr int CHUNK_PAGE = 64;

struct ChunkArgs {
  const void* q;
  int q_ld;
  void* out;
  int out_ld;
  int rows;
  const void* pool;
  int pool_pages;
  const int* page_table;
  int max_slots, max_pages, layers, nq, nkv, layer;
  const int* seq_slot;
  const int* cu_rows;
  const int* kv_len;
  int n_seqs;
  float scale_log2;  // scale * log2(e): the softmax runs in powers of two
};

template <bool BF16>
struct ChunkType;
template <>
struct ChunkType<false> {
  using T = __half;
  static __device__ __forceinline__ float2 to_f32(uint32_t v) { return __half22float2(*reinterpret_cast<__half2*>(&v)); }
  static __device__ __forceinline__ uint32_t from_f32(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};
template <>
struct ChunkType<true> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float2 to_f32(uint32_t v) {
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  }
  static __device__ __forceinline__ uint32_t from_f32(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
};

// Row `kv` (0 = K, 1 = V) of position t, or -1 where the table leads out of the pool.
__device__ __forceinline__ long long chunk_kv_row(const ChunkArgs& a, int slot, int t, int kv, int head) {
  const int page = a.page_table[static_cast<size_t>(slot) * a.max_pages + (t >> 6)];
  if (page < 0 || page >= a.pool_pages) return -1;
  return (((static_cast<long long>(page) * a.layers + a.layer) * 2 + kv) * a.nkv + head) * CHUNK_PAGE + (t & 63);
}

// One warp per (row, query head): lane l holds dims 4l .. 4l + 3.
template <bool BF16>
__global__ void __launch_bounds__(256) attention_chunk_rows_kernel(const __grid_constant__ ChunkArgs a) {
  using TT = ChunkType<BF16>;
  using T = typename TT::T;
  griddep_wait();
  griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const long long unit = static_cast<long long>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int r = static_cast<int>(unit / a.nq), h = static_cast<int>(unit % a.nq);
  if (r >= a.rows) return;
  int lo = 0, hi = a.n_seqs - 1;  // last request that starts at or before r
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.cu_rows[mid] <= r) lo = mid; else hi = mid - 1;
  }
  const int first = a.cu_rows[lo], end = min(a.cu_rows[lo + 1], a.rows);
  if (r < first || r >= end) return;
  const int slot = a.seq_slot[lo];
  int len = slot >= 0 && slot < a.max_slots ? a.kv_len[lo] : 0;
  len = static_cast<int>(min(static_cast<long long>(max(len, 0)), static_cast<long long>(a.max_pages) * 64));
  const int last = len - (end - r);
  const int head = h / (a.nq / a.nkv);
  const T* qp = static_cast<const T*>(a.q) + static_cast<size_t>(r) * a.q_ld + h * CHUNK_DIM + lane * 4;
  const uint2 qv = *reinterpret_cast<const uint2*>(qp);
  const float2 q01 = TT::to_f32(qv.x), q23 = TT::to_f32(qv.y);
  float m = -INFINITY, l = 0.0f, o[4] = {};
  for (int t = 0; t <= last; ++t) {
    const long long kr = chunk_kv_row(a, slot, t, 0, head), vr = chunk_kv_row(a, slot, t, 1, head);
    const int at = (((lane >> 1) ^ (t & 7)) << 3) + (lane & 1) * 4;
    uint2 kv = {}, vv = {};
    if (kr >= 0) {
      kv = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.pool) + kr * CHUNK_DIM + at);
      vv = *reinterpret_cast<const uint2*>(static_cast<const T*>(a.pool) + vr * CHUNK_DIM + at);
    }
    const float2 k01 = TT::to_f32(kv.x), k23 = TT::to_f32(kv.y);
    float s = q01.x * k01.x + q01.y * k01.y + q23.x * k23.x + q23.y * k23.y;
#pragma unroll
    for (int x = 16; x; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
    s *= a.scale_log2;
    const float m2 = fmaxf(m, s);
    const float base = m2 == -INFINITY ? 0.0f : m2;
    const float f = exp2f(m - base), p = exp2f(s - base);
    const float2 v01 = TT::to_f32(vv.x), v23 = TT::to_f32(vv.y);
    l = l * f + p;
    o[0] = o[0] * f + p * v01.x;
    o[1] = o[1] * f + p * v01.y;
    o[2] = o[2] * f + p * v23.x;
    o[3] = o[3] * f + p * v23.y;
    m = m2;
  }
  const float inv = last < 0 ? 0.0f : 1.0f / l;
  uint2 res;
  res.x = TT::from_f32(o[0] * inv, o[1] * inv);
  res.y = TT::from_f32(o[2] * inv, o[3] * inv);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + static_cast<size_t>(r) * a.out_ld + h * CHUNK_DIM + lane * 4) = res;
}

}  // namespace qasr
