// Products with 4-bit weights and group scales at few rows.
//
//   y[r, m] = sum_G s[m, G] sum_{c in G} (u[m, c] - z[m, G]) x[r, c]        u, z in 0..15
//
// Packed layout (pack_w4_kernel): row tiles of 16 x k blocks of 64, 512 bytes each, tile-major,
// so a tile's k range is one contiguous stream.  Within a block, lane l of a warp owns 16 bytes: rows
// l/4 and l/4 + 8, columns 16 (l%4) .. + 15, one word per four columns.  The product is a sum over
// k, so its order may be chosen: word s is handed to the s-th m16n8k16 step as if its columns
// were that step's slots 2t, 2t+1, 2t+8, 2t+9 (t = l%4), which makes a lane's part of x 16
// contiguous values as well.  A word's nibbles are placed so that masks alone yield operand pairs:
//   bits 0, 16: row l/4, columns 0, 1    bits 4, 20: row l/4 + 8, columns 0, 1
//   bits 8, 24: row l/4, columns 2, 3    bits 12, 28: row l/4 + 8, columns 2, 3
// After the codes: f16 scales [tile][group][16 rows], then (optional) uint8 zero points in the same
// order.  Rows past n_out and columns past k are padded with u = 8, s = 0.
#pragma once
#include <cuda_bf16.h>
#include "device_common.cuh"
#include "gemm_tc.cuh"  // griddep_*

namespace qasr {

struct W4Layout {
  int tiles, kblocks, groups;  // groups of the padded k
  long long codes, scales, total;  // byte offsets / sizes
};
__host__ __device__ inline W4Layout w4_layout(int n_out, int k, int group, bool zero) {
  W4Layout l;
  l.tiles = (n_out + 15) / 16;
  l.kblocks = (k + 63) / 64;
  l.groups = (l.kblocks * 64 + group - 1) / group;
  l.codes = static_cast<long long>(l.tiles) * l.kblocks * 512;
  l.scales = static_cast<long long>(l.tiles) * l.groups * 32;
  l.total = l.codes + l.scales + (zero ? static_cast<long long>(l.tiles) * l.groups * 16 : 0);
  return l;
}

__global__ void pack_w4_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scale,
                               const uint8_t* __restrict__ zero, int n_out, int k, int group,
                               uint8_t* __restrict__ packed) {
  const W4Layout L = w4_layout(n_out, k, group, zero != nullptr);
  const int groups = k / group;
  const long long words = L.codes / 4, stride = static_cast<long long>(gridDim.x) * blockDim.x;
  const long long first = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  for (long long w = first; w < words; w += stride) {
    const int s = static_cast<int>(w & 3), lane = static_cast<int>((w >> 2) & 31);
    const long long blk = w >> 7;
    const int tile = static_cast<int>(blk / L.kblocks), kb = static_cast<int>(blk % L.kblocks);
    const int c = kb * 64 + (lane & 3) * 16 + s * 4;  // four columns: two bytes of each row
    uint32_t out = 0;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int m = tile * 16 + (lane >> 2) + 8 * half;
      uint32_t v = 0x8888;
      if (m < n_out && c < k) {
        const uint8_t* at = codes + (static_cast<long long>(m) * k + c) / 2;
        v = at[0] | (at[1] << 8);
      }
      out |= ((v & 15) | ((v >> 4 & 15) << 16) | ((v >> 8 & 15) << 8) | ((v >> 12 & 15) << 24)) << (4 * half);
    }
    reinterpret_cast<uint32_t*>(packed)[w] = out;
  }
  uint16_t* ps = reinterpret_cast<uint16_t*>(packed + L.codes);
  uint8_t* pz = packed + L.codes + L.scales;
  const long long entries = L.scales / 2;
  for (long long e = first; e < entries; e += stride) {
    const int m = static_cast<int>(e / 16 / L.groups) * 16 + static_cast<int>(e & 15);
    const int g = static_cast<int>((e >> 4) % L.groups);
    const bool in = m < n_out && g < groups;
    ps[e] = in ? scale[static_cast<long long>(m) * groups + g] : 0;
    if (zero) pz[e] = in ? zero[static_cast<long long>(m) * groups + g] & 15 : 8;
  }
}

struct W4Args {
  const uint8_t* packed;
  int n_out, k, group_log2;  // group = 1 << group_log2
  const void* x;
  int ldx, rows;
  void* out;
  int ldo, accumulate;
};

template <bool BF16>
struct W4Type;
template <>
struct W4Type<false> {
  using T = __half;
  static __device__ __forceinline__ float to_f32(T v) { return __half2float(v); }
  static __device__ __forceinline__ T from_f32(float v) { return __float2half_rn(v); }
};
template <>
struct W4Type<true> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float to_f32(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T from_f32(float v) { return __float2bfloat16_rn(v); }
};

constexpr int W4_THREADS = 256;

// One CTA per 16-row tile; its warps take k blocks in turn and the tile's sums meet in shared memory.
template <bool BF16, bool ZERO>
__global__ void __launch_bounds__(W4_THREADS) gemv_w4_kernel(const __grid_constant__ W4Args a) {
  using TT = W4Type<BF16>;
  using T = typename TT::T;
  const int tile = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  griddep_wait();
  griddep_launch_dependents();
  const int group = 1 << a.group_log2;
  const W4Layout L = w4_layout(a.n_out, a.k, group, ZERO);
  const T* x = static_cast<const T*>(a.x);
  for (int r = 0; r < a.rows; ++r) {
    __syncthreads();
    float acc[2] = {0.0f, 0.0f};
    for (int kb = warp; kb < L.kblocks; kb += W4_THREADS / 32) {
      const uint4 v = *reinterpret_cast<const uint4*>(
          a.packed + (static_cast<long long>(tile) * L.kblocks + kb) * 512 + lane * 16);
      const uint32_t w[4] = {v.x, v.y, v.z, v.w};
      const int c0 = kb * 64 + (lane & 3) * 16;
      const long long e = (static_cast<long long>(tile) * L.groups + (c0 >> a.group_log2)) * 16 + (lane >> 2);
      float part[2] = {0.0f, 0.0f};
      float z[2] = {8.0f, 8.0f};
      if (ZERO) {
        z[0] = a.packed[L.codes + L.scales + e];
        z[1] = a.packed[L.codes + L.scales + e + 8];
      }
      if (c0 < a.k) {
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float xv = TT::to_f32(x[static_cast<long long>(r) * a.ldx + c0 + s * 4 + j]);
            const int sh = (j & 1) * 16 + (j >> 1) * 8;
            part[0] += (static_cast<float>(w[s] >> sh & 15) - z[0]) * xv;
            part[1] += (static_cast<float>(w[s] >> (sh + 4) & 15) - z[1]) * xv;
          }
      }
      const __half* sc = reinterpret_cast<const __half*>(a.packed + L.codes) + e;
      acc[0] += __half2float(sc[0]) * part[0];
      acc[1] += __half2float(sc[8]) * part[1];
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 1);
      acc[h] += __shfl_xor_sync(0xffffffffu, acc[h], 2);
    }
    __shared__ float part[W4_THREADS / 32][16];
    if ((lane & 3) == 0) part[warp][lane >> 2] = acc[0], part[warp][(lane >> 2) + 8] = acc[1];
    __syncthreads();
    const int m = tile * 16 + tid;
    if (tid < 16 && m < a.n_out) {
      float y = 0.0f;
      for (int w = 0; w < W4_THREADS / 32; ++w) y += part[w][tid];
      T* o = static_cast<T*>(a.out) + static_cast<long long>(r) * a.ldo + m;
      if (a.accumulate) y += TT::to_f32(*o);
      *o = TT::from_f32(y);
    }
    __syncthreads();
  }
}

}  // namespace qasr
