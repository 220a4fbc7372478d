// Products with 4-bit weights and group scales at few rows.
//
//   y[r, m] = sum_G s[m, G] sum_{c in G} (u[m, c] - z[m, G]) x[r, c]        u, z in 0..15
//
// Packed layout (pack_w4_kernel): row tiles of 16 x k blocks of 64, 512 bytes each, tile-major, so a tile's k
// range is one contiguous stream.  Within a block, lane l of a warp owns 16 bytes: rows l/4 and l/4 + 8, one
// word per four columns, word s holding the columns 32 (s/2) + 8 (l%4) + 4 (s%2) .. + 3.  The product is a sum
// over k, so its order may be chosen: word s goes to the s-th m16n8k16 step as if its columns were that step's
// slots 2t, 2t+1, 2t+8, 2t+9 (t = l%4).  A lane's part of x is then eight contiguous values per 32 columns, and
// every step lies inside one group, even of 32.  A word's nibbles are placed so that masks alone yield
// operand pairs:
//   bits 0, 16: row l/4, columns 0, 1    bits 4, 20: row l/4 + 8, columns 0, 1
//   bits 8, 24: row l/4, columns 2, 3    bits 12, 28: row l/4 + 8, columns 2, 3
// After the codes: f16 scales [tile][group][8][rows r, r + 8], then (optional) uint8 zero points in the same
// order, so that a lane's two rows come in one load.  Rows past n_out and columns past k are padded with u = 8, s = 0.
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
    const int c = kb * 64 + (s >> 1) * 32 + (lane & 3) * 8 + (s & 1) * 4;  // four columns: two bytes of each row
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
    const int m = static_cast<int>(e / 16 / L.groups) * 16 + static_cast<int>((e & 15) >> 1) + 8 * static_cast<int>(e & 1);
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

// Operand pairs of the matrix instruction.  An integer below 16 becomes a float by being put into the low mantissa bits
// of a power of two whose step is 1 (f16: 1024, or 16 * u on top of 1024; bf16: 128), which is subtracted again together
// with the zero point: u - z comes out exactly.
template <bool BF16>
struct W4Type;
template <>
struct W4Type<false> {
  using T = __half;
  static __device__ __forceinline__ float to_f32(T v) { return __half2float(v); }
  static __device__ __forceinline__ T from_f32(float v) { return __float2half_rn(v); }
  // what pairs() subtracts for a row's zero point: 1024 + z (rows in the low nibbles), -(64 + z) (in the high ones)
  static __device__ __forceinline__ uint32_t zero_low(uint32_t z) { return (0x6400u | z) * 0x10001u; }
  static __device__ __forceinline__ uint32_t zero_high(uint32_t z) { return (0xd400u | (z << 4)) * 0x10001u; }
  static __device__ __forceinline__ void pairs(uint32_t w, uint32_t zl, uint32_t zh, uint32_t (&a)[4]) {
    const __half2 l = *reinterpret_cast<const __half2*>(&zl), h = *reinterpret_cast<const __half2*>(&zh);
    const __half2 sixteenth = __half2half2(__ushort_as_half(0x2c00));
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint32_t v = x ? w >> 8 : w;
      const uint32_t lo = (v & 0x000f000fu) | 0x64006400u, hi = (v & 0x00f000f0u) | 0x64006400u;
      const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&lo), l);
      const __half2 q = __hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, h);
      a[2 * x] = *reinterpret_cast<const uint32_t*>(&p);
      a[2 * x + 1] = *reinterpret_cast<const uint32_t*>(&q);
    }
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};
template <>
struct W4Type<true> {
  using T = __nv_bfloat16;
  static __device__ __forceinline__ float to_f32(T v) { return __bfloat162float(v); }
  static __device__ __forceinline__ T from_f32(float v) { return __float2bfloat16_rn(v); }
  static __device__ __forceinline__ uint32_t zero_low(uint32_t z) { return (0x4300u | z) * 0x10001u; }
  static __device__ __forceinline__ uint32_t zero_high(uint32_t z) { return (0x4300u | z) * 0x10001u; }
  static __device__ __forceinline__ void pairs(uint32_t w, uint32_t zl, uint32_t zh, uint32_t (&a)[4]) {
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      const uint32_t v = ((w >> (4 * x)) & 0x000f000fu) | 0x43004300u, z = x & 1 ? zh : zl;
      const __nv_bfloat162 p = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&z));
      a[x] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
};

constexpr int W4_WARPS = 8;
constexpr int W4_THREADS = W4_WARPS * 32;

// One CTA per MT row tiles; its warps take k blocks in turn, BATCH at a time so that their loads are in
// flight together, and the warps' sums meet in shared memory in warp order.  NT = ceil(rows / 8): the rows of x are the
// matrix instruction's eight columns, NT times over.  A weight is read once whatever the rows are.
template <bool BF16, bool ZERO, bool G32, int MT, int NT>
__global__ void __launch_bounds__(W4_THREADS) gemv_w4_kernel(const __grid_constant__ W4Args a) {
  using TT = W4Type<BF16>;
  using T = typename TT::T;
  constexpr int BATCH = MT * NT >= 8 ? 1 : MT * NT >= 2 ? 2 : 4;
  constexpr int GB = G32 ? 2 : 1;  // scales per block and row
  __shared__ float sums[W4_WARPS][8 * NT][16 * MT + 1];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 3;
  const int tile0 = blockIdx.x * MT;
  const W4Layout L = w4_layout(a.n_out, a.k, 1 << a.group_log2, ZERO);
  griddep_wait();
  griddep_launch_dependents();
  const uint8_t* zeros = a.packed + L.codes + L.scales;
  float acc[MT][NT][4] = {};
  for (int k0 = warp; k0 < L.kblocks; k0 += W4_WARPS * BATCH) {
    uint4 w[BATCH][MT];
    uint32_t sc[BATCH][MT][GB], z[BATCH][MT][GB];
    uint4 x[BATCH][NT][2];
#pragma unroll
    for (int b = 0; b < BATCH; ++b) {
      const int kb = k0 + b * W4_WARPS;
      const bool in = kb < L.kblocks;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const int tile = tile0 + i;
        const bool on = in && tile < L.tiles;
        const long long blk = static_cast<long long>(tile) * L.kblocks + kb;
        w[b][i] = on ? __ldcs(reinterpret_cast<const uint4*>(a.packed + blk * 512) + lane) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int h = 0; h < GB; ++h) {
          const long long e = ((static_cast<long long>(tile) * L.groups + ((kb * 64 + h * 32) >> a.group_log2)) * 8 + (lane >> 2));
          sc[b][i][h] = on ? __ldg(reinterpret_cast<const uint32_t*>(a.packed + L.codes) + e) : 0u;
          z[b][i][h] = ZERO && on ? __ldg(reinterpret_cast<const uint16_t*>(zeros) + e) : 0x0808u;
        }
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int r = n * 8 + (lane >> 2);
        const T* xr = static_cast<const T*>(a.x) + static_cast<long long>(r) * a.ldx + kb * 64 + t * 8;
        // k is a multiple of 32: a half of a block is there or is not
        x[b][n][0] = in && r < a.rows ? __ldg(reinterpret_cast<const uint4*>(xr)) : make_uint4(0, 0, 0, 0);
        x[b][n][1] = in && r < a.rows && kb * 64 + 32 < a.k ? __ldg(reinterpret_cast<const uint4*>(xr + 32)) : make_uint4(0, 0, 0, 0);
      }
    }
#pragma unroll
    for (int b = 0; b < BATCH; ++b)
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const uint32_t ws[4] = {w[b][i].x, w[b][i].y, w[b][i].z, w[b][i].w};
#pragma unroll
        for (int h = 0; h < GB; ++h) {
          float part[NT][4] = {};
          const uint32_t zl = TT::zero_low(z[b][i][h] & 0xff), zh = TT::zero_high(z[b][i][h] >> 8);
#pragma unroll
          for (int s = h * 2; s < (GB == 2 ? h * 2 + 2 : 4); ++s) {
            uint32_t av[4];
            TT::pairs(ws[s], zl, zh, av);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
              const uint4 xv = x[b][n][s >> 1];
              TT::mma(part[n], av, s & 1 ? xv.z : xv.x, s & 1 ? xv.w : xv.y);
            }
          }
          const __half2 s2 = *reinterpret_cast<const __half2*>(&sc[b][i][h]);
          const float s0 = __low2float(s2), s1 = __high2float(s2);
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[i][n][0] = fmaf(s0, part[n][0], acc[i][n][0]);
            acc[i][n][1] = fmaf(s0, part[n][1], acc[i][n][1]);
            acc[i][n][2] = fmaf(s1, part[n][2], acc[i][n][2]);
            acc[i][n][3] = fmaf(s1, part[n][3], acc[i][n][3]);
          }
        }
      }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int c = 0; c < 4; ++c)
        sums[warp][n * 8 + t * 2 + (c & 1)][i * 16 + (lane >> 2) + (c >> 1) * 8] = acc[i][n][c];
  __syncthreads();
  for (int e = tid; e < a.rows * 16 * MT; e += W4_THREADS) {
    const int r = e / (16 * MT), c = e % (16 * MT), m = tile0 * 16 + c;
    if (m >= a.n_out) continue;
    float y = 0.0f;
#pragma unroll
    for (int v = 0; v < W4_WARPS; ++v) y += sums[v][r][c];
    T* o = static_cast<T*>(a.out) + static_cast<long long>(r) * a.ldo + m;
    if (a.accumulate) y += TT::to_f32(*o);
    *o = TT::from_f32(y);
  }
}

}  // namespace qasr
