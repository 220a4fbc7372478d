// Products with 4-bit weights and group scales at few rows.
//
//   y[r, m] = sum_G s[m, G] sum_{c in G} (u[m, c] - z[m, G]) x[r, c]        u, z in 0..15
//
// Packed layout (pack_w4_kernel): units of 32 rows x 128 columns, all units of a row tile after one another, so that a
// unit is one copy.  It begins with 2 KB of codes in four parts of 512 bytes: rows 0-15, columns
// 0-63 and 64-127, then rows 16-31.  In a part, lane l of a warp owns 16 bytes: rows l/4 and l/4 + 8, one word per
// four columns, word s holding the columns 32 (s/2) + 8 (l%4) + 4 (s%2) .. + 3.  The product is a sum over k, so its
// order may be chosen: word s goes to the s-th m16n8k16 step as if its columns were that step's slots 2t, 2t+1,
// 2t+8, 2t+9 (t = l%4).  A lane's share of x is then eight contiguous values per 32 columns, and every step
// lies inside one group, even of 32.  A word's nibbles are placed so that masks alone yield operand pairs:
//   bits 0, 16: row l/4, columns 0, 1    bits 4, 20: row l/4 + 8, columns 0, 1
//   bits 8, 24: row l/4, columns 2, 3    bits 12, 28: row l/4 + 8, columns 2, 3
// After the codes: f16 scales [group][16-row half][8][rows r, r + 8], so that a lane's two rows come in one load, then
// (optional) uint8 zero points in the same order.  Rows past n_out and columns past k are padded with u = 8, s = 0.
#pragma once
#include <cuda_bf16.h>
#include "device_common.cuh"
#include "gemm_tc.cuh"  // griddep_*

namespace qasr {

struct W4Layout {
  int tiles, units, unit_bytes;  // units per tile
  long long total;               // bytes
};
__host__ __device__ inline W4Layout w4_layout(int n_out, int k, int group, bool zero) {
  W4Layout l;
  l.tiles = (n_out + 31) / 32;
  l.units = (k + 127) / 128;
  l.unit_bytes = 2048 + (128 / group) * (zero ? 96 : 64);
  l.total = static_cast<long long>(l.tiles) * l.units * l.unit_bytes;
  return l;
}

// One warp per unit.
__global__ void pack_w4_kernel(const uint8_t* __restrict__ codes, const uint16_t* __restrict__ scale,
                               const uint8_t* __restrict__ zero, int n_out, int k, int group,
                               uint8_t* __restrict__ packed) {
  const W4Layout L = w4_layout(n_out, k, group, zero != nullptr);
  const int lane = threadIdx.x & 31, groups = k / group, gs = 128 / group;
  const long long all = static_cast<long long>(L.tiles) * L.units, step = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  for (long long unit = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); unit < all; unit += step) {
    const int tile = static_cast<int>(unit / L.units), u = static_cast<int>(unit % L.units);
    uint8_t* dst = packed + unit * L.unit_bytes;
    for (int part = 0; part < 4; ++part) {
      uint32_t out[4];
      for (int s = 0; s < 4; ++s) {
        const int c = u * 128 + (part & 1) * 64 + (s >> 1) * 32 + (lane & 3) * 8 + (s & 1) * 4;  // four columns: two bytes of a row
        out[s] = 0;
        for (int half = 0; half < 2; ++half) {
          const int m = tile * 32 + (part >> 1) * 16 + (lane >> 2) + 8 * half;
          uint32_t v = 0x8888;
          if (m < n_out && c < k) {
            const uint8_t* at = codes + (static_cast<long long>(m) * k + c) / 2;
            v = at[0] | (at[1] << 8);
          }
          out[s] |= ((v & 15) | ((v >> 4 & 15) << 16) | ((v >> 8 & 15) << 8) | ((v >> 12 & 15) << 24)) << (4 * half);
        }
      }
      reinterpret_cast<uint4*>(dst)[part * 32 + lane] = make_uint4(out[0], out[1], out[2], out[3]);
    }
    const int m = tile * 32 + (lane & 16) + ((lane & 15) >> 1) + 8 * (lane & 1);
    for (int h = 0; h < gs; ++h) {
      const int g = u * gs + h;
      const bool in = m < n_out && g < groups;
      const long long e = static_cast<long long>(m) * groups + g;
      reinterpret_cast<uint16_t*>(dst + 2048)[h * 32 + lane] = in ? scale[e] : 0;
      if (zero) (dst + 2048 + gs * 64)[h * 32 + lane] = in ? zero[e] & 15 : 8;
    }
  }
}

struct W4Args {
  const uint8_t* packed;
  int n_out, k;
  const void* x;
  int ldx, rows;
  void* out;
  int ldo, accumulate;
  int wk_log2;   // warps that share a tile's k
  int cluster;   // CTAs that share a tile's k
};

// Operand pairs of the matrix instruction.  An integer below 16 becomes a float by being put into the low mantissa bits
// of a power of two whose step is 1 (f16: 1024, or 16 * u on top of 1024; bf16: 128), which is subtracted again together
// with the zero point: u - z comes out exactly.
__device__ __forceinline__ uint32_t and_or(uint32_t v, uint32_t mask, uint32_t bits) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(v), "r"(mask), "r"(bits));
  return d;
}
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
      const uint32_t lo = and_or(v, 0x000f000fu, 0x64006400u), hi = and_or(v, 0x00f000f0u, 0x64006400u);
      const __half2 p = __hsub2(*reinterpret_cast<const __half2*>(&lo), l);
      const __half2 q = __hfma2(*reinterpret_cast<const __half2*>(&hi), sixteenth, h);
      a[2 * x] = *reinterpret_cast<const uint32_t*>(&p);
      a[2 * x + 1] = *reinterpret_cast<const uint32_t*>(&q);
    }
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // the first step of a sum
  static __device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
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
      const uint32_t v = and_or(w >> (4 * x), 0x000f000fu, 0x43004300u), z = x & 1 ? zh : zl;
      const __nv_bfloat162 p = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&z));
      a[x] = *reinterpret_cast<const uint32_t*>(&p);
    }
  }
  static __device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // the first step of a sum
  static __device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
  }
};

// Every warp streams its units of the packed weight, codes and scales, through a ring of its own in shared memory
// by bulk copies that it issues itself, so warps wait for data but not for one another, a unit costs next to no address
// arithmetic, and enough bytes are in flight whatever a tile's k is.  wk = 8 warps share a row tile's k (fewer when
// it has fewer units: the others then have the tiles behind it), and their sums meet in shared memory, in warp
// order.  x comes through L1, where it stays.  When there are few row tiles, the CTAs of a cluster share their k as well
// and the first joins their sums, in order.
// NT = ceil(rows / 8): the rows of x are the matrix instruction's eight columns, NT times over.  A weight is read and
// taken apart once whatever the rows are (9 instructions per 8 weights and lane).  Measured (B200, us in a graph): 60000 x 8192 at one
// row 50 (5.1 TB/s, 78% of the measured copy rate), 8 rows 55, 16 rows 76, 32 rows 148 (there x's way from L1 and the matrix
// instructions bound it), 33 rows 260 and 64 rows 280 (255 registers a thread and spills), 151936 x 2048 at one row 35 (4.6
// TB/s, 37.5 under the power cap: a warp has only two units between the joins of its tile), 2048 x 6144 at one row 4.4,
// 1024 x 2048 2.8 (latency).
// A wait for a copy that gives up is recorded in w4_status, and every output whose sum then lacks a part is NaN.
constexpr int W4_WARPS = 8;
constexpr int W4_THREADS = W4_WARPS * 32;
constexpr int W4_MAX_CLUSTER = 4;

template <bool ZERO, int GS, int NT>
struct W4Plan {
  static constexpr int unit_bytes = 2048 + GS * 64 + (ZERO ? GS * 32 : 0);
  static constexpr int per_sm = NT == 1 ? 3 : NT == 2 ? 2 : 1;  // resident CTAs, by their registers
  static constexpr int bufs = NT <= 2 ? 2 : 1;
  static constexpr int sums_bytes = bufs * W4_WARPS * 8 * NT * 33 * 4;
  static constexpr int bars_bytes = 512;
  static constexpr int room = (227 * 1024) / per_sm - 1024 - sums_bytes - bars_bytes;
  static constexpr int fit = room / (W4_WARPS * unit_bytes);
  static constexpr int slots = fit > 6 ? 6 : fit;  // of a warp's ring
  static constexpr int smem = bars_bytes + slots * W4_WARPS * unit_bytes + sums_bytes;
};

// {error, site} of the first wait that gave up since the words were last read (report_error).
static __device__ uint32_t w4_status[2];
constexpr uint32_t W4_WAIT_SITE = 0x40;

// How a unit comes into its slot (a test loses one here).
struct W4Copy {
  static __device__ __forceinline__ void unit(void* slot, const uint8_t* from, uint32_t bytes, uint64_t* full, int /*tile*/, int /*unit*/) {
    mbar_arrive_expect_tx(full, bytes);
    bulk_load(slot, from, bytes, full);
  }
};

template <bool BF16, bool ZERO, int GS, int NT, class COPY = W4Copy>
__global__ void __launch_bounds__(W4_THREADS, (W4Plan<ZERO, GS, NT>::per_sm)) gemv_w4_kernel(const __grid_constant__ W4Args a) {
  using TT = W4Type<BF16>;
  using T = typename TT::T;
  using P = W4Plan<ZERO, GS, NT>;
  constexpr int SLOTS = P::slots;
  extern __shared__ __align__(128) uint8_t w4_smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, t = lane & 3;
  uint64_t* full = reinterpret_cast<uint64_t*>(w4_smem) + warp * SLOTS;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(w4_smem + P::bars_bytes - 16);
  uint8_t* ring = w4_smem + P::bars_bytes + warp * SLOTS * P::unit_bytes;
  float* sums = reinterpret_cast<float*>(w4_smem + P::bars_bytes + W4_WARPS * SLOTS * P::unit_bytes);  // [bufs][warp][8 NT][33]
  const W4Layout L = w4_layout(a.n_out, a.k, 128 / GS, ZERO);
  const int wk_n = 1 << a.wk_log2, wk = warp & (wk_n - 1), wt = warp >> a.wk_log2;
  const int wt_n = W4_WARPS >> a.wk_log2;  // tiles of a group
  const int rank = blockIdx.x % a.cluster, group0 = blockIdx.x / a.cluster, group_step = gridDim.x / a.cluster;
  const int groups = (L.tiles + wt_n - 1) / wt_n;
  // this CTA's units of a tile (all of them unless a cluster shares the tile), and this warp's: wk, wk + wk_n, ...
  const int u0 = static_cast<int>(static_cast<long long>(L.units) * rank / a.cluster) + wk;
  const int u1 = static_cast<int>(static_cast<long long>(L.units) * (rank + 1) / a.cluster);
  if (lane == 0)
    for (int i = 0; i < SLOTS; ++i) mbar_init(&full[i], 1);
  if (tid == 0) *abort_flag = 0;
  fence_mbar_init();
  __syncthreads();
  griddep_wait();
  griddep_launch_dependents();

  // the copies' place in the walk over this warp's units, SLOTS ahead of the products'
  int cg = group0, cu = u0;
  const uint8_t* from = nullptr;
  const int stride = wk_n * P::unit_bytes;
  auto enter = [&] {  // the next group in which this warp has a unit
    while (cg < groups && (cg * wt_n + wt >= L.tiles || u0 >= u1)) cg += group_step;
    from = a.packed + (static_cast<long long>(cg * wt_n + wt) * L.units + u0) * P::unit_bytes;
    cu = u0;
  };
  auto copy_next = [&](int slot) {  // lane 0
    if (cg >= groups) return;
    COPY::unit(ring + slot * P::unit_bytes, from, P::unit_bytes, &full[slot], cg * wt_n + wt, cu);
    cu += wk_n;
    from += stride;
    if (cu >= u1) {
      cg += group_step;
      enter();
    }
  };
  if (lane == 0) {
    enter();
    for (int i = 0; i < SLOTS; ++i) copy_next(i);
  }
  __syncwarp();

  {
    // Columns of the product past the last row of x are never stored, so those lanes read a row that is there.
    const T* xr[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
      xr[n] = static_cast<const T*>(a.x) + static_cast<long long>(min(n * 8 + (lane >> 2), a.rows - 1)) * a.ldx + t * 8;
    float acc[2][NT][4];
    // a unit's products; the last one of a k that is no multiple of 128 lacks some of its 32-column quarters
    // At 32 rows and below a unit's share of x is asked for before its weights are waited for.  (Plain loads: the kernel may
    // have started while x was still being written, so it is not read-only for its whole life.)
    constexpr bool PRE = NT <= 4;
    uint4 px[PRE ? 4 : 1][NT];
    auto fetch_x = [&](int u) {
      const int left = a.k - u * 128;
      if (left >= 128) {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int m = 0; m < NT; ++m) px[q][m] = *reinterpret_cast<const uint4*>(xr[m] + u * 128 + q * 32);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
          for (int m = 0; m < NT; ++m)
            px[q][m] = q * 32 < left ? *reinterpret_cast<const uint4*>(xr[m] + u * 128 + q * 32) : make_uint4(0, 0, 0, 0);
      }
    };
    auto product = [&](auto whole, int u, const uint8_t* unit) {
      constexpr bool FULL = decltype(whole)::value;
      const uint4* codes = reinterpret_cast<const uint4*>(unit) + lane;
      const uint32_t* sc = reinterpret_cast<const uint32_t*>(unit + 2048) + (lane >> 2);
      const uint16_t* ze = reinterpret_cast<const uint16_t*>(unit + 2048 + GS * 64) + (lane >> 2);
      const int left = a.k - u * 128;
      uint4 w[2];
      float part[2][NT][4];
      uint32_t zl[2], zh[2];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        constexpr int per = 4 / GS;  // quarters under one scale
        uint4 xv[NT];
#pragma unroll
        for (int m = 0; m < NT; ++m) {
          if (PRE) xv[m] = px[q][m];
          else xv[m] = FULL || q * 32 < left ? *reinterpret_cast<const uint4*>(xr[m] + u * 128 + q * 32) : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (q % 2 == 0) w[i] = codes[i * 64 + q / 2 * 32];
          if (q % per == 0) {
            const uint32_t z = ZERO ? ze[(q / per) * 16 + i * 8] : 0x0808u;
            zl[i] = TT::zero_low(z & 0xff);
            zh[i] = TT::zero_high(z >> 8);
          }
          uint32_t av[4];
          TT::pairs(q % 2 ? w[i].z : w[i].x, zl[i], zh[i], av);
#pragma unroll
          for (int m = 0; m < NT; ++m) {
            if (q % per == 0) TT::mma_first(part[i][m], av, xv[m].x, xv[m].y);
            else TT::mma(part[i][m], av, xv[m].x, xv[m].y);
          }
          TT::pairs(q % 2 ? w[i].w : w[i].y, zl[i], zh[i], av);
#pragma unroll
          for (int m = 0; m < NT; ++m) TT::mma(part[i][m], av, xv[m].z, xv[m].w);
          if (q % per == per - 1) {
            const uint32_t sv = sc[(q / per) * 16 + i * 8];
            const __half2 s2 = *reinterpret_cast<const __half2*>(&sv);
            const float s0 = __low2float(s2), s1 = __high2float(s2);
#pragma unroll
            for (int m = 0; m < NT; ++m) {
              acc[i][m][0] = fmaf(s0, part[i][m][0], acc[i][m][0]);
              acc[i][m][1] = fmaf(s0, part[i][m][1], acc[i][m][1]);
              acc[i][m][2] = fmaf(s1, part[i][m][2], acc[i][m][2]);
              acc[i][m][3] = fmaf(s1, part[i][m][3], acc[i][m][3]);
            }
          }
        }
      }
    };
    uint32_t slot = 0, parity = 0;
    int buf = 0;
    bool lost = false;  // a wait gave up: the rest is walked through, barriers and all, without the weights
    for (int g = group0; g < groups; g += group_step) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < NT; ++m) acc[i][m][0] = acc[i][m][1] = acc[i][m][2] = acc[i][m][3] = 0.0f;
      if (g * wt_n + wt < L.tiles) {
        for (int u = u0; u < u1 && !lost; u += wk_n) {
          if constexpr (PRE) fetch_x(u);
          if (!__all_sync(0xffffffffu, mbar_try_wait(&full[slot], parity)) &&
              !mbar_wait_warp(&full[slot], parity, abort_flag, w4_status, W4_WAIT_SITE)) {
            lost = true;
            break;
          }
          if (PRE || u * 128 + 128 <= a.k) product(std::true_type{}, u, ring + slot * P::unit_bytes);
          else product(std::false_type{}, u, ring + slot * P::unit_bytes);
          __syncwarp();
          if (lane == 0) copy_next(static_cast<int>(slot));  // into the slot that was read just now
          if (++slot == SLOTS) {
            slot = 0;
            parity ^= 1;
          }
        }
      }
      // ---- the group's sums
      float* mysums = sums + (buf * W4_WARPS + warp) * (8 * NT * 33);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int m = 0; m < NT; ++m)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            mysums[(m * 8 + t * 2 + (c & 1)) * 33 + i * 16 + (lane >> 2) + (c >> 1) * 8] =
                lost ? __uint_as_float(0x7fffffffu) : acc[i][m][c];  // NaN: the sum lacks this warp's part, or some of it
      __syncthreads();
      for (int e = tid; e < a.rows * 32 * wt_n; e += W4_THREADS) {
        const int c = e % (32 * wt_n), r = e / (32 * wt_n);
        float* first = sums + (buf * W4_WARPS + ((c >> 5) << a.wk_log2)) * (8 * NT * 33) + r * 33 + (c & 31);
        float y = 0.0f;
        for (int v = 0; v < wk_n; ++v) y += first[v * (8 * NT * 33)];
        const long long m = static_cast<long long>(g) * wt_n * 32 + c;
        if (a.cluster > 1) {
          first[0] = y;  // only this thread reads it again, or another CTA after the cluster's barrier
        } else if (m < a.n_out) {
          T* o = static_cast<T*>(a.out) + static_cast<long long>(r) * a.ldo + m;
          if (a.accumulate) y += TT::to_f32(*o);
          *o = TT::from_f32(y);
        }
      }
      if (P::bufs == 2) buf ^= 1;
      else __syncthreads();
    }
  }
  if (a.cluster > 1) {
    // one group per cluster (the launch sees to it): its sums stand in buffer 0, warp 0's place
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0) {
      for (int e = tid; e < a.rows * 32; e += W4_THREADS) {
        const int c = e % 32, r = e / 32;
        const uint32_t at = smem_u32(sums + r * 33 + c);
        float y = 0.0f;
        for (int v = 0; v < a.cluster; ++v) {
          uint32_t far;
          float f;
          asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(at), "r"(v));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(f) : "r"(far) : "memory");
          y += f;
        }
        const long long m = static_cast<long long>(group0) * 32 + c;
        if (m < a.n_out) {
          T* o = static_cast<T*>(a.out) + static_cast<long long>(r) * a.ldo + m;
          if (a.accumulate) y += TT::to_f32(*o);
          *o = TT::from_f32(y);
        }
      }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (*abort_flag && tid == 0) {
    // copies in flight land before the shared memory is given back, bounded
    const uint64_t t0 = globaltimer();
    for (int i = 0; i < SLOTS * W4_WARPS; ++i)  // (warp 0's `full` is the first of all)
      for (uint32_t x = 0; x < 2; ++x)
        while (!mbar_try_wait(&full[i], x) && globaltimer() - t0 < 20000000ull) {
        }
  }
}

}  // namespace qasr
