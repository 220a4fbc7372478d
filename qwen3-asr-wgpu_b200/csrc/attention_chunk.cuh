// GQA attention of chunks of new tokens over the paged cache.
//
// Request i brings n_i query rows whose last stands at position kv_len[i] - 1; row j (position
// p = kv_len[i] - n_i + j) attends the positions 0..p of its slot:
//   s_t = scale * q . k_t,   o = sum_t e^(s_t - m) v_t / sum_t e^(s_t - m)
// with the running maximum m and sum of an online softmax, so K and V are passed over once.
//
// The products are tcgen05 MMAs of 128 rows.  A kv head's nq / nkv = G query heads share its keys, so
// the rows of a tile are packed: row r is token r / G, head r % G of the group (T tokens a tile, T the
// largest multiple of 8 with T * G <= 128).  A block is two row tiles; per page of 64 keys
//   S = Q K^T        A: Q in shared memory, B: K in shared memory (positions x dims, K-major)
//   P = 2^(S - m)    one thread per row, straight from and back to tensor memory, where P takes S's place
//   O += P V         A: P in tensor memory, B: V in shared memory (MN-major), O in tensor memory
// A page's swizzle (chunk c of position p at c ^ (p % 8)) is, for each 64-dim half of its rows, the
// tensor core's own 128-byte swizzle, so pages are copied by TMA as they are and used as operands.
// Tensor memory holds two S tiles and O of each row tile: while a tile's softmax runs, the next tile's
// product is under way.  (Two S tiles of 128 keys would not fit beside O.  Of 64 keys Q K^T runs at 3/4 of the tensor
// cores' rate, its operands coming from shared memory, and still costs less than the wait for the only S tile of 128: 8192
// rows took 293 us that way.)
// P is rounded to the cache's type for the second product, as the tensor core wants it; the sum of P
// is taken before that rounding.  m is raised, and O rescaled, only when a row's maximum has grown by more than
// 2^8 (P then stays below 2^8, far inside f16), so the rescaling, a round trip over O, is rare.
//
// Roles: three threads, one a warp, steer: warp 0's issues Q K^T, warp 1's P V, each with its own ring of pages, so neither's
// waits hold up the other; warp 2's copies Q and the pages.  Warp 3 walks the schedule and hands the others one block
// after the other through shared memory, which keeps the walk out of their registers, and clears V rows for
// warp 1.  Warps 4-7 and 8-11 are two softmax groups, one per row tile.  A block of one row tile only (a
// decode step, a short chunk) gives its even key tiles to the first group and the odd ones to the second; both
// results stand in the same tensor memory lanes, and each group then joins them for half of the dims.  So both always have
// work.
//
// Work split: every (request, kv head, block) costs its key tiles plus CHUNK_BLOCK_COST; the costs of the whole call,
// laid end to end, are cut into one equal range per CTA.  A block that a cut goes through leaves f32
// partials (o, m, l) in the workspace and attention_chunk_combine_kernel joins them, in key order.
// Nothing about the lengths is known on the host: every CTA sums the costs itself.
//
// Measured (B200, us a call in a graph; first a burst of milliseconds, then under the power cap after seconds of nothing
// else, with the SM clock seen): 512 slots of 256-4096 positions 712 (6.3 TB/s, 96% of the measured copy rate) / 845 (1450 MHz), 8192
// rows from nothing 252 (1090 TFLOP/s, 66% of measured bf16) / 294 (1545 MHz; 935 TFLOP/s, 67% of the sustained rate).  Bursts:
// 32 slots of 100-1500 31, one token over 224 positions 10.8 (latency: launch 2, first block found 3, pages 1, three
// dependent products and softmaxes 3, join 2), 64 requests of 13 rows 58-76.  With 8192 rows the chain P -> P V -> Q K^T -> S of
// each group takes about 1850 cycles for 64 keys where the tensor cores need 1280 for both groups' products and the exponential unit
// 768: what is long is S to P, 1300 cycles of one thread's row in which no unit is busy half of the time.
//
// Masked keys: S is replaced, never added to, so whatever stands there cannot matter; their P is 0, and
// V rows behind the block's last position are zeroed in shared memory, so that 0 * NaN cannot arise.  What remains
// is a V that is not finite at a position which later rows of the same block may see and earlier ones may not, or an
// infinite one under a P that was rounded to 0: a row that is not finite, and not because of what it may see, is
// computed again without matrix instructions (chunk_row).
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
  int group, tile_tokens;  // nq / nkv; tokens of a row tile (chunk_tile_tokens)
  const int* seq_slot;
  const int* cu_rows;
  const int* kv_len;
  int n_seqs;
  float scale_log2;  // |scale| * log2(e): the softmax runs in powers of two
  int negate;        // the scale is negative
  uint8_t* ws;       // ChunkMeta[grid], then the partials
};

constexpr int CHUNK_THREADS = 384;
constexpr int CHUNK_KT = CHUNK_PAGE;              // keys per tile
constexpr int CHUNK_K_STAGES = 4, CHUNK_V_STAGES = 5;  // V is held until its P is there
constexpr int CHUNK_STAGE_BYTES = CHUNK_KT * CHUNK_DIM * 2;
constexpr int CHUNK_HALF_BYTES = CHUNK_KT * 128;  // the rows' first or second 64 dims
constexpr int CHUNK_Q_TILE = 128 * CHUNK_DIM * 2, CHUNK_Q_HALF = CHUNK_Q_TILE / 2;
constexpr int CHUNK_Q_BYTES = 2 * CHUNK_Q_TILE;
constexpr int CHUNK_OUT_BYTES = 32 * 64;           // per softmax warp: a quarter of its rows' output
constexpr int CHUNK_SMEM = CHUNK_Q_BYTES + (CHUNK_K_STAGES + CHUNK_V_STAGES) * CHUNK_STAGE_BYTES + 8 * CHUNK_OUT_BYTES + 3 * 1024;  // (m and l, ChunkBars)
constexpr int CHUNK_BLOCK_COST = 4;               // a block's Q copy, first and last steps, in key tiles (us at 2 / 4 / 6: 32 slots 34.1 / 31.3 / 31.3, 512 slots 700 / 683 / 684, 64 x 13 rows 70-82 / 58-63 / 62-69, a mixed step 71-75 / 68-71 / 72-74)
constexpr int CHUNK_SNAP = 2;                     // a cut this near to a block's edge moves onto it
constexpr float CHUNK_RESCALE = 8.0f;
constexpr uint32_t CHUNK_WAIT_STEPS = (10 * QASR_WAIT_NS) >> 20;  // chunk_row keeps the others waiting: 2.6 s for 32 rows of 2^20 positions
constexpr int CHUNK_PART_ROWS = 256;
constexpr int CHUNK_PART_LD = CHUNK_DIM + 4;                     // a row's o, m, l
constexpr int CHUNK_PART_FLOATS = CHUNK_PART_LD * CHUNK_PART_ROWS;

// What CTA c leaves behind: at most one block that it began and others finish (partials in slot 2c + 1), and one
// that it only went on with (slot 2c).
struct ChunkMeta {
  int state;  // 1: it began such a block; 2: a wait gave up
  int row0, ntok, head, pos0;
  int went_on;  // 1: it went on with the block of the CTAs before it; 2: and finished it
  int unused[2];
  uint32_t lost[4];  // chunk_lost(0..3) once a wait of any call has given up: no call clears it, only the check does
};
// Four words that a workspace of arbitrary content does not hold by chance.
__host__ __device__ constexpr uint32_t chunk_lost(int i) { return 0x6c6f7374u * (2 * i + 1) + 0x9e3779b9u; }
__host__ __device__ constexpr long long chunk_meta_bytes(int grid) { return (grid * 64ll + 255) / 256 * 256; }
__host__ __device__ constexpr long long chunk_ws_bytes(int grid) {
  return chunk_meta_bytes(grid) + 2ll * grid * CHUNK_PART_FLOATS * 4;
}
__device__ __forceinline__ float* chunk_part(const ChunkArgs& a, int grid, int slot) {
  return reinterpret_cast<float*>(a.ws + chunk_meta_bytes(grid)) + static_cast<size_t>(slot) * CHUNK_PART_FLOATS;
}
__host__ __device__ constexpr int chunk_tile_tokens(int group) { return (128 / group) & ~7; }

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

// ---------------------------------------------------------------- the schedule
struct ChunkSeq {
  int row0, n, len, slot;  // first row, rows, cached positions (its rows' included), slot (-1: none)
};
__device__ __forceinline__ ChunkSeq chunk_seq(const ChunkArgs& a, int i) {
  ChunkSeq s;
  s.row0 = min(max(a.cu_rows[i], 0), a.rows);
  s.n = min(max(a.cu_rows[i + 1], 0), a.rows) - s.row0;
  if (s.n < 0) s.n = 0;
  s.slot = a.seq_slot[i];
  if (s.slot < 0 || s.slot >= a.max_slots) s.slot = -1;
  s.len = s.slot < 0 ? 0 : min(max(a.kv_len[i], 0), a.max_pages * CHUNK_PAGE);
  return s;
}
// key tiles of block k (rows [k * bt, min(n, (k + 1) * bt)) of the request): at least one, so that a
// block which sees nothing is visited and written
__device__ __forceinline__ int chunk_blocks(int n, int bt) { return n <= bt ? (n > 0) : (n + bt - 1) / bt; }
__device__ __forceinline__ int chunk_tiles(const ChunkSeq& s, int k, int bt) {
  const int end = s.len - s.n + min(s.n, (k + 1) * bt);
  return max(1, (end + CHUNK_KT - 1) / CHUNK_KT);
}
__device__ __forceinline__ long long chunk_head_cost(const ChunkSeq& s, int bt) {
  long long c = 0;
  const int nb = chunk_blocks(s.n, bt);
  for (int k = 0; k < nb; ++k) c += chunk_tiles(s, k, bt) + CHUNK_BLOCK_COST;
  return c;
}
__device__ __forceinline__ long long chunk_bound(long long total, int c, int grid) {
  if (total < (1 << 22))  // (grid <= 512) a 64-bit division is a slow routine
    return static_cast<uint32_t>(total) * static_cast<uint32_t>(c) / static_cast<uint32_t>(grid);
  return total * c / grid;
}
// The first key tile behind a cut `x` cost units into a block.
__device__ __forceinline__ int chunk_cut(int x, int nt) {
  const int t = x - CHUNK_BLOCK_COST;
  if (t >= nt) return nt;
  if (t <= CHUNK_SNAP) return 0;
  return nt - t <= CHUNK_SNAP ? nt : t;
}

struct ChunkWalk {
  int i, g, k, nb, nt, t0, t1;
  int at, hi;  // the block's and the range's end, counted from the range's start
  ChunkSeq s;
};
// On to the next block; false past the last.
__device__ __forceinline__ bool chunk_step(const ChunkArgs& a, ChunkWalk& w, int bt) {
  w.at += w.nt + CHUNK_BLOCK_COST;
  if (++w.k < w.nb) return true;
  w.k = 0;
  if (++w.g < a.nkv) return true;
  w.g = 0;
  do {
    if (++w.i >= a.n_seqs) return false;
    w.s = chunk_seq(a, w.i);
  } while (w.s.n == 0);
  w.nb = chunk_blocks(w.s.n, bt);
  return true;
}
// Fit the walk's block to the CTA's range, passing over blocks without a tile in it; false past its end.
__device__ __forceinline__ bool chunk_fit(const ChunkArgs& a, ChunkWalk& w, int bt) {
  while (w.at < w.hi) {
    w.nt = chunk_tiles(w.s, w.k, bt);
    w.t0 = chunk_cut(-w.at, w.nt);
    w.t1 = chunk_cut(w.hi - w.at, w.nt);
    if (w.t1 > w.t0) return true;
    if (!chunk_step(a, w, bt)) return false;
  }
  return false;
}

// The first block of CTA `cta`'s range, found by one warp.  The requests are cut into 32 runs, one a lane; 32 requests of a
// run are read at a time, and a scan over the runs' costs, then one inside the run that holds the start, finds the request.
__device__ __forceinline__ bool chunk_begin(const ChunkArgs& a, ChunkWalk& w, int cta, int grid, int bt) {
  const int lane = threadIdx.x & 31, steps = (a.n_seqs + 1023) / 1024, runs = (a.n_seqs + steps * 32 - 1) / (steps * 32);
  auto cost_of = [&](ChunkSeq& s, int i) {
    if (i >= a.n_seqs) return 0ll;
    s = chunk_seq(a, i);
    return chunk_head_cost(s, bt) * a.nkv;
  };
  auto scan = [&](long long v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += u;
    }
    return v;
  };
  ChunkSeq s{};
  long long cost = 0, mine = 0;
  const bool one = runs == 1 && steps == 1;  // one read is all
  if (one) cost = cost_of(s, lane);
  for (int r = 0; !one && r < runs; r += 4) {  // four runs' reads at a time
    long long sum[4] = {};
    for (int x = 0; x < steps; ++x)
#pragma unroll
      for (int y = 0; y < 4; ++y) sum[y] += cost_of(s, ((r + y) * steps + x) * 32 + lane);
#pragma unroll
    for (int y = 0; y < 4; ++y) {
#pragma unroll
      for (int o = 16; o; o >>= 1) sum[y] += __shfl_xor_sync(0xffffffffu, sum[y], o);
      if (lane == r + y) mine = sum[y];
    }
  }
  long long total, at = 0;  // `at`: the cost before the run, then before the request
  int run = 0;
  long long incl = scan(one ? cost : mine);
  total = __shfl_sync(0xffffffffu, incl, 31);
  const long long lo = chunk_bound(total, cta, grid), hi = chunk_bound(total, cta + 1, grid);
  if (lo >= hi) return false;
  int src = __ffs(__ballot_sync(0xffffffffu, lo < incl)) - 1, i = 0;
  if (!one) {
    run = src;
    at = __shfl_sync(0xffffffffu, incl - mine, src);
    for (int x = 0;; ++x) {
      i = (run * steps + x) * 32;
      cost = cost_of(s, i + lane);
      incl = scan(cost) + at;
      const unsigned in = __ballot_sync(0xffffffffu, lo < incl);
      if (in) {
        src = __ffs(in) - 1;
        break;
      }
      at = __shfl_sync(0xffffffffu, incl, 31);
    }
  }
  w.hi = static_cast<int>(min(hi - lo, 0x7fffffffll));
  w.i = i + src;
  at = __shfl_sync(0xffffffffu, incl - cost, src) - lo;  // <= 0 from here on
  w.s.row0 = __shfl_sync(0xffffffffu, s.row0, src);
  w.s.n = __shfl_sync(0xffffffffu, s.n, src);
  w.s.len = __shfl_sync(0xffffffffu, s.len, src);
  w.s.slot = __shfl_sync(0xffffffffu, s.slot, src);
  const long long head = chunk_head_cost(w.s, bt);
  for (w.g = 0; at + head <= 0; ++w.g) at += head;
  w.nb = chunk_blocks(w.s.n, bt);
  for (w.k = 0;; ++w.k) {
    const int c = chunk_tiles(w.s, w.k, bt) + CHUNK_BLOCK_COST;
    if (at + c > 0) break;
    at += c;
  }
  w.at = static_cast<int>(at);
  return chunk_fit(a, w, bt);
}

// ---------------------------------------------------------------- pieces
__device__ __forceinline__ void tmem_ld_x32(uint32_t taddr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tma_load_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int32_t x, int32_t y,
                                            int32_t z, int32_t u) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(u)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive_n(uint64_t* bar, uint32_t n) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(n) : "memory");
}
__device__ __forceinline__ void fence_proxy_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// two f32 at a time
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// 2^x for two x <= CHUNK_RESCALE (right for any x < 127.5) on the FMA pipe: x = n + f with n the nearest integer, 2^f by the polynomial of degree 4 with the
// smallest largest relative error on [-1/2, 1/2] and value 1 at 0 (2.9e-6 in f32, found by weighted least squares; f16 rounds P
// to 4.9e-4), n added to the exponent.  At -127 and below, a masked score's -inf among them, the result is exactly 0.  What is
// not a number becomes the largest f32: P rounds it to infinity, and the sum shows it (2^127 and more).
static_assert(CHUNK_RESCALE < 15.0f, "P, up to 2^CHUNK_RESCALE, is finite in f16, and ex2_poly2 has no overflow to handle");
__device__ __forceinline__ void ex2_poly2(uint64_t x2, float& a, float& b) {
  float xa, xb;
  unpack2(x2, xa, xb);
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(xa) : "f"(-127.0f));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(xb) : "f"(-127.0f));
  x2 = pack2(xa, xb);
  const uint64_t magic = pack2(12582912.0f, 12582912.0f);  // 1.5 * 2^23: the sum's low bits are the integer
  const uint64_t t = add2(x2, magic);
  const uint64_t f = fma2(add2(t, pack2(-12582912.0f, -12582912.0f)), pack2(-1.0f, -1.0f), x2);
  uint64_t p = fma2(pack2(0.009582853f, 0.009582853f), f, pack2(0.055906426f, 0.055906426f));
  p = fma2(p, f, pack2(0.24024099f, 0.24024099f));
  p = fma2(p, f, pack2(0.69312418f, 0.69312418f));
  p = fma2(p, f, pack2(1.0f, 1.0f));
  float ta, tb, pa, pb;
  unpack2(t, ta, tb);
  unpack2(p, pa, pb);
  a = __uint_as_float(__float_as_uint(pa) + (__float_as_uint(ta) << 23));
  b = __uint_as_float(__float_as_uint(pb) + (__float_as_uint(tb) << 23));
}
// Shared-memory descriptor of V as the second operand, MN-major with 128-byte swizzle: 64-dim halves
// CHUNK_HALF_BYTES apart (LBO), groups of 8 positions 1024 bytes apart (SBO).
__device__ __forceinline__ uint64_t smem_desc_v(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3fffu) | (static_cast<uint64_t>(CHUNK_HALF_BYTES >> 4) << 16) |
         (static_cast<uint64_t>(1024u >> 4) << 32) | (static_cast<uint64_t>(1u) << 46) |
         (static_cast<uint64_t>(2u) << 61);
}
template <bool BF16>
__host__ __device__ constexpr uint32_t chunk_idesc(uint32_t n, bool b_mn_major) {
  return umma_idesc_f16_m128(n) | (BF16 ? (1u << 7) | (1u << 10) : 0u) | (b_mn_major ? 1u << 16 : 0u);
}

// One lane of a converged warp, the same one each time.  (Behind this the compiler issues MMAs from uniform registers; behind
// `lane == 0` it does not, and an MMA takes 85 cycles next to busy warps instead of 69.)
__device__ __forceinline__ bool elect_one() {
  uint32_t one;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
  return one != 0;
}

// A bounded wait of a whole warp: every lane sees the phase complete, or all of them give up together.
// (The clock is a slow read: it is looked at only once a good number of tries, each of which may itself be suspended
// for a while, has gone by.)
__device__ __forceinline__ bool chunk_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  uint32_t t0 = 0;  // the clock's bits 20 and up (steps of about a millisecond)
  for (uint32_t n = 1;; ++n) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if ((n & 63) == 0) {
      const uint32_t now = static_cast<uint32_t>(globaltimer() >> 20);
      if (n == 64) t0 = now;
      int quit = 0;
      if ((threadIdx.x & 31) == 0) {
        if (now - t0 > CHUNK_WAIT_STEPS) *abort_flag = 1;
        quit = *abort_flag;
      }
      if (__shfl_sync(0xffffffffu, quit, 0)) return false;
    }
  }
}

// The same for one thread.
__device__ __forceinline__ bool chunk_wait_one(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  uint32_t t0 = 0;
  for (uint32_t n = 1; !mbar_try_wait(bar, parity); ++n) {
    if ((n & 63) == 0) {
      const uint32_t now = static_cast<uint32_t>(globaltimer() >> 20);
      if (n == 64) t0 = now;
      if (now - t0 > CHUNK_WAIT_STEPS) *abort_flag = 1;
      if (*abort_flag) return false;
    }
  }
  return true;
}

// A row whose tensor core result is not finite, over the positions [t0, t1), by a warp whose lane l holds the dims 4l .. 4l + 3 (and
// leaves them alone unless `mine`).  Done as soon as what the row sees explains it: a NaN where a V is NaN, an infinity where one
// is infinite.  Else the row is computed without matrix instructions, into `part` (under the maximum r_m that stands
// there) or, where that is null, the output.  32 positions at a time (of one page), their loads under way together, since
// latency is what this takes.  For the scores a lane holds the dims of chunk l % 16 of 16 positions, whose sums over the lanes are
// exchanged so that each lane ends up with its own position's.
// (ms, 2048 rows from nothing, all finite 0.055: a V that is not finite at position 0, seen by all, 0.37; one at the end, seen by the
// last rows only and computed again for the others of the last block, 5.1.)
template <bool BF16>
__device__ __noinline__ void chunk_row(const ChunkArgs& a, int slot, int row, int qhead, int t0, int t1, bool mine, float* part,
                                       float r_m) {
  using TT = ChunkType<BF16>;
  using T = typename TT::T;
  const int lane = threadIdx.x & 31, chunk = lane & 15, upper = lane & 16, head = qhead / a.group;
  const float scale = a.negate ? -a.scale_log2 : a.scale_log2;
  const uint4 q = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + static_cast<size_t>(row) * a.q_ld + qhead * CHUNK_DIM + chunk * 8);
  auto dot = [](uint4 x, uint4 y) {
    const uint32_t u[4] = {x.x, x.y, x.z, x.w}, v[4] = {y.x, y.y, y.z, y.w};
    float d = 0.0f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = TT::to_f32(u[i]), g = TT::to_f32(v[i]);
      d = fmaf(f.x, g.x, fmaf(f.y, g.y, d));
    }
    return d;
  };
  unsigned want = 0, seen = 0;  // bits x, 4 + x: dim x is NaN, is infinite; a V there is
  auto kind = [](float f, int x) { return fabsf(f) < INFINITY ? 0u : f != f ? 1u << x : 16u << x; };
  float4* part_at = reinterpret_cast<float4*>(part) + lane;
  uint2* out_at = reinterpret_cast<uint2*>(static_cast<T*>(a.out) + static_cast<size_t>(row) * a.out_ld + qhead * CHUNK_DIM) + lane;
  if (mine) {
    float4 was;
    if (part) {
      was = *part_at;
    } else {
      const float2 w01 = TT::to_f32(out_at->x), w23 = TT::to_f32(out_at->y);
      was = make_float4(w01.x, w01.y, w23.x, w23.y);
    }
    want = kind(was.x, 0) | kind(was.y, 1) | kind(was.z, 2) | kind(was.w, 3);
  }
  float m = -INFINITY, l = 0.0f;  // l: of this lane's positions
  float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int t = t0; t < t1; t += 32) {
    const int n = min(32, t1 - t);
    const long long k_row = chunk_kv_row(a, slot, t, 0, head), v_row = k_row + static_cast<long long>(a.nkv) * CHUNK_PAGE;
    const T* k = static_cast<const T*>(a.pool) + k_row * CHUNK_DIM;
    const T* v = static_cast<const T*>(a.pool) + v_row * CHUNK_DIM + (lane & 1) * 4;
    uint4 kw[16];
    uint2 vw[16];
#pragma unroll
    for (int y = 0; y < 16; ++y)  // (a page out of the pool reads as zeros)
      kw[y] = k_row < 0 || y + upper >= n ? make_uint4(0, 0, 0, 0) : *reinterpret_cast<const uint4*>(k + (y + upper) * CHUNK_DIM + (chunk ^ (y & 7)) * 8);
    auto load_v = [&](int y0) {
#pragma unroll
      for (int y = 0; y < 16; ++y)
        vw[y] = k_row < 0 || y0 + y >= n ? make_uint2(0, 0) : *reinterpret_cast<const uint2*>(v + (y0 + y) * CHUNK_DIM + (((lane >> 1) ^ (y & 7)) << 3));
    };
    load_v(0);
    float s[16];
#pragma unroll
    for (int y = 0; y < 16; ++y) s[y] = dot(q, kw[y]);
#pragma unroll
    for (int w = 8; w; w >>= 1)
#pragma unroll
      for (int y = 0; y < w; ++y) {
        const float give = lane & w ? s[y] : s[y + w], keep = lane & w ? s[y + w] : s[y];
        s[y] = keep + __shfl_xor_sync(0xffffffffu, give, w);
      }
    const float d = lane < n ? s[0] * scale : -INFINITY;
    float top = d;
#pragma unroll
    for (int i = 16; i; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
    top = fmaxf(m, top);
    const float base = top == -INFINITY ? 0.0f : top, f = ex2(m - base), p = ex2(d - base);
    m = top;
    l = l * f + p;
#pragma unroll
    for (int x = 0; x < 4; ++x) o[x] *= f;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int y = 0; y < 16; ++y) {
        const float2 v01 = TT::to_f32(vw[y].x), v23 = TT::to_f32(vw[y].y);
        const float py = __shfl_sync(0xffffffffu, p, half * 16 + y), fv[4] = {v01.x, v01.y, v23.x, v23.y};
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          o[x] = fmaf(py, fv[x], o[x]);
          if (want) seen |= kind(fv[x], x);
        }
      }
      if (half == 0) load_v(16);
    }
    if (__all_sync(0xffffffffu, (want & ~seen) == 0)) return;
  }
#pragma unroll
  for (int i = 16; i; i >>= 1) l += __shfl_xor_sync(0xffffffffu, l, i);
  if (!mine) return;
  // (a score that is not a number makes l NaN, and m with it for the join)
  const float f = part ? ex2((l != l ? l : m) - r_m) : 1.0f / l;
  if (part) *part_at = make_float4(o[0] * f, o[1] * f, o[2] * f, o[3] * f);
  else *out_at = make_uint2(TT::from_f32(o[0] * f, o[1] * f), TT::from_f32(o[2] * f, o[3] * f));
}

// One block's part in a CTA's range, as the walk hands it on.
struct ChunkBlock {
  int more;            // 0: the range is over
  int row0, ntok;      // its rows of the call
  int pos0;            // the position of the first of them
  int head, slot;
  int t0, nt, tiles;   // key tiles [t0, t0 + nt) of the block's `tiles`
  int nt0;             // of two row tiles: how many of the nt the first one sees
  int pages[16];       // the first pages of the range
};
constexpr int CHUNK_BLOCKS = 3;

struct ChunkBars {
  uint64_t q_full[2], q_free[2];               // of a row tile's place
  uint64_t kv_full[CHUNK_K_STAGES + CHUNK_V_STAGES], kv_free[CHUNK_K_STAGES + CHUNK_V_STAGES];  // of K, then of V
  uint64_t s_full[2][2], p_full[2][2], pv_done[2][2], o_done[2], o_free[2], ml_full[2];
  uint64_t clear_ask, clear_done;              // rows of a V stage to be zeroed
  uint8_t* clear_at;
  int clear_from;
  uint64_t block_full[CHUNK_BLOCKS], block_free[CHUNK_BLOCKS];
  ChunkBlock block[CHUNK_BLOCKS];
  uint32_t tmem;
  int abort_flag;
};
static_assert(sizeof(ChunkBars) <= 1024, "ChunkBars sits in the last KB of the shared memory");

template <bool BF16>
__global__ void __launch_bounds__(CHUNK_THREADS, 1)
    attention_chunk_kernel(const __grid_constant__ CUtensorMap q_big, const __grid_constant__ CUtensorMap q_small,
                           const __grid_constant__ CUtensorMap kv_map, const __grid_constant__ ChunkArgs a) {
  using TT = ChunkType<BF16>;
  using T = typename TT::T;
  extern __shared__ __align__(1024) uint8_t chunk_dsmem[];
  uint8_t* smem = chunk_dsmem;  // (there is no other shared memory: it begins on a 1 KB boundary)
  uint8_t* sm_q = smem;                                    // two row tiles, each [2 halves][128 rows][128 B]
  uint8_t* sm_kv = smem + CHUNK_Q_BYTES;                   // stages of K, then of V: [2 halves][64 positions][128 B]
  uint8_t* sm_out = sm_kv + (CHUNK_K_STAGES + CHUNK_V_STAGES) * CHUNK_STAGE_BYTES;  // per softmax warp [32 rows][64 B], chunks swizzled
  float* sm_ml = reinterpret_cast<float*>(sm_out + 8 * CHUNK_OUT_BYTES);  // [2 groups][m, l][128]
  ChunkBars& B = *reinterpret_cast<ChunkBars*>(reinterpret_cast<uint8_t*>(sm_ml) + 2048);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int grid = gridDim.x, cta = blockIdx.x;
  const int group = a.group, T_tok = a.tile_tokens, bt = 2 * T_tok;

  if (tid == 0) {
    mbar_init(&B.clear_ask, 1);
    mbar_init(&B.clear_done, 1);
    for (int i = 0; i < CHUNK_K_STAGES + CHUNK_V_STAGES; ++i) {
      mbar_init(&B.kv_full[i], 1);
      mbar_init(&B.kv_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B.s_full[i][0], 1);
      mbar_init(&B.s_full[i][1], 1);
      mbar_init(&B.o_done[i], 1);
      mbar_init(&B.q_full[i], 1);
      mbar_init(&B.q_free[i], 1);
      mbar_init(&B.p_full[i][0], 4);
      mbar_init(&B.p_full[i][1], 4);
      mbar_init(&B.pv_done[i][0], 1);
      mbar_init(&B.pv_done[i][1], 1);
      mbar_init(&B.o_free[i], 8);
      mbar_init(&B.ml_full[i], 4);
    }
    for (int i = 0; i < CHUNK_BLOCKS; ++i) {
      mbar_init(&B.block_full[i], 1);
      mbar_init(&B.block_free[i], 11);
    }
    B.abort_flag = 0;
    fence_mbar_init();
  }
  if (warp == 0) {
    tmem_alloc(&B.tmem, 512);
    tmem_relinquish();
  }
  if (warp == 2 && lane == 0) {
    tma_prefetch_desc(&q_big);
    tma_prefetch_desc(&q_small);
    tma_prefetch_desc(&kv_map);
  }
  griddep_wait();
  griddep_launch_dependents();

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = B.tmem;
  volatile int* abort_flag = &B.abort_flag;
  // block n of the range: 1 there, 0 the range is over, -1 a wait gave up
  auto take = [&](uint32_t n) {
    if (!chunk_wait(&B.block_full[n % CHUNK_BLOCKS], (n / CHUNK_BLOCKS) & 1, abort_flag)) return -1;
    return B.block[n % CHUNK_BLOCKS].more;
  };
  auto give_back = [&](uint32_t n) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&B.block_free[n % CHUNK_BLOCKS]);
  };
  // the same for the threads that steer
  auto wait_one = [&](uint64_t* bar, uint32_t parity) { return chunk_wait_one(bar, parity, abort_flag); };
  auto take_one = [&](uint32_t n) {
    if (!wait_one(&B.block_full[n % CHUNK_BLOCKS], (n / CHUNK_BLOCKS) & 1)) return -1;
    return B.block[n % CHUNK_BLOCKS].more;
  };
  ChunkMeta* meta = reinterpret_cast<ChunkMeta*>(a.ws + static_cast<size_t>(cta) * 64);
  if (tid == 128) meta->state = meta->went_on = 0;  // (the thread that may set them)

  if (warp >= 4) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");  // 256 x 208 + 128 x 88 = the launch's 384 x 168
    // ================================================================ softmax and output
    const int grp = (warp >> 2) - 1, row = (warp & 3) * 32 + lane;
    const int row_tok = row / group, row_head = row % group;
    const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + grp * 128 + lanes, t_o = tmem + 256 + grp * 128 + lanes;
    uint32_t n_tile = 0, n_out = 0, n_merge = 0;  // this group's tiles and blocks, and merges, so far
    for (uint32_t n_unit = 0; take(n_unit) == 1; give_back(n_unit), ++n_unit) {
      const ChunkBlock& d = B.block[n_unit % CHUNK_BLOCKS];
      const int nt = d.nt;
      const bool pair = d.ntok > T_tok;
      const bool valid = row_tok < T_tok && (pair ? grp * T_tok : 0) + row_tok < d.ntok;
      const bool live = __any_sync(0xffffffffu, valid);
      // the last key that the row sees, counted from the range's first
      const int limit = valid ? d.pos0 + (pair ? grp * T_tok : 0) + row_tok - d.t0 * CHUNK_KT : -1;
      const int step = pair ? 1 : 2, first = pair ? 0 : grp, count = pair && grp == 0 ? d.nt0 : nt;
      float m = -INFINITY, l = 0.0f;
      for (int j = first; j < count; j += step, ++n_tile) {
        const uint32_t t_buf = t_s + (n_tile & 1) * CHUNK_KT;
        if (!chunk_wait(&B.s_full[grp][n_tile & 1], (n_tile >> 1) & 1, abort_flag)) goto softmax_out;
        tc_fence_after();
        if (live) {
          float s[CHUNK_KT];
          tmem_ld_x32(t_buf, s);
          tmem_ld_x32(t_buf + 32, s + 32);
          tmem_wait_ld();
          if (a.negate) {
#pragma unroll
            for (int c = 0; c < CHUNK_KT; ++c) s[c] = -s[c];
          }
          const int last = limit - j * CHUNK_KT;  // in this tile
          if (__any_sync(0xffffffffu, last < CHUNK_KT - 1)) {
#pragma unroll
            for (int c = 0; c < CHUNK_KT; ++c) s[c] = c <= last ? s[c] : -INFINITY;
          }
          float mx[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) mx[c] = max3(s[c], s[c + 4], s[c + 8]);
#pragma unroll
          for (int c = 12; c < 60; c += 8)
#pragma unroll
            for (int x = 0; x < 4; ++x) mx[x] = max3(mx[x], s[c + x], s[c + x + 4]);
          const float top =
              fmaxf(max3(mx[0], mx[1], mx[2]), max3(mx[3], fmaxf(s[60], s[61]), fmaxf(s[62], s[63]))) * a.scale_log2;
          const bool raise = top > m + CHUNK_RESCALE;
          if (j == first) {
            m = top;
          } else if (__any_sync(0xffffffffu, raise)) {
            // O holds the sums under the old maximum: bring it under the new one
            if (!chunk_wait(&B.pv_done[grp][(n_tile - 1) & 1], ((n_tile - 1) >> 1) & 1, abort_flag)) goto softmax_out;
            tc_fence_after();
            const float f = raise ? ex2(m - top) : 1.0f;
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              uint32_t o[32];
              tmem_ld_x32(t_o + c * 32, reinterpret_cast<float*>(o));
              tmem_wait_ld();
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f);
              tmem_st_x32(t_o + c * 32, o);
            }
            tmem_wait_st();
            l *= f;
            if (raise) m = top;
          }
          const float base = m == -INFINITY ? 0.0f : m;
          const uint64_t scale2 = pack2(a.scale_log2, a.scale_log2), base2 = pack2(-base, -base);
          uint64_t sum[2] = {0, 0};
          uint32_t p[32];
#pragma unroll
          for (int c = 0; c < 32; ++c) {
            // every fourth pair on the FMA pipe, so that the exponential unit is not what a tile waits for (8192 rows: none
            // 261 us, a fourth 247, a third 250 at the time; 252 now)
            const uint64_t e = fma2(pack2(s[2 * c], s[2 * c + 1]), scale2, base2);
            float p0, p1;
            if (c % 4 == 3) {
              ex2_poly2(e, p0, p1);
            } else {
              unpack2(e, p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
            }
            sum[c & 1] = add2(sum[c & 1], pack2(p0, p1));
            p[c] = TT::from_f32(p0, p1);
          }
          tmem_st_x32(t_buf, p);
          float s0, s1;
          unpack2(add2(sum[0], sum[1]), s0, s1);
          l += s0 + s1;
          tmem_wait_st();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.p_full[grp][n_tile & 1]);
      }
      // A score that is not a number must show in every join.  ex2_poly2 makes 2^128 of it, which no sum of real
      // probabilities reaches (each is at most 2^CHUNK_RESCALE), and m may be -inf beside it: a maximum passes over it.
      if (!(l < 0x1p127f)) m = l = __uint_as_float(0x7fffffffu);
      // ---- the block's end
      const bool had = first < count;  // this group had tiles
      if (had) {
        if (!chunk_wait(&B.o_done[grp], n_out & 1, abort_flag)) goto softmax_out;
        ++n_out;
        tc_fence_after();
      }
      // two row tiles: each group has its own; one: both groups' results are joined, each group taking 64 dims
      const bool merge = !pair && nt > 1;
      if (grp == 1 && !pair && !merge) continue;
      uint32_t t_a = t_o;
      float f_a = 1.0f, f_b = 0.0f;
      // a range in which the row saw nothing (m = -inf) is left out of every sum: its O may be anything
      bool has_a = m != -INFINITY, has_b = false;
      if (merge) {
        sm_ml[grp * 256 + row] = m;
        sm_ml[grp * 256 + 128 + row] = l;
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.ml_full[grp]);
        if (!chunk_wait(&B.ml_full[grp ^ 1], n_merge & 1, abort_flag)) goto softmax_out;
        ++n_merge;
        tc_fence_after();
        const float m_a = sm_ml[row], l_a = sm_ml[128 + row], m_b = sm_ml[256 + row], l_b = sm_ml[384 + row];
        const float top = fmaxf(m_a, m_b);
        has_a = m_a != -INFINITY;
        has_b = m_b != -INFINITY;
        f_a = has_a ? ex2(m_a - top) : 0.0f;
        f_b = has_b ? ex2(m_b - top) : 0.0f;
        l = (has_a ? l_a * f_a : 0.0f) + (has_b ? l_b * f_b : 0.0f);
        m = l != l ? l : top;
        t_a = tmem + 256 + lanes;
      }
      const int c_begin = merge ? 2 * grp : 0, c_end = merge ? c_begin + 2 : 4;  // in 32 dims
      const bool whole = nt == d.tiles;
      const int tok = (pair ? grp * T_tok : 0) + row_tok, pos = d.pos0 + tok;
      const bool seen = pos >= 0;
      const int out_row = d.row0 + tok, qhead = d.head * group + row_head;
      const int prow = (pair ? grp * 128 : 0) + row;
      float* part = chunk_part(a, grid, d.t0 == 0 ? 2 * cta + 1 : 2 * cta);
      float bad = 0.0f;
      if (live) {
        const float inv = whole ? 1.0f / l : 1.0f;
        const float g_a = seen ? f_a * inv : 0.0f, g_b = seen ? f_b * inv : 0.0f;
        const uint64_t ga2 = pack2(g_a, g_a), gb2 = pack2(g_b, g_b);
        const unsigned rows_valid = __ballot_sync(0xffffffffu, valid);
        // In nearly every block all rows saw keys in what is joined; where one did not, O may hold anything there.
        const bool plain = !__any_sync(0xffffffffu, valid && !(seen && has_a && (has_b || !merge)));
        uint8_t* stage = sm_out + (warp - 4) * CHUNK_OUT_BYTES;
        uint64_t bad2 = 0;
        // dims 32c .. 32c + 31 of this thread's row
        auto fetch = [&](int c, float (&o)[32]) {
          tmem_ld_x32(t_a + c * 32, o);
          if (merge) {
            float o1[32];
            tmem_ld_x32(t_a + 128 + c * 32, o1);
            tmem_wait_ld();
            if (!plain) {
#pragma unroll
              for (int x = 0; x < 32; ++x) {
                o[x] = has_a ? o[x] : 0.0f;
                o1[x] = has_b ? o1[x] : 0.0f;
              }
            }
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const uint64_t v = fma2(pack2(o1[x], o1[x + 1]), gb2, mul2(pack2(o[x], o[x + 1]), ga2));
              bad2 = fma2(v, 0, bad2);  // NaN once a value is not finite
              unpack2(v, o[x], o[x + 1]);
            }
          } else {
            tmem_wait_ld();
            if (!plain) {
#pragma unroll
              for (int x = 0; x < 32; ++x) o[x] = has_a ? o[x] : 0.0f;
            }
#pragma unroll
            for (int x = 0; x < 32; x += 2) {
              const uint64_t v = mul2(pack2(o[x], o[x + 1]), ga2);
              bad2 = fma2(v, 0, bad2);
              unpack2(v, o[x], o[x + 1]);
            }
          }
          if (!plain) {
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = seen ? o[x] : 0.0f;  // zeros, whatever stands there
          }
        };
        auto pack8 = [&](const float* o) {
          uint4 v;
          v.x = TT::from_f32(o[0], o[1]);
          v.y = TT::from_f32(o[2], o[3]);
          v.z = TT::from_f32(o[4], o[5]);
          v.w = TT::from_f32(o[6], o[7]);
          return v;
        };
        float* my_part = part + prow * CHUNK_PART_LD;
        if (__popc(rows_valid) <= 4) {  // as in a decode step: straight out of the rows' threads (us, through shared memory / straight: 32 slots of two rows 32.2 / 31.3, one token 11.1 / 10.8; of eight rows 21-23 / 22-24)
          T* to = static_cast<T*>(a.out) + static_cast<size_t>(out_row) * a.out_ld + qhead * CHUNK_DIM;
#pragma unroll 1
          for (int c = c_begin; c < c_end; ++c) {
            float o[32];
            fetch(c, o);
            if (!valid) continue;
#pragma unroll
            for (int x = 0; x < 32; x += 8) {
              if (whole) {
                *reinterpret_cast<uint4*>(to + c * 32 + x) = pack8(o + x);
              } else {
                *reinterpret_cast<float4*>(my_part + c * 32 + x) = make_float4(o[x], o[x + 1], o[x + 2], o[x + 3]);
                *reinterpret_cast<float4*>(my_part + c * 32 + x + 4) = make_float4(o[x + 4], o[x + 5], o[x + 6], o[x + 7]);
              }
            }
          }
        } else {
          // Through shared memory, 64 bytes a row, so that a store covers whole sectors of 8 rows: 32 dims in the
          // output's type, or the partial's in two halves.
          uint4* put = reinterpret_cast<uint4*>(stage + lane * 64);
          const int put_x = lane >> 1 & 3;
          // lane's rows 8 y + lane / 4, its chunk of each
          auto send = [&](auto to) {
            __syncwarp();
            uint4 v[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int r = y * 8 + (lane >> 2);
              v[y] = *reinterpret_cast<const uint4*>(stage + r * 64 + (((lane & 3) ^ (r >> 1 & 3)) * 16));
            }
#pragma unroll
            for (int y = 0; y < 4; ++y)
              if (rows_valid >> (y * 8 + (lane >> 2)) & 1) to(y, v[y]);
            __syncwarp();
          };
          if (whole) {
            T* to[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const int r = y * 8 + (lane >> 2);
              to[y] = static_cast<T*>(a.out) + static_cast<size_t>(__shfl_sync(0xffffffffu, out_row, r)) * a.out_ld +
                      __shfl_sync(0xffffffffu, qhead, r) * CHUNK_DIM + (lane & 3) * 8;
            }
#pragma unroll 1
            for (int c = c_begin; c < c_end; ++c) {
              float o[32];
              fetch(c, o);
#pragma unroll
              for (int x = 0; x < 4; ++x) put[x ^ put_x] = pack8(o + 8 * x);
              send([&](int y, uint4 v) { *reinterpret_cast<uint4*>(to[y] + c * 32) = v; });
            }
          } else {
            float* to = my_part - lane * CHUNK_PART_LD + (lane >> 2) * CHUNK_PART_LD + (lane & 3) * 4;
#pragma unroll 1
            for (int c = c_begin; c < c_end; ++c) {
              float o[32];
              fetch(c, o);
#pragma unroll
              for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                  const float* f = o + h * 16 + 4 * x;
                  put[x ^ put_x] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
                }
                send([&](int y, uint4 v) { *reinterpret_cast<uint4*>(to + y * 8 * CHUNK_PART_LD + c * 32 + h * 16) = v; });
              }
            }
          }
        }
        float b0, b1;
        unpack2(bad2, b0, b1);
        bad = seen ? b0 + b1 : 0.0f;
        if (valid && !whole && c_begin == 0) {
          my_part[CHUNK_DIM] = m;
          my_part[CHUNK_DIM + 1] = l;
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (merge) {  // both groups read both
          mbar_arrive(&B.o_free[0]);
          mbar_arrive(&B.o_free[1]);
        } else if (had) {
          mbar_arrive_n(&B.o_free[grp], 2);
        }
      }
      // rows that came out not finite, one after the other (not those with an l that is NaN, a score of their own not being a
      // number: they are NaN throughout as they should be)
      for (unsigned again = __ballot_sync(0xffffffffu, valid && l == l && !(bad == 0.0f)); again; again &= again - 1) {
        const int src = __ffs(again) - 1, r_prow = __shfl_sync(0xffffffffu, prow, src);
        chunk_row<BF16>(a, d.slot, __shfl_sync(0xffffffffu, out_row, src), __shfl_sync(0xffffffffu, qhead, src), d.t0 * CHUNK_KT,
                        min((d.t0 + nt) * CHUNK_KT, __shfl_sync(0xffffffffu, pos, src) + 1), lane >> 3 >= c_begin && lane >> 3 < c_end,
                        whole ? nullptr : part + r_prow * CHUNK_PART_LD, __shfl_sync(0xffffffffu, m, src));
      }
      if (!whole && grp == 0 && row == 0) {
        if (d.t0 == 0) {
          meta->row0 = d.row0;
          meta->ntok = d.ntok;
          meta->head = d.head;
          meta->pos0 = d.pos0;
          meta->state = 1;
        } else {
          meta->went_on = d.t0 + nt == d.tiles ? 2 : 1;
        }
      }
    }
  softmax_out:;
  } else if (warp == 0) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ================================================================ S = Q K^T
    if (elect_one()) {
      constexpr uint32_t idesc = chunk_idesc<BF16>(CHUNK_KT, false);
      uint32_t n_s[2] = {0, 0}, n_q[2] = {0, 0}, st = 0, parity = 0;
      const uint64_t desc_q = smem_desc_sw128(smem_u32(sm_q)), desc_k = smem_desc_sw128(smem_u32(sm_kv));
      for (uint32_t n = 0; take_one(n) == 1; ++n) {
        const ChunkBlock& d = B.block[n % CHUNK_BLOCKS];
        const int nt = d.nt, nt0 = d.nt0;
        const bool pair = d.ntok > T_tok;
        mbar_arrive(&B.block_free[n % CHUNK_BLOCKS]);
        const int place = pair ? 0 : n & 1;  // of Q; a pair takes both
        bool ok = true;
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (pair || x == place) ok = ok && wait_one(&B.q_full[x], n_q[x]++ & 1);
        for (int j = 0; ok && j < nt; ++j) {
          if (!(ok = wait_one(&B.kv_full[st], parity))) break;
          const uint64_t dk = desc_k + st * (CHUNK_STAGE_BYTES >> 4);
          // a pair's groups share the key tiles; those of a one-tile block take them in turn
          const int who = pair ? (j < nt0 ? 3 : 2) : 1 << (j & 1);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (!(who >> g & 1)) continue;
            const uint32_t c = n_s[g]++, buf = c & 1;
            // the buffer's last P has been read
            if (c >= 2 && !(ok = wait_one(&B.pv_done[g][buf], ((c >> 1) - 1) & 1))) break;
            tc_fence_after();
            const uint64_t dq = desc_q + (pair ? g : place) * (CHUNK_Q_TILE >> 4);
#pragma unroll
            for (int x = 0; x < 8; ++x)
              umma_f16_ss(tmem + g * 128 + buf * CHUNK_KT, dq + (((x >> 2) * CHUNK_Q_HALF + (x & 3) * 32) >> 4),
                          dk + (((x >> 2) * CHUNK_HALF_BYTES + (x & 3) * 32) >> 4), idesc, x > 0 ? 1u : 0u);
            umma_commit(&B.s_full[g][buf]);
          }
          umma_commit(&B.kv_free[st]);
          if (++st == CHUNK_K_STAGES) {
            st = 0;
            parity ^= 1;
          }
        }
        if (!ok) break;
        for (int x = place; x < (pair ? 2 : place + 1); ++x) umma_commit(&B.q_free[x]);
      }
    }
    __syncwarp();
  } else if (warp == 1) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ================================================================ O += P V
    if (elect_one()) {
      constexpr uint32_t idesc = chunk_idesc<BF16>(CHUNK_DIM, true);
      uint32_t n_p[2] = {0, 0}, n_out[2] = {0, 0}, n_clear = 0, st = 0, parity = 0;
      uint8_t* sm_v = sm_kv + CHUNK_K_STAGES * CHUNK_STAGE_BYTES;
      const uint64_t desc_v = smem_desc_v(smem_u32(sm_v));
      for (uint32_t n = 0; take_one(n) == 1; ++n) {
        const ChunkBlock& d = B.block[n % CHUNK_BLOCKS];
        const int nt = d.nt, nt0 = d.nt0, held = d.pos0 + d.ntok - (d.t0 + nt - 1) * CHUNK_KT;  // positions of the last tile
        const bool pair = d.ntok > T_tok;
        mbar_arrive(&B.block_free[n % CHUNK_BLOCKS]);
        bool ok = true;
        for (int j = 0; ok && j < nt; ++j) {
          if (!(ok = wait_one(&B.kv_full[CHUNK_K_STAGES + st], parity))) break;
          if (j == nt - 1 && held < CHUNK_KT) {  // behind the block's last position: rows that P's zeros must not meet
            B.clear_at = sm_v + st * CHUNK_STAGE_BYTES;
            B.clear_from = max(held, 0);
            mbar_arrive(&B.clear_ask);
            if (!(ok = wait_one(&B.clear_done, n_clear++ & 1))) break;
          }
          const uint64_t dv = desc_v + st * (CHUNK_STAGE_BYTES >> 4);
          const int who = pair ? (j < nt0 ? 3 : 2) : 1 << (j & 1);
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            if (!(who >> g & 1)) continue;
            const bool first = pair ? j == 0 : j < 2, last = pair ? j == (g ? nt : nt0) - 1 : j + 2 >= nt;
            // the block before has been read out
            if (first && n_out[g]++ && !(ok = wait_one(&B.o_free[g], n_out[g] & 1))) break;
            const uint32_t c = n_p[g]++, buf = c & 1;
            if (!(ok = wait_one(&B.p_full[g][buf], (c >> 1) & 1))) break;
            tc_fence_after();
#pragma unroll
            for (int x = 0; x < 4; ++x)
              umma_f16_ts(tmem + 256 + g * 128, tmem + g * 128 + buf * CHUNK_KT + x * 8, dv + x * (2048 >> 4), idesc,
                          (!first || x > 0) ? 1u : 0u);
            umma_commit(&B.pv_done[g][buf]);
            if (last) umma_commit(&B.o_done[g]);
          }
          umma_commit(&B.kv_free[CHUNK_K_STAGES + st]);
          if (++st == CHUNK_V_STAGES) {
            st = 0;
            parity ^= 1;
          }
        }
        if (!ok) break;
      }
    }
    __syncwarp();
  } else if (warp == 2) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ================================================================ copies
    if (elect_one()) {
      uint32_t n_q0 = 0, n_q1 = 0, st_k = 0, lap_k = 0, st_v = 0, lap_v = 0;
      const int no_row = a.pool_pages * a.layers * 2 * a.nkv * CHUNK_PAGE;  // behind the map's last row: reads as zeros
      const int page_rows = a.layers * 2 * a.nkv * CHUNK_PAGE;
      bool ok = true;
      for (uint32_t n = 0; ok && take_one(n) == 1; ++n) {
        const ChunkBlock& d = B.block[n % CHUNK_BLOCKS];
        const int ntok = d.ntok, nt = d.nt, t0 = d.t0, row0 = d.row0, head = d.head;
        const bool pair = ntok > T_tok, small = ntok <= 8;
        // pages that hold anything the block sees
        const int have = min((max(d.pos0 + ntok, 0) + CHUNK_PAGE - 1) / CHUNK_PAGE - t0, nt);
        const int* table = a.page_table + static_cast<size_t>(max(d.slot, 0)) * a.max_pages + t0;
        const int row_k = (a.layer * 2 * a.nkv + head) * CHUNK_PAGE, row_v = row_k + a.nkv * CHUNK_PAGE;
        auto load_q = [&](int x, uint32_t& used) {
          if (used && !wait_one(&B.q_free[x], (used - 1) & 1)) return false;
          ++used;
          mbar_arrive_expect_tx(&B.q_full[x], 2 * (small ? 8 : T_tok) * group * 128);
          for (int h = 0; h < 2; ++h)
            tma_load_4d(sm_q + x * CHUNK_Q_TILE + h * CHUNK_Q_HALF, small ? &q_small : &q_big, &B.q_full[x], 0, head * group,
                        row0 + (pair ? x * T_tok : 0), h);
          return true;
        };
        auto load_page = [&](int at, uint32_t lap, int page, int row_of, bool there) {
          if (lap && !wait_one(&B.kv_free[at], (lap - 1) & 1)) return false;
          if (there) {
            mbar_arrive_expect_tx(&B.kv_full[at], CHUNK_STAGE_BYTES);
            tma_load_3d(sm_kv + at * CHUNK_STAGE_BYTES, &kv_map, &B.kv_full[at], 0,
                        page < 0 || page >= a.pool_pages ? no_row : page * page_rows + row_of, 0);
          } else {
            mbar_arrive(&B.kv_full[at]);
          }
          return true;
        };
        // K runs two tiles ahead of V: K0 K1 K2 V0 K3 V1 ...  Q goes first where its place is free (one row tile: the
        // places alternate), else behind the first K, whose stages free up with the block before.
        if (!pair) ok = n & 1 ? load_q(1, n_q1) : load_q(0, n_q0);
        int id0 = -1, id1 = -1, id2 = -1, next = have > 0 ? d.pages[0] : -1;
        for (int j = 0; ok && j < nt + 2; ++j) {
          id0 = id1;
          id1 = id2;
          id2 = next;
          if (j < nt) {
            if (j + 1 < have) next = j + 1 < 16 ? d.pages[j + 1] : table[j + 1];
            ok = load_page(st_k, lap_k, id2, row_k, j < have);
            if (++st_k == CHUNK_K_STAGES) {
              st_k = 0;
              ++lap_k;
            }
            if (ok && pair && j == 0) ok = load_q(0, n_q0) && load_q(1, n_q1);
          }
          if (ok && j >= 2) {
            ok = load_page(CHUNK_K_STAGES + st_v, lap_v, id0, row_v, j - 2 < have);
            if (++st_v == CHUNK_V_STAGES) {
              st_v = 0;
              ++lap_v;
            }
          }
        }
        mbar_arrive(&B.block_free[n % CHUNK_BLOCKS]);
      }
      if (*abort_flag) {
        // copies still in flight land before the shared memory is given back: the newest of each stage, bounded
        const uint64_t t0 = globaltimer();
        for (int x = 0; x < CHUNK_K_STAGES + CHUNK_V_STAGES; ++x)
          for (uint32_t y = 0; y < 2; ++y)
            while (!mbar_try_wait(&B.kv_full[x], y) && globaltimer() - t0 < 20000000ull) {
            }
        for (uint32_t x = 0; x < 4; ++x)
          while (!mbar_try_wait(&B.q_full[x >> 1], x & 1) && globaltimer() - t0 < 40000000ull) {
          }
      }
    }
    __syncwarp();
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    // ================================================================ the walk
    ChunkWalk w;
    bool more = chunk_begin(a, w, cta, grid, bt);
    // Block n is handed on while block n - 1 is worked at; then comes the clearing for block n - 1, so nothing that a
    // block waits for ever stands behind a wait for that block.
    uint32_t n_clear = 0;
    bool clear = false, clear_before = false;  // block n, n - 1 wants V rows cleared
    for (uint32_t n = 0;; ++n) {
      if (n >= CHUNK_BLOCKS && !chunk_wait(&B.block_free[n % CHUNK_BLOCKS], (n / CHUNK_BLOCKS - 1) & 1, abort_flag)) break;
      ChunkBlock& d = B.block[n % CHUNK_BLOCKS];
      if (more) {
        const int tok0 = w.k * bt, pos0 = w.s.len - w.s.n + tok0, ntok = min(w.s.n - tok0, bt), end = pos0 + ntok;
        const int have = min((max(end, 0) + CHUNK_PAGE - 1) / CHUNK_PAGE, w.t1);
        if (lane < 16)
          d.pages[lane] = w.t0 + lane < have ? a.page_table[static_cast<size_t>(w.s.slot) * a.max_pages + w.t0 + lane] : -1;
        clear = end - (w.t1 - 1) * CHUNK_KT < CHUNK_KT;
        if (lane == 0) {
          d.row0 = w.s.row0 + tok0;
          d.ntok = ntok;
          d.pos0 = pos0;
          d.head = w.g;
          d.slot = w.s.slot;
          d.t0 = w.t0;
          d.nt = w.t1 - w.t0;
          d.tiles = w.nt;
          d.nt0 = min(max((pos0 + T_tok + CHUNK_KT - 1) / CHUNK_KT - w.t0, 0), d.nt);  // (0 where nothing is seen)
        }
      }
      __syncwarp();
      if (lane == 0) {
        d.more = more;
        mbar_arrive(&B.block_full[n % CHUNK_BLOCKS]);
      }
      if (clear_before) {
        if (!chunk_wait(&B.clear_ask, n_clear++ & 1, abort_flag)) break;
        uint8_t* v = B.clear_at;
        for (int x = B.clear_from * 8 + lane; x < CHUNK_KT * 8; x += 32) {
          reinterpret_cast<uint4*>(v)[x] = make_uint4(0, 0, 0, 0);
          reinterpret_cast<uint4*>(v + CHUNK_HALF_BYTES)[x] = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.clear_done);
      }
      if (!more) break;
      clear_before = clear;
      more = chunk_step(a, w, bt) && chunk_fit(a, w, bt);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (tid == 0 && B.abort_flag) {
    meta->state = 2;
    for (int i = 0; i < 4; ++i) meta->lost[i] = chunk_lost(i);
  }
  if (warp == 0) tmem_dealloc(tmem, 512);
}

// Joins the partials of the block that CTA blockIdx.x began and the CTAs behind it went on with: a warp a row, a lane four
// dims.  Bound by its chain of loads (what was left behind, then m and l of all parts at once, then o).
constexpr int CHUNK_COMBINE_WARPS = 8;
template <bool BF16>
__global__ void __launch_bounds__(CHUNK_COMBINE_WARPS * 32) attention_chunk_combine_kernel(const __grid_constant__ ChunkArgs a, int grid) {
  using TT = ChunkType<BF16>;
  using T = typename TT::T;
  const int lane = threadIdx.x & 31, c0 = blockIdx.x;
  const int prow = blockIdx.y * CHUNK_COMBINE_WARPS + (threadIdx.x >> 5);
  const int group = a.group, T_tok = a.tile_tokens;
  const int tok = (prow >> 7) * T_tok + (prow & 127) / group, head_of = (prow & 127) % group;
  griddep_wait();
  griddep_launch_dependents();
  auto line = [&](int c) { return reinterpret_cast<const ChunkMeta*>(a.ws + static_cast<size_t>(c) * 64); };
  const ChunkMeta mine = *line(c0);
  int next = c0 + 1 + lane < grid ? line(c0 + 1 + lane)->went_on : 0;
  if (mine.state != 1 || (prow & 127) >= T_tok * group || tok >= mine.ntok) return;
  // parts: this CTA's, then those of the CTAs that went on, up to the one that finished; 32 CTAs at a time
  const float* first = chunk_part(a, grid, 2 * c0 + 1) + prow * CHUNK_PART_LD;
  float top = first[CHUNK_DIM], sum = first[CHUNK_DIM + 1];
  float4 o = *reinterpret_cast<const float4*>(first + lane * 4);
  if (top == -INFINITY) {
    sum = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  for (int c1 = c0 + 1; c1 < grid; c1 += 32) {
    const unsigned ends = __ballot_sync(0xffffffffu, next == 2);
    unsigned on = __ballot_sync(0xffffffffu, next != 0);
    if (ends) on &= (2u << (__ffs(ends) - 1)) - 1;
    const float* part = chunk_part(a, grid, 2 * min(c1 + lane, grid - 1)) + prow * CHUNK_PART_LD;
    const float2 ml = on >> lane & 1 ? *reinterpret_cast<const float2*>(part + CHUNK_DIM) : make_float2(-INFINITY, 0.0f);
    for (; on; on &= on - 1) {
      const int i = __ffs(on) - 1;
      const float m = __shfl_sync(0xffffffffu, ml.x, i), l = __shfl_sync(0xffffffffu, ml.y, i);
      const float4 v = *reinterpret_cast<const float4*>(chunk_part(a, grid, 2 * (c1 + i)) + prow * CHUNK_PART_LD + lane * 4);
      if (m == -INFINITY) continue;  // it saw nothing of this row's: its o may be anything
      const float t = fmaxf(top, m), f0 = top == -INFINITY ? 0.0f : ex2(top - t), f1 = ex2(m - t);
      sum = sum * f0 + l * f1;
      o.x = o.x * f0 + v.x * f1;
      o.y = o.y * f0 + v.y * f1;
      o.z = o.z * f0 + v.z * f1;
      o.w = o.w * f0 + v.w * f1;
      top = t;
    }
    if (ends) break;
    next = c1 + 32 + lane < grid ? line(c1 + 32 + lane)->went_on : 0;
  }
  const float inv = mine.pos0 + tok < 0 ? 0.0f : 1.0f / sum;
  uint2 v;
  v.x = TT::from_f32(o.x * inv, o.y * inv);
  v.y = TT::from_f32(o.z * inv, o.w * inv);
  *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + static_cast<size_t>(mine.row0 + tok) * a.out_ld +
                            (mine.head * group + head_of) * CHUNK_DIM + lane * 4) = v;
}

}  // namespace qasr
