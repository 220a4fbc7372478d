// Page table entries and row maps of a serving step, built on the device from the requests'
// lengths, and the return of finished requests' pages to the free stack.
//
// With a_i positions held, n_i added and pages of 64: two exclusive scans over the requests
// (rows n_i, pages ceil((a_i + n_i) / 64) - ceil(a_i / 64)) place every output; the rest is a gather off
// the free stack and an expansion of the row scan.  Nothing to compute: a step of 32 requests is
// bound by one launch and the few dependent reads below, a large admission by the row maps it
// writes (8 bytes a row).
//
// One cluster does the scans and the pages, and the row maps as well where they are short; long ones (more than
// PLAN_MAPS_ROWS) are left to kv_row_maps_kernel on all SMs, which expands the finished scan.  (us in a graph, cluster
// alone / both: 8000 rows 3.8 / 5.1, 24,000 rows 4.5 / 5.2, 32,000 4.95 / 5.2, 40,000 5.4 / 5.25, 64,000 6.8 / 5.4, 1.1
// million 81 / 9.8.)  Every CTA of the cluster reads the lengths and scans them for itself (a few KB out
// of L2, cheaper than handing the sums over); a cluster barrier then stands between the last
// read and the first write, so that the outputs may be the inputs' own arrays, and the CTAs
// share the writes.
#pragma once
#include "device_common.cuh"
#include "gemm_tc.cuh"  // griddep_*
#include "qasr_b200_kernels.h"

namespace qasr {

constexpr int PLAN_THREADS = 1024;
constexpr int PLAN_MAX_CLUSTER = 8;  // the portable cluster size
constexpr int PLAN_MAPS_ROWS = 4 * PLAN_MAX_CLUSTER * PLAN_THREADS;

struct PlanArgs {
  const int* seq_slot;
  const int* kv_len;
  const int* new_len;  // null: 1 each
  int n_seqs, max_slots;
  int* page_table;
  int max_pages;
  int* free_pages;
  int pool_pages;
  const int* free_count;
  int* kv_len_out;
  int* free_count_out;
  int* cu_rows;
  int* row_slot;
  int* row_pos;
  int rows_cap;
  int* status;
  int maps;  // the row maps are written here
};

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}

// dynamic shared memory: per request the first row, first page, kv_len and slot, then one bit per slot
__host__ __device__ __forceinline__ size_t plan_smem_bytes(int n_seqs, int max_slots) {
  return static_cast<size_t>(4) * (4 * static_cast<size_t>(n_seqs) + 2 + (max_slots + 31) / 32);
}

template <bool RELEASE>
__global__ void __launch_bounds__(PLAN_THREADS) kv_plan_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int plan_smem[];
  __shared__ long long warp_rows[32], warp_pages[32];
  __shared__ long long base_rows, base_pages;
  __shared__ int first_bad, first_full;
  const int n = a.n_seqs, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int* row0 = plan_smem;             // [n + 1]
  int* page0 = row0 + n + 1;         // [n + 1]
  int* held = page0 + n + 1;         // [n]
  int* slot = held + n;              // [n]
  unsigned int* seen = reinterpret_cast<unsigned int*>(slot + n);  // [ceil(max_slots / 32)]
  for (int i = tid; i < (a.max_slots + 31) / 32; i += PLAN_THREADS) seen[i] = 0;
  if (tid == 0) {
    base_rows = base_pages = 0;
    first_bad = first_full = 0x7fffffff;
  }
  griddep_wait();
  griddep_launch_dependents();
  const int free_count = a.free_count[0];
  __syncthreads();

  const long long max_pos = static_cast<long long>(a.max_pages) * 64;
  for (int i0 = 0; i0 < n; i0 += PLAN_THREADS) {
    const int i = i0 + tid;
    long long rows = 0, pages = 0;
    if (i < n) {
      const int s = a.seq_slot[i], h = a.kv_len[i], add = RELEASE ? 0 : (a.new_len ? a.new_len[i] : 1);
      held[i] = h;
      slot[i] = s;
      if (s < 0 || s >= a.max_slots || h < 0 || h > max_pos || add < 0) {
        atomicMin(&first_bad, i);
      } else {
        const long long end = static_cast<long long>(h) + add;
        if (end > max_pos) atomicMin(&first_full, i);
        rows = add;
        pages = RELEASE ? (h + 63) >> 6 : ((end + 63) >> 6) - ((h + 63) >> 6);
      }
    }
    long long r = rows, p = pages;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long r2 = __shfl_up_sync(0xffffffffu, r, o), p2 = __shfl_up_sync(0xffffffffu, p, o);
      if (lane >= o) r += r2, p += p2;
    }
    if (lane == 31) warp_rows[warp] = r, warp_pages[warp] = p;
    __syncthreads();
    if (warp == 0) {
      long long wr = warp_rows[lane], wp = warp_pages[lane];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long r2 = __shfl_up_sync(0xffffffffu, wr, o), p2 = __shfl_up_sync(0xffffffffu, wp, o);
        if (lane >= o) wr += r2, wp += p2;
      }
      warp_rows[lane] = wr;
      warp_pages[lane] = wp;
    }
    __syncthreads();
    // sums past 31 bits are cut here and refused below, by the totals
    const long long br = base_rows + (warp ? warp_rows[warp - 1] : 0) + r;
    const long long bp = base_pages + (warp ? warp_pages[warp - 1] : 0) + p;
    if (i < n) {
      row0[i + 1] = static_cast<int>(min(br, 0x7fffffffll));
      page0[i + 1] = static_cast<int>(min(bp, 0x7fffffffll));
    }
    __syncthreads();
    if (tid == 0) {
      base_rows += warp_rows[31];
      base_pages += warp_pages[31];
    }
    __syncthreads();
  }
  if (tid == 0) row0[0] = page0[0] = 0;
  // a slot listed twice: every listing but the first is bad.  The bit is set in request order
  // (one pass per warp-sized step would be exact but slow); instead any clash sends thread 0
  // over the list once.
  __shared__ int clash;
  if (tid == 0) clash = 0;
  __syncthreads();
  for (int i = tid; i < n; i += PLAN_THREADS) {
    const int s = slot[i];
    if (s >= 0 && s < a.max_slots && ((atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31)) & 1)) clash = 1;
  }
  __syncthreads();
  if (clash) {
    for (int i = tid; i < (a.max_slots + 31) / 32; i += PLAN_THREADS) seen[i] = 0;
    __syncthreads();
    if (tid == 0) {
      for (int i = 0; i < n; ++i) {
        const int s = slot[i];
        if (s < 0 || s >= a.max_slots) continue;
        if ((seen[s >> 5] >> (s & 31)) & 1) {
          if (i < first_bad) first_bad = i;
          break;
        }
        seen[s >> 5] |= 1u << (s & 31);
      }
    }
    __syncthreads();
  }
  const long long rows = base_rows, pages = base_pages;
  int code = 0, where = 0;
  if (first_bad != 0x7fffffff) {
    code = QASR_ERR_INVALID_ARG, where = first_bad;
  } else if (free_count < 0 || free_count > a.pool_pages) {
    code = QASR_ERR_INVALID_ARG, where = -3;
  } else if (first_full != 0x7fffffff) {
    code = QASR_ERR_CAPACITY, where = first_full;
  } else if (RELEASE ? free_count + pages > a.pool_pages : pages > free_count) {
    code = QASR_ERR_CAPACITY, where = -1;
  } else if (!RELEASE && rows > a.rows_cap) {
    code = QASR_ERR_CAPACITY, where = -2;
  }
  // every input but the page ids is in registers and shared memory now, in every CTA
  cluster_sync_all();

  const int ctas = gridDim.x, me = blockIdx.x;
  const int gt = me * PLAN_THREADS + tid, threads = ctas * PLAN_THREADS;
  if (gt == 0) {
    a.status[0] = code;
    a.status[1] = where;
    a.free_count_out[0] = code ? free_count : static_cast<int>(RELEASE ? free_count + pages : free_count - pages);
  }
  if (code) {
    for (int i = gt; i <= n; i += threads) {
      if (!RELEASE) a.cu_rows[i] = 0;
      if (i < n) a.kv_len_out[i] = held[i];
    }
    return;
  }
  for (int i = gt; i <= n; i += threads) {
    if (!RELEASE) a.cu_rows[i] = row0[i];
    if (i < n) a.kv_len_out[i] = RELEASE ? 0 : held[i] + (row0[i + 1] - row0[i]);
  }
  // pages: the page's request by bisection of the page scan
  for (int p = gt; p < static_cast<int>(pages); p += threads) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (page0[mid] <= p) lo = mid; else hi = mid - 1;
    }
    const size_t line = static_cast<size_t>(slot[lo]) * a.max_pages;
    if (RELEASE)
      a.free_pages[free_count + p] = a.page_table[line + (p - page0[lo])];
    else
      a.page_table[line + ((held[lo] + 63) >> 6) + (p - page0[lo])] = a.free_pages[free_count - 1 - p];
  }
  for (int r = gt; !RELEASE && a.maps && r < static_cast<int>(rows); r += threads) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (row0[mid] <= r) lo = mid; else hi = mid - 1;
    }
    a.row_slot[r] = slot[lo];
    a.row_pos[r] = held[lo] + (r - row0[lo]);
  }
}

constexpr int MAPS_THREADS = 256;
constexpr int MAPS_ROWS = 4;  // consecutive rows of a thread: one 16-byte store to each map

// row_slot / row_pos of the rows that cu_rows gives the requests (none after a refused plan, whose cu_rows are 0).
__global__ void __launch_bounds__(MAPS_THREADS) kv_row_maps_kernel(const __grid_constant__ PlanArgs a) {
  extern __shared__ int first_row[];  // [n_seqs + 1]
  griddep_wait();
  griddep_launch_dependents();
  const int n = a.n_seqs;
  for (int i = threadIdx.x; i <= n; i += MAPS_THREADS) first_row[i] = a.cu_rows[i];
  __syncthreads();
  const int rows = min(first_row[n], a.rows_cap);
  const bool wide = ((reinterpret_cast<uintptr_t>(a.row_slot) | reinterpret_cast<uintptr_t>(a.row_pos)) & 15) == 0;
  const long long step = static_cast<long long>(gridDim.x) * MAPS_THREADS * MAPS_ROWS;
  for (long long r0 = (static_cast<long long>(blockIdx.x) * MAPS_THREADS + threadIdx.x) * MAPS_ROWS; r0 < rows; r0 += step) {
    int lo = 0, hi = n - 1;  // the last request that starts at or before r0
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first_row[mid] <= r0) lo = mid; else hi = mid - 1;
    }
    int slot[MAPS_ROWS], pos[MAPS_ROWS];
    int s = a.seq_slot[lo], base = a.kv_len_out[lo] - first_row[lo + 1];  // position of row r: base + r
#pragma unroll
    for (int x = 0; x < MAPS_ROWS; ++x) {
      const int r = static_cast<int>(r0) + x;
      if (r < rows && r >= first_row[lo + 1]) {
        do ++lo; while (first_row[lo + 1] <= r);
        s = a.seq_slot[lo];
        base = a.kv_len_out[lo] - first_row[lo + 1];
      }
      slot[x] = s;
      pos[x] = base + r;
    }
    if (wide && r0 + MAPS_ROWS <= rows) {
      *reinterpret_cast<int4*>(a.row_slot + r0) = make_int4(slot[0], slot[1], slot[2], slot[3]);
      *reinterpret_cast<int4*>(a.row_pos + r0) = make_int4(pos[0], pos[1], pos[2], pos[3]);
    } else {
#pragma unroll
      for (int x = 0; x < MAPS_ROWS; ++x)
        if (r0 + x < rows) {
          a.row_slot[r0 + x] = slot[x];
          a.row_pos[r0 + x] = pos[x];
        }
    }
  }
}

// The planned step's new K and V rows, written through its maps.  Only the rows that the plan gave out are
// written (their count is read here: a refused plan has none, and its maps are an earlier step's), and no entry of
// the maps or of the table is followed out of its range.  A copy: each thread moves 16 bytes of K and of V.
// Measured (B200, us in a graph, 8 kv heads): 32 rows 2.0 (a launch and a chain of three reads), 832 rows 2.5, 8192 rows 8.1
// (67 MB, partly out of L2).
constexpr int APPEND_THREADS = 256;
struct AppendArgs {
  const uint4 *k, *v;
  uint4* pool;
  int pool_pages;
  const int* page_table;
  int max_slots, max_pages, layers, nkv, layer;
  const int *row_slot, *row_pos;
  int rows_cap;
  const int* row_count;
};
__global__ void __launch_bounds__(APPEND_THREADS) kv_append_planned_kernel(const __grid_constant__ AppendArgs a) {
  constexpr int CHUNKS = 16;  // of 16 bytes in a row of 128
  griddep_wait();
  griddep_launch_dependents();
  const long long all = static_cast<long long>(min(a.row_count[0], a.rows_cap)) * a.nkv * CHUNKS;
  const long long step = static_cast<long long>(gridDim.x) * APPEND_THREADS;
  for (long long e = static_cast<long long>(blockIdx.x) * APPEND_THREADS + threadIdx.x; e < all; e += step) {
    const long long rh = e / CHUNKS;
    const int c = static_cast<int>(e % CHUNKS), r = static_cast<int>(rh / a.nkv), h = static_cast<int>(rh % a.nkv);
    const int slot = a.row_slot[r], pos = a.row_pos[r];
    if (slot < 0 || slot >= a.max_slots || pos < 0 || pos >> 6 >= a.max_pages) continue;
    const int page = a.page_table[static_cast<size_t>(slot) * a.max_pages + (pos >> 6)];
    if (page < 0 || page >= a.pool_pages) continue;
    const long long k_row = (((static_cast<long long>(page) * a.layers + a.layer) * 2) * a.nkv + h) * 64 + (pos & 63);
    const int at = c ^ (pos & 7);
    a.pool[k_row * CHUNKS + at] = a.k[e];
    a.pool[(k_row + static_cast<long long>(a.nkv) * 64) * CHUNKS + at] = a.v[e];
  }
}

}  // namespace qasr
