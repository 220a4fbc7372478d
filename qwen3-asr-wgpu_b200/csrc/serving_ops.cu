// C entry points of the serving step over the paged cache (include/qasr_b200_kernels.h):
// page and row maps and the append through them, chunk attention, 4-bit products.  The calls check their scalar arguments,
// enqueue on the caller's stream and return; nothing is allocated, kept or synchronised, and the
// thread's current device is put back.
#include <cuda.h>
#include <cuda_runtime.h>

#include <atomic>
#include <cmath>
#include <cstddef>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <string>

#include "attention_chunk.cuh"
#include "gemv_w4.cuh"
#include "host_gemm.cuh"
#include "kv_plan.cuh"
#include "qasr_b200_kernels.h"

using namespace qasr;

namespace {

constexpr int kMaxDevices = 16;

qasr_status op_err(char* err, int errlen, qasr_status s, const char* m) noexcept {
  if (err && errlen > 0) std::snprintf(err, errlen, "%s", m);
  return s;
}
qasr_status op_cuda(char* err, int errlen, cudaError_t e, const char* what) noexcept {
  if (err && errlen > 0) std::snprintf(err, errlen, "%s: %s", what, cudaGetErrorString(e));
  return QASR_ERR_DEVICE;
}

// `device` current for the call's length.
class DeviceScope {
 public:
  explicit DeviceScope(int device) noexcept {
    error = device < 0 || device >= kMaxDevices ? cudaErrorInvalidDevice : cudaGetDevice(&before_);
    if (error == cudaSuccess && before_ != device) {
      error = cudaSetDevice(device);
      changed_ = error == cudaSuccess;
    }
  }
  ~DeviceScope() {
    if (changed_) cudaSetDevice(before_);
  }
  DeviceScope(const DeviceScope&) = delete;
  DeviceScope& operator=(const DeviceScope&) = delete;
  cudaError_t error = cudaSuccess;

 private:
  int before_ = 0;
  bool changed_ = false;
};

bool misaligned(const void* p, uintptr_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) != 0; }

// kv_plan_kernel may want more than the 48 KB of dynamic shared memory a kernel has by default.
cudaError_t plan_attrs(int device) noexcept {
  static std::once_flag once[kMaxDevices];
  static cudaError_t result[kMaxDevices] = {};
  try {
    std::call_once(once[device], [device] {
      const int most = static_cast<int>(plan_smem_bytes(QASR_KV_PLAN_MAX_SEQS, QASR_KV_PLAN_MAX_SLOTS));
      cudaError_t e = cudaFuncSetAttribute(kv_plan_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(kv_plan_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, most);
      result[device] = e;
    });
  } catch (...) {
    return cudaErrorUnknown;
  }
  return result[device];
}

int sm_count(int device) noexcept {
  static std::atomic<int> known[kMaxDevices];
  if (device < 0 || device >= kMaxDevices) return -1;
  int n = known[device].load(std::memory_order_relaxed);
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess) return -1;
    known[device].store(n, std::memory_order_relaxed);
  }
  return n;
}

cudaError_t chunk_attrs(int device) noexcept {
  static std::once_flag once[kMaxDevices];
  static cudaError_t result[kMaxDevices] = {};
  try {
    std::call_once(once[device], [device] {
      cudaError_t e =
          cudaFuncSetAttribute(attention_chunk_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, CHUNK_SMEM);
      if (e == cudaSuccess)
        e = cudaFuncSetAttribute(attention_chunk_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, CHUNK_SMEM);
      result[device] = e;
    });
  } catch (...) {
    return cudaErrorUnknown;
  }
  return result[device];
}

bool encode_map(CUtensorMap* m, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
                const cuuint32_t* box, bool swizzle) noexcept {
  try {
    const EncodeTiledFn fn = encode_fn(nullptr);
    const cuuint32_t step[5] = {1, 1, 1, 1, 1};
    return fn && fn(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base), dims, strides, box, step,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                    CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  } catch (...) {
    return false;
  }
}

template <bool RELEASE>
qasr_status launch_plan(int device, void* stream, const PlanArgs& a, char* err, int errlen) {
  DeviceScope dev(device);
  if (dev.error != cudaSuccess) return op_cuda(err, errlen, dev.error, "device");
  cudaError_t e = plan_attrs(device);
  if (e != cudaSuccess) return op_cuda(err, errlen, e, "kernel attributes");
  // One CTA while it writes everything in a round or two, else a whole cluster (us in a graph, one CTA / eight: 8000
  // rows 5.9 / 3.7; 200 requests released, 2600 pages, 5.1 / 3.6; a decode step of 32 needs no more than one: 3.8).
  const bool small = RELEASE ? a.n_seqs <= 64 : a.n_seqs <= 256 && a.rows_cap <= PLAN_THREADS;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(small ? 1 : PLAN_MAX_CLUSTER);
  cfg.blockDim = dim3(PLAN_THREADS);
  cfg.dynamicSmemBytes = plan_smem_bytes(a.n_seqs, a.max_slots);
  cfg.stream = static_cast<cudaStream_t>(stream);
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl_enabled() ? 2 : 1;
  g_launches.fetch_add(1, std::memory_order_relaxed);
  e = cudaLaunchKernelEx(&cfg, kv_plan_kernel<RELEASE>, a);
  if (e == cudaSuccess && !RELEASE && !a.maps) {
    const int sms = sm_count(device);
    const long long ctas = (static_cast<long long>(a.rows_cap) + MAPS_THREADS * MAPS_ROWS - 1) / (MAPS_THREADS * MAPS_ROWS);
    e = sms <= 0 ? cudaErrorInvalidDevice
                 : launch_k(kv_row_maps_kernel, dim3(static_cast<unsigned>(std::min<long long>(ctas, sms * 4))), dim3(MAPS_THREADS),
                            (a.n_seqs + 1) * sizeof(int), static_cast<cudaStream_t>(stream), true, a);
  }
  return e == cudaSuccess ? QASR_OK : op_cuda(err, errlen, e, "kv plan launch");
}

bool bad_plan_sizes(int n_seqs, int max_slots, int max_pages, int pool_pages) {
  return n_seqs <= 0 || n_seqs > QASR_KV_PLAN_MAX_SEQS || max_slots <= 0 || max_slots > QASR_KV_PLAN_MAX_SLOTS ||
         max_pages <= 0 || max_pages >= (1 << 25) || pool_pages < 0;
}

bool bad_w4_sizes(int n_out, int k, int group) {
  return n_out <= 0 || k <= 0 || (group != 32 && group != 64 && group != 128) || k % group != 0 ||
         n_out > (1 << 30) || k > (1 << 30);
}

template <bool BF16, bool ZERO, int GS, int NT>
cudaError_t launch_w4_kernel(W4Args a, int device, int sms, cudaStream_t st) {
  using P = W4Plan<ZERO, GS, NT>;
  static_assert(P::slots >= 2 && P::slots * W4_WARPS * 8 <= P::bars_bytes - 16, "a ring has two slots at least");
  const auto kernel = gemv_w4_kernel<BF16, ZERO, GS, NT>;
  static std::once_flag once[kMaxDevices];
  static cudaError_t ready[kMaxDevices] = {};
  try {
    std::call_once(once[device], [kernel, device] {
      ready[device] = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, P::smem);
    });
  } catch (...) {
    return cudaErrorUnknown;
  }
  if (ready[device] != cudaSuccess) return ready[device];
  const W4Layout L = w4_layout(a.n_out, a.k, 128 / GS, ZERO);
  a.wk_log2 = 3;
  while ((1 << a.wk_log2) > L.units) --a.wk_log2;
  // Few row tiles and a long k: two or four CTAs share each tile, as long as they fit the SMs and every warp keeps a few
  // units (us, alone / shared: 2048 x 6144 at one row 5.3 / 4.4, at 32 rows 10.6 / 9.0; 2048 x 2048, where a warp would
  // be left with one unit, 2.8 / 3.15).
  a.cluster = 1;
  while (a.cluster < W4_MAX_CLUSTER && L.tiles * a.cluster * 2 <= sms && L.units >= 32 * a.cluster) a.cluster *= 2;
  const int per_cta = W4_WARPS >> a.wk_log2;
  const int groups = (L.tiles + per_cta - 1) / per_cta;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.cluster > 1 ? groups * a.cluster : std::min(groups, sms * P::per_sm));
  cfg.blockDim = dim3(W4_THREADS);
  cfg.dynamicSmemBytes = P::smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (a.cluster > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = a.cluster;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return cudaLaunchKernelEx(&cfg, kernel, a);
}
// Eight rows to an instance, doubled.  (us of 33 to 64 rows in one launch / as 32 and the rest in two: 60000 x 8192, 40 rows 263 / 209,
// 48 rows 268 / 226, 64 rows 279 / 296; 12288 x 2048, 40 rows 21.5 / 18.7, 48 rows 22.2 / 22.4, 64 rows 23.5 / 26.9; 2048 x 6144, 40
// rows 12.7 / 15.7, 64 rows 14.2 / 16.9; 1024 x 2048, 40 rows 7.95 / 7.95, 64 rows 8.7 / 10.3.  Two launches win up to 48 rows of
// large weights only; one is kept throughout.)
template <bool BF16, bool ZERO, int GS>
cudaError_t launch_w4_rows(const W4Args& a, int device, int sms, cudaStream_t st) {
  if (a.rows <= 8) return launch_w4_kernel<BF16, ZERO, GS, 1>(a, device, sms, st);
  if (a.rows <= 16) return launch_w4_kernel<BF16, ZERO, GS, 2>(a, device, sms, st);
  if (a.rows <= 32) return launch_w4_kernel<BF16, ZERO, GS, 4>(a, device, sms, st);
  return launch_w4_kernel<BF16, ZERO, GS, 8>(a, device, sms, st);
}
template <bool BF16>
cudaError_t launch_w4(const W4Args& a, int group, bool zero, int device, int sms, cudaStream_t st) {
  switch (group) {
    case 32: return zero ? launch_w4_rows<BF16, true, 4>(a, device, sms, st) : launch_w4_rows<BF16, false, 4>(a, device, sms, st);
    case 64: return zero ? launch_w4_rows<BF16, true, 2>(a, device, sms, st) : launch_w4_rows<BF16, false, 2>(a, device, sms, st);
    default: return zero ? launch_w4_rows<BF16, true, 1>(a, device, sms, st) : launch_w4_rows<BF16, false, 1>(a, device, sms, st);
  }
}

}  // namespace

extern "C" {

qasr_status qasr_kernel_kv_plan(int device, void* stream, const int* seq_slot, const int* kv_len, const int* new_len,
                                int n_seqs, int max_slots, int* page_table, int max_pages, const int* free_pages,
                                int pool_pages, const int* free_count, int* kv_len_out, int* free_count_out,
                                int* cu_rows, int* row_slot, int* row_pos, int rows_cap, int* status, char* err,
                                int errlen) {
  if (!seq_slot || !kv_len || !page_table || !free_pages || !free_count || !kv_len_out || !free_count_out || !cu_rows ||
      !row_slot || !row_pos || !status || rows_cap < 0 || bad_plan_sizes(n_seqs, max_slots, max_pages, pool_pages))
    return op_err(err, errlen, QASR_ERR_INVALID_ARG, "bad kv plan arguments");
  PlanArgs a{seq_slot, kv_len, new_len, n_seqs, max_slots, page_table, max_pages, const_cast<int*>(free_pages),
             pool_pages, free_count, kv_len_out, free_count_out, cu_rows, row_slot, row_pos, rows_cap, status, rows_cap <= PLAN_MAPS_ROWS};
  return launch_plan<false>(device, stream, a, err, errlen);
}

qasr_status qasr_kernel_kv_release(int device, void* stream, const int* seq_slot, const int* kv_len, int n_seqs,
                                   int max_slots, const int* page_table, int max_pages, int* free_pages, int pool_pages,
                                   const int* free_count, int* kv_len_out, int* free_count_out, int* status, char* err,
                                   int errlen) {
  if (!seq_slot || !kv_len || !page_table || !free_pages || !free_count || !kv_len_out || !free_count_out || !status ||
      bad_plan_sizes(n_seqs, max_slots, max_pages, pool_pages))
    return op_err(err, errlen, QASR_ERR_INVALID_ARG, "bad kv release arguments");
  PlanArgs a{seq_slot, kv_len, nullptr, n_seqs, max_slots, const_cast<int*>(page_table), max_pages, free_pages,
             pool_pages, free_count, kv_len_out, free_count_out, nullptr, nullptr, nullptr, 0, status, 0};
  return launch_plan<true>(device, stream, a, err, errlen);
}

qasr_status qasr_kernel_kv_append_planned(int device, void* stream, const uint16_t* k, const uint16_t* v, uint16_t* kv_pool,
                                          int pool_pages, const int* page_table, int max_slots, int max_pages, int layers,
                                          int nkv, int layer, const int* row_slot, const int* row_pos, int rows_cap,
                                          const int* row_count, char* err, int errlen) {
  if (!k || !v || !kv_pool || !page_table || !row_slot || !row_pos || !row_count || pool_pages <= 0 || max_slots <= 0 ||
      max_pages <= 0 || max_pages >= (1 << 25) || layers <= 0 || layer < 0 || layer >= layers || nkv <= 0 || nkv > (1 << 20) ||
      rows_cap <= 0 || misaligned(k, 16) || misaligned(v, 16) || misaligned(kv_pool, 16))
    return op_err(err, errlen, QASR_ERR_INVALID_ARG, "bad planned kv append arguments");
  DeviceScope dev(device);
  if (dev.error != cudaSuccess) return op_cuda(err, errlen, dev.error, "device");
  const int sms = sm_count(device);
  if (sms <= 0) return op_err(err, errlen, QASR_ERR_DEVICE, "device attributes");
  const AppendArgs a{reinterpret_cast<const uint4*>(k), reinterpret_cast<const uint4*>(v), reinterpret_cast<uint4*>(kv_pool),
                     pool_pages, page_table, max_slots, max_pages, layers, nkv, layer, row_slot, row_pos, rows_cap, row_count};
  const long long ctas = (static_cast<long long>(rows_cap) * nkv * 16 + APPEND_THREADS - 1) / APPEND_THREADS;
  const cudaError_t e = launch_k(kv_append_planned_kernel, dim3(static_cast<unsigned>(std::min<long long>(ctas, sms * 8))),
                                 dim3(APPEND_THREADS), 0, static_cast<cudaStream_t>(stream), true, a);
  return e == cudaSuccess ? QASR_OK : op_cuda(err, errlen, e, "planned kv append launch");
}

int64_t qasr_kernel_attention_chunk_workspace(int device) {
  const int sms = sm_count(device);
  return sms <= 0 ? -1 : chunk_ws_bytes(sms);
}

qasr_status qasr_kernel_attention_chunk(int device, void* stream, int type, const void* q, int q_ld, void* out,
                                        int out_ld, int rows, const void* kv_pool, int pool_pages,
                                        const int* page_table, int max_slots, int max_pages, int layers, int nq,
                                        int nkv, int layer, const int* seq_slot, const int* cu_rows, const int* kv_len,
                                        int n_seqs, float scale, void* ws, int64_t ws_bytes, char* err, int errlen) {
  if (!q || !out || !kv_pool || !page_table || !seq_slot || !cu_rows || !kv_len || !ws || rows <= 0 || n_seqs <= 0 ||
      pool_pages <= 0 || max_slots <= 0 || max_pages <= 0 || max_pages >= (1 << 25) || layers <= 0 || layer < 0 ||
      layer >= layers || nkv <= 0 || nq <= 0 || nq % nkv != 0 || nq / nkv > 16 || nq > (1 << 20) ||
      q_ld < nq * CHUNK_DIM || out_ld < nq * CHUNK_DIM || q_ld % 8 || out_ld % 8 || misaligned(q, 16) ||
      misaligned(out, 16) || misaligned(kv_pool, 16) || misaligned(ws, 256) || !(std::fabs(scale) < 0x1p127f) ||
      (type != QASR_TYPE_F16 && type != QASR_TYPE_BF16) ||
      static_cast<__int128>(pool_pages) * layers * 2 * nkv * CHUNK_PAGE > 0x7fffffff)
    return op_err(err, errlen, QASR_ERR_INVALID_ARG, "bad chunk attention arguments");
  DeviceScope dev(device);
  if (dev.error != cudaSuccess) return op_cuda(err, errlen, dev.error, "device");
  const int grid = sm_count(device);
  if (grid <= 0 || grid > 512) return op_err(err, errlen, QASR_ERR_DEVICE, "device attributes");
  if (ws_bytes < chunk_ws_bytes(grid))
    return op_err(err, errlen, QASR_ERR_CAPACITY, "chunk attention workspace too small");
  cudaError_t e = chunk_attrs(device);
  if (e != cudaSuccess) return op_cuda(err, errlen, e, "kernel attributes");
  const int group = nq / nkv;
  const uint64_t kv_rows = static_cast<uint64_t>(pool_pages) * layers * 2 * nkv * CHUNK_PAGE;
  // Q as {64 dims, heads, rows, 2 halves}: a box is one half of a group's heads of some rows, in the order in which
  // a row tile packs them, under the tensor core's 128-byte swizzle.  The cache as {64 dims, rows, 2
  // halves}: a box is a page, half after half, copied as it is (its rows are swizzled already).
  CUtensorMap q_big, q_small, kv_map;
  const cuuint64_t q_dims[4] = {64, static_cast<cuuint64_t>(nq), static_cast<cuuint64_t>(rows), 2};
  const cuuint64_t q_strides[3] = {CHUNK_DIM * 2, static_cast<cuuint64_t>(q_ld) * 2, 128};
  const cuuint32_t big[4] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(chunk_tile_tokens(group)), 1};
  const cuuint32_t small[4] = {64, static_cast<cuuint32_t>(group), 8, 1};
  const cuuint64_t kv_dims[3] = {64, kv_rows, 2}, kv_strides[2] = {CHUNK_DIM * 2, 128};
  const cuuint32_t kv_box[3] = {64, CHUNK_PAGE, 2};
  if (!encode_map(&q_big, q, 4, q_dims, q_strides, big, true) || !encode_map(&q_small, q, 4, q_dims, q_strides, small, true) ||
      !encode_map(&kv_map, kv_pool, 3, kv_dims, kv_strides, kv_box, false))
    return op_err(err, errlen, QASR_ERR_DEVICE, "chunk attention tensor maps");
  // A scale of 0 becomes the smallest number: masked scores stay -inf under it, and no finite score moves a probability
  // by more than 2^-20 (2^128 * 2^-149).
  const float s2 = scale == 0.0f ? 0x1p-149f : std::fabs(scale) * 1.4426950408889634f;
  const ChunkArgs a{q, q_ld, out, out_ld, rows, kv_pool, pool_pages, page_table, max_slots, max_pages, layers, nq, nkv,
                    layer, group, chunk_tile_tokens(group), seq_slot, cu_rows, kv_len, n_seqs, s2, scale < 0.0f, static_cast<uint8_t*>(ws)};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool bf = type == QASR_TYPE_BF16;
  e = bf ? launch_k(attention_chunk_kernel<true>, dim3(grid), dim3(CHUNK_THREADS), CHUNK_SMEM, st, true, q_big, q_small, kv_map, a)
         : launch_k(attention_chunk_kernel<false>, dim3(grid), dim3(CHUNK_THREADS), CHUNK_SMEM, st, true, q_big, q_small, kv_map, a);
  if (e != cudaSuccess) return op_cuda(err, errlen, e, "chunk attention launch");
  // a warp per packed row of a block, of which none has more than the call
  const int packed = rows <= chunk_tile_tokens(group) ? rows * group : CHUNK_PART_ROWS;
  const dim3 cgrid(grid, (packed + CHUNK_COMBINE_WARPS - 1) / CHUNK_COMBINE_WARPS);
  e = bf ? launch_k(attention_chunk_combine_kernel<true>, cgrid, dim3(CHUNK_COMBINE_WARPS * 32), 0, st, true, a, grid)
         : launch_k(attention_chunk_combine_kernel<false>, cgrid, dim3(CHUNK_COMBINE_WARPS * 32), 0, st, true, a, grid);
  return e == cudaSuccess ? QASR_OK : op_cuda(err, errlen, e, "chunk attention combine launch");
}

qasr_status qasr_kernel_attention_chunk_check(int device, void* stream, void* ws, char* err, int errlen) {
  if (!ws || misaligned(ws, 256)) return op_err(err, errlen, QASR_ERR_INVALID_ARG, "bad chunk attention workspace");
  DeviceScope dev(device);
  if (dev.error != cudaSuccess) return op_cuda(err, errlen, dev.error, "device");
  const int grid = sm_count(device);
  static_assert(sizeof(ChunkMeta) <= 64, "one 64-byte line per CTA");
  if (grid <= 0 || grid > 512) return op_err(err, errlen, QASR_ERR_DEVICE, "device attributes");
  alignas(8) unsigned char lines[512 * 64];
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemcpyAsync(lines, ws, static_cast<size_t>(grid) * 64, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return op_cuda(err, errlen, e, "chunk attention status");
  bool lost = false;
  for (int c = 0; c < grid; ++c) {
    ChunkMeta m;
    std::memcpy(&m, lines + c * 64, sizeof m);
    lost |= m.lost[0] == chunk_lost(0) && m.lost[1] == chunk_lost(1) && m.lost[2] == chunk_lost(2) && m.lost[3] == chunk_lost(3);
  }
  if (!lost) return QASR_OK;
  e = cudaMemset2DAsync(static_cast<uint8_t*>(ws) + offsetof(ChunkMeta, lost), 64, 0, sizeof ChunkMeta::lost, grid, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return op_cuda(err, errlen, e, "chunk attention status");
  return op_err(err, errlen, QASR_ERR_DEVICE_TIMEOUT, "a device-side wait of the chunk attention timed out");
}

int64_t qasr_kernel_w4_packed_bytes(int n_out, int k, int group, int has_zero) {
  return bad_w4_sizes(n_out, k, group) ? -1 : w4_layout(n_out, k, group, has_zero != 0).total;
}

qasr_status qasr_kernel_pack_w4(int device, void* stream, const uint8_t* codes, const uint16_t* scale,
                                const uint8_t* zero, int n_out, int k, int group, void* packed, char* err, int errlen) {
  if (!codes || !scale || !packed || bad_w4_sizes(n_out, k, group) || misaligned(packed, 16))
    return op_err(err, errlen, QASR_ERR_INVALID_ARG, "bad w4 pack arguments");
  DeviceScope dev(device);
  if (dev.error != cudaSuccess) return op_cuda(err, errlen, dev.error, "device");
  const cudaError_t e = launch_k(pack_w4_kernel, dim3(148 * 8), dim3(256), 0, static_cast<cudaStream_t>(stream), false,
                                 codes, scale, zero, n_out, k, group, static_cast<uint8_t*>(packed));
  return e == cudaSuccess ? QASR_OK : op_cuda(err, errlen, e, "w4 pack launch");
}

qasr_status qasr_kernel_gemv_w4(int device, void* stream, int type, const void* packed, int has_zero, int n_out, int k,
                                int group, const void* x, int ldx, int rows, void* out, int ldo, int accumulate,
                                char* err, int errlen) {
  if (!packed || !x || !out || bad_w4_sizes(n_out, k, group) || rows <= 0 || rows > QASR_W4_MAX_ROWS || ldx < k ||
      ldx % 8 || ldo < n_out || misaligned(packed, 16) || misaligned(x, 16) || misaligned(out, 2) ||
      (type != QASR_TYPE_F16 && type != QASR_TYPE_BF16))
    return op_err(err, errlen, QASR_ERR_INVALID_ARG, "bad w4 gemv arguments");
  DeviceScope dev(device);
  if (dev.error != cudaSuccess) return op_cuda(err, errlen, dev.error, "device");
  const int sms = sm_count(device);
  if (sms <= 0) return op_err(err, errlen, QASR_ERR_DEVICE, "device attributes");
  const W4Args a{static_cast<const uint8_t*>(packed), n_out, k, x, ldx, rows, out, ldo, accumulate != 0, 0, 1};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = type == QASR_TYPE_BF16 ? launch_w4<true>(a, group, has_zero != 0, device, sms, st)
                                               : launch_w4<false>(a, group, has_zero != 0, device, sms, st);
  return e == cudaSuccess ? QASR_OK : op_cuda(err, errlen, e, "w4 gemv launch");
}

qasr_status qasr_kernel_gemv_w4_check(int device, void* stream, char* err, int errlen) {
  DeviceScope dev(device);
  if (dev.error != cudaSuccess) return op_cuda(err, errlen, dev.error, "device");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  uint32_t got[2] = {0, 0}, none[2] = {0, 0};
  cudaError_t e = cudaMemcpyFromSymbolAsync(got, w4_status, sizeof got, 0, cudaMemcpyDeviceToHost, st);
  if (e == cudaSuccess) e = cudaStreamSynchronize(st);
  if (e == cudaSuccess && got[0]) e = cudaMemcpyToSymbolAsync(w4_status, none, sizeof none, 0, cudaMemcpyHostToDevice, st);
  if (e == cudaSuccess && got[0]) e = cudaStreamSynchronize(st);
  if (e != cudaSuccess) return op_cuda(err, errlen, e, "w4 gemv status");
  return got[0] ? op_err(err, errlen, QASR_ERR_DEVICE_TIMEOUT, "a device-side wait of a w4 gemv timed out") : QASR_OK;
}

}  // extern "C"
