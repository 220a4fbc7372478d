/*
 * qasr_b200_kernels.h — device-pointer entry points of the individual B200 kernels.
 *
 * The reference checks and measures its kernels one by one with dedicated probes:
 * src/bin/w8_probe.rs (W8 GEMV/GEMM vs an f64 reference), src/bin/batch_gemv_bench.rs
 * (batched GEMV bandwidth), src/bin/attn_bench.rs and src/bin/attn_slots_probe.rs
 * (decode attention).  These calls are the same seams for the B200 kernels: all
 * pointers are device pointers, `stream` is a cudaStream_t (NULL = legacy default
 * stream), nothing is synchronised.  Workspaces are cached per device inside the
 * library and only grow.  Errors are written to `err` (if non-NULL, `errlen` bytes).
 */
#ifndef QASR_B200_KERNELS_H
#define QASR_B200_KERNELS_H

#include <stdint.h>

#include "qasr_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Re-lay a row-major weight [n_out, k] (f16 or int8) into the tiled HBM layout the
 * GEMM streams: 16 KB blocks of 128 rows x 128 bytes, one per (row tile, k block),
 * 128-byte swizzle applied.  w_tiled must hold n_out * k * element-size bytes.
 * (The reference uploads the file bytes verbatim, src/weights.rs:300-308; the B200
 * loader re-lays them once at load.) */
qasr_status qasr_kernel_pack_weights(int device, void* stream, int weight_format,
                                     const void* w_rowmajor, int n_out, int k, void* w_tiled,
                                     char* err, int errlen);

/* out[r, m] = f16(sum_k W[m, k] x[r, k])            (accumulate == 0)
 * out[r, m] = f16(f32(out[r, m]) + sum_k ...)         (accumulate != 0)
 * W: [n_out, k] f16 (weight_format QASR_WEIGHTS_F16) or int8 + a per-row scale, f16
 * (QASR_WEIGHTS_INT8) or f32 (QASR_WEIGHTS_INT8_F32), value f16(f32(q) * s), in the
 * layout qasr_kernel_pack_weights produces.  n_out % 128 == 0; k % 128 == 0; x is
 * [rows, ldx] and out [rows, ldo] f16 with ldx >= k, ldo >= n_out (ldx * 2 a multiple of
 * 16 bytes, the activation copy's stride).
 * Replaces gemv / gemv_w8 / gemv_batch_slots / prefill_gemm(_w8)
 * (src/shaders.rs:273-889, 2995-3082). */
qasr_status qasr_kernel_gemm(int device, void* stream, int weight_format, const void* w,
                             const void* scale, int n_out, int k, const uint16_t* x, int ldx,
                             int rows, uint16_t* out, int ldo, int accumulate, char* err,
                             int errlen);

/* qasr_kernel_gemm with a latency trace: if `trace` (device, grid * 12 uint64) is
 * non-NULL each CTA records %globaltimer stamps of its pipeline milestones (entry, setup,
 * first weight/activation copies issued, first stage seen/built, first/last MMA, first
 * accumulator, last store, split fixup, exit); *grid_out receives the CTA count. */
qasr_status qasr_kernel_gemm_traced(int device, void* stream, int weight_format, const void* w,
                                    const void* scale, int n_out, int k, const uint16_t* x,
                                    int ldx, int rows, uint16_t* out, int ldo, int accumulate,
                                    unsigned long long* trace, int* grid_out, char* err,
                                    int errlen);

/* GQA attention of `rows` query rows over their slot's paged KV (gqa_decode_* /
 * gqa_split_merge, src/shaders.rs:1881-2905).  q/out: [rows, q_ld] f16 (q heads 2g and
 * 2g+1 read kv head g); kv_pool: [pages][layers][2][nkv][64][128] f16 with each
 * 128-dim row stored swizzled: dim d of position p sits at column
 * ((d/8) ^ (p%8))*8 + d%8 (16-byte chunks permuted by the position's low 3 bits, so
 * tensor-core fragment loads from shared memory are bank-conflict free); page_table:
 * [slots][max_pages] int32; row r attends positions 0..row_pos[r] of slot row_slot[r].
 * The device arrays are taken as given (the call checks only its scalar arguments):
 * row_pos[r] < max_pages * 64, and every page id the rows reach lies in kv_pool.
 * Only enqueues (for timing with the caller's events): a bounded device-side wait that
 * gives up is not reported by this call; the traced and no-alloc variants report it. */
qasr_status qasr_kernel_attention(int device, void* stream, const uint16_t* q, int q_ld,
                                  uint16_t* out, const uint16_t* kv_pool, const int* page_table,
                                  int max_pages, int layers, int nkv, int layer,
                                  const int* row_slot, const int* row_pos, int rows, char* err,
                                  int errlen);

/* qasr_kernel_attention with a latency trace: if `trace` (device, SM count x 8 uint64) is
 * non-NULL each CTA records %globaltimer stamps (entry, unit table ready, first stage
 * landed, first unit merged, last stage consumed, last unit merged, producer done) and
 * the number of units it processed.  Waits for its launches and returns
 * QASR_ERR_DEVICE_TIMEOUT if a bounded device-side wait gave up. */
qasr_status qasr_kernel_attention_traced(int device, void* stream, const uint16_t* q, int q_ld,
                                         uint16_t* out, const uint16_t* kv_pool,
                                         const int* page_table, int max_pages, int layers,
                                         int nkv, int layer, const int* row_slot,
                                         const int* row_pos, int rows, unsigned long long* trace,
                                         char* err, int errlen);

/* qasr_kernel_attention without any device allocation — for callers that may not call
 * cudaMalloc: hosts that hand the library a fixed memory budget up front (an embedding
 * application that owns all device memory), and real-time audio paths that must not
 * touch the allocator between frames (an allocation can block on the driver for
 * milliseconds).  No counterpart in the reference (its wgpu decoder owns all buffers).
 * The scratch is one static device array inside the library (about 2 MiB) plus an
 * 8-byte status word, held by every GPU that loads the library until the process exits, so:
 *   - at most 64 query rows and 8 kv heads per call; larger calls fail with
 *     QASR_ERR_CAPACITY (use qasr_kernel_attention);
 *   - the first call on a device looks the array's address up
 *     (cudaGetSymbolAddress): make that first call before any stream capture;
 *   - all calls share the array and the status word: calls that overlap on the GPU
 *     (other streams, other threads) race and must be serialised by the caller;
 *   - the call waits for its kernels on `stream` and reads the status word back, so a
 *     bounded device-side wait that gave up returns QASR_ERR_DEVICE_TIMEOUT.
 * Same inputs, outputs and results as qasr_kernel_attention. */
qasr_status qasr_kernel_attention_noalloc(int device, void* stream, const uint16_t* q, int q_ld,
                                          uint16_t* out, const uint16_t* kv_pool,
                                          const int* page_table, int max_pages, int layers,
                                          int nkv, int layer, const int* row_slot,
                                          const int* row_pos, int rows, char* err, int errlen);

/* Append K and V rows ([rows, nkv*128] f16 each) at (row_slot[r], row_pos[r]) of
 * layer `layer`, in the swizzled row layout qasr_kernel_attention reads — the cache
 * writes of qkv_extract(_slots) (src/shaders.rs:1376-1635).  All `rows` are written and their maps and the
 * table taken as given; a step planned on the device has qasr_kernel_kv_append_planned. */
qasr_status qasr_kernel_kv_append(int device, void* stream, const uint16_t* k, const uint16_t* v,
                                  uint16_t* kv_pool, const int* page_table, int max_pages,
                                  int layers, int nkv, int layer, const int* row_slot,
                                  const int* row_pos, int rows, char* err, int errlen);

/* ------------------------------------------------------------------ serving over the paged cache
 * A serving step on the device, with no read-back of lengths to the host: qasr_kernel_kv_plan
 * gives each request the pages and row maps of its new positions, the projections may read 4-bit
 * weights (qasr_kernel_gemv_w4), qasr_kernel_kv_append_planned writes the new rows, and
 * qasr_kernel_attention_chunk attends them.  No counterpart in the reference, whose decoder
 * keeps one contiguous cache per slot (fork_capped, src/decoder.rs:2453).
 * These calls allocate nothing and keep nothing between calls, so they may be captured into a
 * CUDA graph, and they leave the calling thread's current device as it was. */

/* Element types of activations and caches. */
enum {
  QASR_TYPE_F16 = 0,
  QASR_TYPE_BF16 = 1
};

#define QASR_KV_PLAN_MAX_SEQS 8192
#define QASR_KV_PLAN_MAX_SLOTS 65536

/* Page table entries and row maps of one step, from the requests' lengths (device int32
 * arrays).  Request i (0 <= i < n_seqs) holds kv_len[i] positions in slot seq_slot[i] and adds
 * new_len[i] >= 0 (new_len NULL: one each).  With pages of 64 positions:
 *   cu_rows[0] = 0, cu_rows[i+1] = cu_rows[i] + new_len[i]              (n_seqs + 1 entries)
 *   row_slot[r] = seq_slot[i], row_pos[r] = kv_len[i] + r - cu_rows[i]  (cu_rows[i] <= r < cu_rows[i+1])
 *   kv_len_out[i] = kv_len[i] + new_len[i]
 *   the pages that request i lacks are popped off the free stack free_pages[0 .. *free_count),
 *   the topmost first, in request order, into page_table[seq_slot[i]][...];
 *   *free_count_out = *free_count - pages popped.
 * row_slot / row_pos hold rows_cap entries; those behind the last row are left as they were.
 * kv_len_out may be kv_len and free_count_out may be free_count (a step replayed in a graph then
 * advances its own state); no other arrays may overlap.
 * All or nothing: status (two int32 on the device) is {0, 0}, or {code, where} with
 *   code QASR_ERR_INVALID_ARG: where = the first request whose slot is outside [0, max_slots) or
 *     is listed before, whose kv_len is outside [0, max_pages * 64] or whose new_len is negative;
 *     where = -3: *free_count outside [0, pool_pages];
 *   code QASR_ERR_CAPACITY: where = the first request that does not fit max_pages * 64
 *     positions; -1: the free stack is too short; -2: more rows than rows_cap.
 * (Invalid arguments come before capacity, the requests before -1, -1 before -2.)
 * Then every cu_rows entry is 0 (the step has no rows), kv_len_out = kv_len, free_count_out =
 * free_count and nothing else is written: the row maps then still hold an earlier step's rows, as their
 * entries behind the last row always do, so what writes through them has to stop at
 * cu_rows[n_seqs] rows (qasr_kernel_kv_append_planned does; qasr_kernel_kv_append writes the `rows`
 * that it is told).  The page ids on the stack are taken as given.
 * n_seqs <= QASR_KV_PLAN_MAX_SEQS, max_slots <= QASR_KV_PLAN_MAX_SLOTS, max_pages < 2^25. */
qasr_status qasr_kernel_kv_plan(int device, void* stream, const int* seq_slot, const int* kv_len,
                                const int* new_len, int n_seqs, int max_slots, int* page_table,
                                int max_pages, const int* free_pages, int pool_pages,
                                const int* free_count, int* kv_len_out, int* free_count_out,
                                int* cu_rows, int* row_slot, int* row_pos, int rows_cap, int* status,
                                char* err, int errlen);

/* Give the pages of finished requests back: free_pages[*free_count + ...] receives, in request
 * order, the ceil(kv_len[i] / 64) pages of page_table[seq_slot[i]] in table order; kv_len_out[i] =
 * 0, *free_count_out = *free_count + the pages pushed.  The table keeps its entries.  The same
 * aliasing, limits and status as qasr_kernel_kv_plan; {QASR_ERR_CAPACITY, -1} when the stack
 * would hold more than pool_pages entries. */
qasr_status qasr_kernel_kv_release(int device, void* stream, const int* seq_slot, const int* kv_len,
                                   int n_seqs, int max_slots, const int* page_table, int max_pages,
                                   int* free_pages, int pool_pages, const int* free_count,
                                   int* kv_len_out, int* free_count_out, int* status, char* err,
                                   int errlen);

/* Append the new K and V rows of a planned step ([rows_cap, nkv * 128] each, f16 or bf16) to layer `layer` of the
 * cache: row r goes to (row_slot[r], row_pos[r]) as in qasr_kernel_kv_append, for 0 <= r < min(*row_count,
 * rows_cap).  row_count is a device int, cu_rows + n_seqs of the plan: rows that the plan did not give out
 * (all of them after a refused one) are neither read nor written, whatever the maps hold there.  A row whose
 * slot, position or page lies outside [0, max_slots), [0, max_pages * 64), [0, pool_pages) is left out.
 * k, v and kv_pool on 16-byte boundaries; kv_pool and page_table as in qasr_kernel_attention_chunk. */
qasr_status qasr_kernel_kv_append_planned(int device, void* stream, const uint16_t* k, const uint16_t* v,
                                          uint16_t* kv_pool, int pool_pages, const int* page_table,
                                          int max_slots, int max_pages, int layers, int nkv, int layer,
                                          const int* row_slot, const int* row_pos, int rows_cap,
                                          const int* row_count, char* err, int errlen);

/* GQA attention of chunks of new tokens over the paged cache.  Request i has the query rows
 * cu_rows[i] .. cu_rows[i+1]-1 and kv_len[i] cached positions, its new ones among them (what
 * qasr_kernel_kv_plan writes: cu_rows and kv_len_out); its j-th of n rows stands at position
 * p = kv_len[i] - n + j and attends the positions 0..p of slot seq_slot[i]:
 *   out[r, h] = sum_{t<=p} softmax_t(scale * q[r, h] . k_t) v_t,   kv head = h / (nq / nkv)
 * A row at p < 0 sees nothing and is written as zeros; rows that no request owns are left as they
 * were.  Chunks of any length go into one call: a decode step is n = 1 everywhere.
 * type: QASR_TYPE_F16 or QASR_TYPE_BF16, of q, out and the cache.  q [rows, q_ld], out [rows,
 * out_ld], |scale| < 2^127: q_ld, out_ld >= nq * 128 and multiples of 8, both pointers and kv_pool on 16-byte
 * boundaries; out may not overlap q.  nq a multiple of nkv, nq / nkv <= 16.  kv_pool
 * [pool_pages][layers][2][nkv][64][128] in the layout of qasr_kernel_attention; at most 2^31 - 1
 * rows of 128.  page_table [max_slots][max_pages], max_pages < 2^25.
 * What lies behind a request's last position in its last page is never used, whatever it holds,
 * and neither do values at later positions reach earlier rows.  Device arrays outside their
 * ranges cannot lead out of the buffers: cu_rows is cut to [0, rows], kv_len to max_pages * 64, a
 * slot outside [0, max_slots) counts as an empty cache and a page outside [0, pool_pages) as zeros.
 * Scores, softmax sums and outputs are held in f32; probabilities are rounded to `type` for the
 * product with V.  The keys are cut over the GPU as the whole call's lengths allow, so the last
 * bits of a row depend on the other rows of the call; the same call gives the same bits.
 * ws: qasr_kernel_attention_chunk_workspace(device) bytes on a 256-byte boundary, of any content;
 * calls that may overlap on the GPU (streams, captured graphs) need one each. */
int64_t qasr_kernel_attention_chunk_workspace(int device);
qasr_status qasr_kernel_attention_chunk(int device, void* stream, int type, const void* q, int q_ld,
                                        void* out, int out_ld, int rows, const void* kv_pool,
                                        int pool_pages, const int* page_table, int max_slots,
                                        int max_pages, int layers, int nq, int nkv, int layer,
                                        const int* seq_slot, const int* cu_rows, const int* kv_len,
                                        int n_seqs, float scale, void* ws, int64_t ws_bytes, char* err,
                                        int errlen);
/* Waits for `stream`; QASR_ERR_DEVICE_TIMEOUT if a bounded device-side wait of any qasr_kernel_attention_chunk over `ws`
 * gave up since this was last asked (the outputs of such a call are not to be used).  Calls leave a mark in ws
 * that later calls keep and this one clears, so once after all layers, or after several steps, is enough. */
qasr_status qasr_kernel_attention_chunk_check(int device, void* stream, void* ws, char* err, int errlen);

#define QASR_W4_MAX_ROWS 64

/* 4-bit weights with group scales: W[m, c] = scale[m, c / group] * (code[m, c] - zero), group 32, 64
 * or 128 along k, zero = zero[m, c / group] (0..15) or 8 without zero points.
 * qasr_kernel_pack_w4 lays the row-major codes (uint8 [n_out, k / 2], even c in the low four
 * bits), scales (f16 [n_out, k / group]) and zero points (uint8 [n_out, k / group] or NULL) out once
 * into `packed` (qasr_kernel_w4_packed_bytes bytes, 16-byte aligned), in the order in which the
 * product streams them.  n_out >= 1 of any size, k a multiple of group.
 * qasr_kernel_w4_packed_bytes returns -1 for sizes that are refused. */
int64_t qasr_kernel_w4_packed_bytes(int n_out, int k, int group, int has_zero);
qasr_status qasr_kernel_pack_w4(int device, void* stream, const uint8_t* codes, const uint16_t* scale,
                                const uint8_t* zero, int n_out, int k, int group, void* packed,
                                char* err, int errlen);

/* out[r, m] = type(sum_c W[m, c] x[r, c])                          (accumulate == 0)
 * out[r, m] = type(f32(out[r, m]) + sum_c W[m, c] x[r, c])         (accumulate != 0)
 * for 1 <= rows <= QASR_W4_MAX_ROWS; x [rows, ldx], out [rows, ldo] of `type`, ldx >= k a multiple
 * of 8, ldo >= n_out, x on a 16-byte boundary; out may overlap neither x nor packed.  Codes and zero
 * points enter the product exactly, each group's sum and the sum over groups are f32.
 * Only enqueues.  If a bounded device-side wait for its own copies gives up, the outputs whose sums lack a
 * part are NaN, and qasr_kernel_gemv_w4_check tells. */
qasr_status qasr_kernel_gemv_w4(int device, void* stream, int type, const void* packed, int has_zero,
                                int n_out, int k, int group, const void* x, int ldx, int rows, void* out,
                                int ldo, int accumulate, char* err, int errlen);
/* Waits for `stream`; QASR_ERR_DEVICE_TIMEOUT if a wait of any qasr_kernel_gemv_w4 on `device` gave up since
 * this was last asked (one word per device, whatever the stream: only the first to ask is told). */
qasr_status qasr_kernel_gemv_w4_check(int device, void* stream, char* err, int errlen);

/* Number of kernels this library launched since load (all contexts and probes). */
uint64_t qasr_kernel_launch_count(void);

#ifdef __cplusplus
}
#endif
#endif /* QASR_B200_KERNELS_H */
