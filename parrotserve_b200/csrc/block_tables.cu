// Block tables, slots, positions and row lengths of an iteration, from the requests' lengths.
//
// With c, n the context and the new tokens of a request, B the block size, W its table's width:
//     have = ceil(c / B),  need = ceil((c + n) / B) - have   (0 if it would pass W: the request fails)
//     at   = head + exclusive scan of need over the requests; the request fails if need > 0 and at + need > free blocks
// Up to kFusedRequests requests one kernel does it all: every CTA scans the requests for itself (rows and blocks taken), then a warp
// per row writes what the row is given and a warp per request appends its new blocks to its table. More requests are scanned
// by a kernel of one CTA in front. Nothing a warp reads is written by another one: the blocks a request is about to get are
// read from the free list, those it has from its table. Bound by latency: lengths -> scan -> table entry -> store.
// (24 decodes, Python included: 32 us a call with two kernels, 22 with one and fewer tensors made; the kernel itself takes 4.)
//
// Reference counterpart: the host loops of init_iteration_state (parrot/engine/builtin/attn_func.py:461-599) and of the
// token pool (parrot/engine/context/block_context.py:43-84).
#include "common.cuh"

namespace pb {
namespace {

struct TablesDev {
  const int32_t* context_lens;
  const int32_t* new_lens;
  int32_t* block_tables;
  const int32_t* free_blocks;
  const int32_t* free_head;
  const int32_t* prefix_lens;
  long long* slot_mapping;
  long long* positions;
  int32_t* row_offsets;
  int32_t* kv_lens;
  int32_t* suffix_lens;
  int32_t* suffix_tables;
  int32_t* free_head_out;
  int32_t* num_failed;
  int32_t* taken;  // [requests] entry of free_blocks where the request's new blocks begin; -1: it failed
  long long table_stride, num_tokens;
  int requests, width, num_free, block_size, num_prefills;
};

constexpr int kScanThreads = 1024;

__device__ __forceinline__ int warp_inclusive(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}

__global__ void __launch_bounds__(kScanThreads) tables_scan_kernel(const TablesDev d) {
  __shared__ int sums[2][33];
  __shared__ int failed_total, head_end;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  pdl_trigger();
  if (tid == 0) { failed_total = 0; head_end = max(*d.free_head, 0); }
  const int head = max(*d.free_head, 0);
  __syncthreads();
  int row0 = 0, block0 = 0, failed = 0, end = head;
  for (int base = 0; base < d.requests; base += kScanThreads) {
    const int r = base + tid;
    const bool live = r < d.requests;
    const int c = live ? max(d.context_lens[r], 0) : 0, n = live ? max(d.new_lens[r], 0) : 0;
    const int have = (int)(((long long)c + d.block_size - 1) / d.block_size);
    const long long want = ((long long)c + n + d.block_size - 1) / d.block_size;
    const bool wide = want > d.width;
    const int need = wide ? 0 : (int)want - have;
    const int rows_in = warp_inclusive(n), blocks_in = warp_inclusive(need);
    if (lane == 31) { sums[0][warp] = rows_in; sums[1][warp] = blocks_in; }
    __syncthreads();
    if (warp < 2) {
      const int w = sums[warp][lane], in = warp_inclusive(w);
      sums[warp][lane] = in - w;
      if (lane == 31) sums[warp][32] = in;
    }
    __syncthreads();
    const int rows_before = row0 + sums[0][warp] + rows_in - n, blocks_before = block0 + sums[1][warp] + blocks_in - need;
    if (live) {
      const long long last = (long long)head + blocks_before + need;
      const bool fails = wide || (need > 0 && last > d.num_free);
      d.row_offsets[r] = rows_before;
      d.kv_lens[r] = fails ? c : c + n;
      d.taken[r] = fails ? -1 : head + blocks_before;
      if (fails) ++failed;
      else if (need > 0) end = (int)last;
      if (r == d.requests - 1) d.row_offsets[r + 1] = rows_before + n;
    }
    row0 += sums[0][32];
    block0 += sums[1][32];
    __syncthreads();
  }
  if (failed) atomicAdd(&failed_total, failed);
  if (end > head) atomicMax(&head_end, end);
  __syncthreads();
  if (tid == 0) {
    *d.num_failed = failed_total;
    *d.free_head_out = head_end;
    if (d.requests == 0) d.row_offsets[0] = 0;
  }
}

constexpr int kRowWarps = 8;

// Task t: a row of the call (t < num_tokens), or behind the rows a request that appends its new blocks. offsets, taken: of the scan.
__device__ __forceinline__ void row_task(const TablesDev& d, long long t, const int32_t* offsets, const int32_t* taken, int lane) {
  if (t >= d.num_tokens) {
    const long long q = t - d.num_tokens;
    const int c = max(d.context_lens[q], 0), n = max(d.new_lens[q], 0), at = taken[q];
    if (at < 0) return;
    const int have = (int)(((long long)c + d.block_size - 1) / d.block_size);
    const int want = (int)(((long long)c + n + d.block_size - 1) / d.block_size);
    for (int j = have + lane; j < want; j += 32) d.block_tables[(size_t)q * d.table_stride + j] = d.free_blocks[at + j - have];
    return;
  }
  int32_t* row_table = d.suffix_tables ? d.suffix_tables + (size_t)t * d.width : nullptr;
  const int total = offsets[d.requests];
  long long slot = -1, position = 0;
  int suffix = 0, listed = 0;
  if (t < total) {
    int lo = 0, hi = d.requests - 1;  // last request whose rows start at t or before (those without rows start where the next one does)
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (offsets[mid] <= t) lo = mid; else hi = mid - 1;
    }
    const int r = lo, i = (int)t - offsets[r];
    const int c = max(d.context_lens[r], 0);
    const int have = (int)(((long long)c + d.block_size - 1) / d.block_size), at = taken[r];
    const int32_t* table = d.block_tables + (size_t)r * d.table_stride;
    const int p = c + i;
    position = (long long)p + (d.prefix_lens ? d.prefix_lens[r] : 0);
    if (at >= 0) {
      auto block = [&](int j) { return j < have ? table[j] : d.free_blocks[at + j - have]; };
      slot = (long long)block(p / d.block_size) * d.block_size + p % d.block_size;
      if (r >= d.num_prefills) {
        suffix = p + 1;
        listed = (suffix + d.block_size - 1) / d.block_size;
        if (row_table)
          for (int j = lane; j < listed; j += 32) row_table[j] = block(j);
      }
    }
  }
  if (row_table)
    for (int j = listed + lane; j < d.width; j += 32) row_table[j] = 0;
  if (lane == 0) {
    d.slot_mapping[t] = slot;
    d.positions[t] = position;
    d.suffix_lens[t] = suffix;
  }
}

// (Neither kernel releases the next one early: it may be the planner, which reads lengths before it waits.)
__global__ void __launch_bounds__(kRowWarps * 32) tables_rows_kernel(const TablesDev d) {
  pdl_wait();
  const long long t = (long long)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  if (t < d.num_tokens + d.requests) row_task(d, t, d.row_offsets, d.taken, threadIdx.x & 31);
}

constexpr int kFusedRequests = 1024;
constexpr int kPerThread = kFusedRequests / (kRowWarps * 32);

__global__ void __launch_bounds__(kRowWarps * 32) tables_fused_kernel(const TablesDev d) {
  __shared__ int offsets[kFusedRequests + 1], taken[kFusedRequests], sums[2][kRowWarps], failed_total, head_end;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  pdl_wait();
  const int head = max(*d.free_head, 0);
  if (tid == 0) { failed_total = 0; head_end = head; }
  int n[kPerThread], need[kPerThread], rows_in = 0, blocks_in = 0;  // need < 0: the table row is too short
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int r = tid * kPerThread + k;
    const int c = r < d.requests ? max(d.context_lens[r], 0) : 0;
    n[k] = r < d.requests ? max(d.new_lens[r], 0) : 0;
    const long long have = ((long long)c + d.block_size - 1) / d.block_size, want = ((long long)c + n[k] + d.block_size - 1) / d.block_size;
    need[k] = want > d.width ? -1 : (int)(want - have);
    rows_in += n[k];
    blocks_in += max(need[k], 0);
  }
  const int rows_incl = warp_inclusive(rows_in), blocks_incl = warp_inclusive(blocks_in);
  if (lane == 31) { sums[0][warp] = rows_incl; sums[1][warp] = blocks_incl; }
  __syncthreads();
  int row = rows_incl - rows_in, block = blocks_incl - blocks_in;
  for (int w = 0; w < warp; ++w) { row += sums[0][w]; block += sums[1][w]; }
  int failed = 0, end = head;
#pragma unroll
  for (int k = 0; k < kPerThread; ++k) {
    const int r = tid * kPerThread + k;
    const long long last = (long long)head + block + max(need[k], 0);
    const bool fails = need[k] < 0 || (need[k] > 0 && last > d.num_free);
    if (r < d.requests) {
      offsets[r] = row;
      taken[r] = fails ? -1 : head + block;
      if (r == d.requests - 1) offsets[r + 1] = row + n[k];
      if (fails) ++failed;
      else if (need[k] > 0) end = (int)last;
      if (blockIdx.x == 0) {
        d.row_offsets[r] = row;
        d.kv_lens[r] = max(d.context_lens[r], 0) + (fails ? 0 : n[k]);
        if (r == d.requests - 1) d.row_offsets[r + 1] = row + n[k];
      }
    }
    row += n[k];
    block += max(need[k], 0);
  }
  if (d.requests == 0 && tid == 0) {
    offsets[0] = 0;
    if (blockIdx.x == 0) d.row_offsets[0] = 0;
  }
  if (blockIdx.x == 0) {
    if (failed) atomicAdd(&failed_total, failed);
    if (end > head) atomicMax(&head_end, end);
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    *d.num_failed = failed_total;
    *d.free_head_out = head_end;
  }
  for (long long t = (long long)blockIdx.x * kRowWarps + warp; t < d.num_tokens + d.requests; t += (long long)gridDim.x * kRowWarps)
    row_task(d, t, offsets, taken, lane);
}

}  // namespace
}  // namespace pb

extern "C" {

size_t pb_block_tables_workspace_bytes(int32_t num_requests) {
  return num_requests <= pb::kFusedRequests ? 0 : ((size_t)num_requests * sizeof(int32_t) + 255) / 256 * 256;
}

int pb_build_block_tables(const int32_t* context_lens, const int32_t* new_lens, int32_t num_requests, int32_t* block_tables,
                          int32_t table_width, int64_t table_stride, const int32_t* free_blocks, int32_t num_free,
                          const int32_t* free_head, const int32_t* prefix_lens, int32_t block_size, int32_t num_prefills,
                          int64_t num_tokens, int64_t* slot_mapping, int64_t* positions, int32_t* row_offsets,
                          int32_t* kv_lens, int32_t* suffix_lens, int32_t* suffix_tables, int32_t* free_head_out,
                          int32_t* num_failed, void* workspace, size_t workspace_bytes, void* stream) {
  if (num_requests < 0 || num_tokens < 0 || num_tokens > 0x7fffffff || num_free < 0 || table_width < 0 || num_prefills < 0 ||
      num_prefills > num_requests || block_size <= 0)
    return PB_ERR_INVALID_ARG;
  if (!free_head || !row_offsets || !free_head_out || !num_failed || (num_free > 0 && !free_blocks)) return PB_ERR_INVALID_ARG;
  if (num_requests > 0 && (!context_lens || !new_lens || !kv_lens || (table_width > 0 && !block_tables))) return PB_ERR_INVALID_ARG;
  if (num_tokens > 0 && (!slot_mapping || !positions || !suffix_lens)) return PB_ERR_INVALID_ARG;
  if (num_requests > 1 && table_stride < table_width) return PB_ERR_INVALID_ARG;
  const size_t need = pb_block_tables_workspace_bytes(num_requests);
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < need)) return PB_ERR_WORKSPACE;
  // Every CTA reads the inputs for itself while others write results: no result may lie on an input, nor on another result.
  const int64_t r = num_requests, t = num_tokens;
  const struct { const void* p; int64_t bytes; } spans[] = {
      // results, the workspace among them
      {block_tables, r > 0 && table_width > 0 ? 4 * ((r - 1) * table_stride + table_width) : 0}, {slot_mapping, 8 * t}, {positions, 8 * t},
      {row_offsets, 4 * (r + 1)}, {kv_lens, 4 * r}, {suffix_lens, 4 * t}, {suffix_tables, 4 * t * table_width}, {free_head_out, 4},
      {num_failed, 4}, {workspace, (int64_t)need},
      // inputs
      {context_lens, 4 * r}, {new_lens, 4 * r}, {free_blocks, 4 * (int64_t)num_free}, {free_head, 4}, {prefix_lens, 4 * r}};
  constexpr int kResults = 10, kSpans = sizeof(spans) / sizeof(spans[0]);
  for (int i = 0; i < kResults; ++i)
    for (int j = i + 1; j < kSpans; ++j) {
      const uintptr_t a = reinterpret_cast<uintptr_t>(spans[i].p), b = reinterpret_cast<uintptr_t>(spans[j].p);
      if (a && b && spans[i].bytes > 0 && spans[j].bytes > 0 && a < b + spans[j].bytes && b < a + spans[i].bytes) return PB_ERR_INVALID_ARG;
    }
  pb::TablesDev d;
  d.context_lens = context_lens; d.new_lens = new_lens; d.block_tables = block_tables; d.free_blocks = free_blocks;
  d.free_head = free_head; d.prefix_lens = prefix_lens;
  d.slot_mapping = reinterpret_cast<long long*>(slot_mapping); d.positions = reinterpret_cast<long long*>(positions);
  d.row_offsets = row_offsets; d.kv_lens = kv_lens; d.suffix_lens = suffix_lens; d.suffix_tables = suffix_tables;
  d.free_head_out = free_head_out; d.num_failed = num_failed; d.taken = static_cast<int32_t*>(workspace);
  d.table_stride = table_stride; d.num_tokens = num_tokens;
  d.requests = num_requests; d.width = table_width; d.num_free = num_free; d.block_size = block_size; d.num_prefills = num_prefills;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const int64_t warps = num_tokens + num_requests, ctas = (warps + pb::kRowWarps - 1) / pb::kRowWarps;
  cudaError_t e;
  if (num_requests <= pb::kFusedRequests) {
    const int64_t most = (int64_t)pb::sm_count() * 8;  // (a full chip: what follows is done by the same CTAs, without a scan of their own)
    e = pb::launch_kernel(pb::tables_fused_kernel, (unsigned)(ctas < 1 ? 1 : ctas < most ? ctas : most), pb::kRowWarps * 32, 0, s, true, d);
  } else {
    e = pb::launch_kernel(pb::tables_scan_kernel, 1, pb::kScanThreads, 0, s, true, d);
    if (e == cudaSuccess) e = pb::launch_kernel(pb::tables_rows_kernel, (unsigned)ctas, pb::kRowWarps * 32, 0, s, true, d);
  }
  if (e != cudaSuccess) {
    pb::set_cuda_error(e);
    return PB_ERR_LAUNCH;
  }
  return PB_OK;
}

}  // extern "C"
