// Single-query paged attention over the 8-bit cache: the bandwidth-bound "suffix" stage of single_query.cuh with half the
// bytes per token.
//
// For the tokens t of a block with scales (ks, vs), codes k8, v8 and a query row q:
//     s_t = c * ks * (q . k8_t),  c = scale * log2(e)          p_t = 2^(s_t - m),  l = sum p_t
//     O   = sum w_t v8_t,         w_t = 2^(s_t + log2(vs) - M)
// The value's scale enters as an offset of the exponent, with a reference M of its own: M follows max(s + log2 vs), so the
// largest weight of a row is near 2^7 whatever the scales of its blocks are, and a block with vs = 0 adds to l alone. The
// partial that goes to the merge is (m, l, O * 2^(M - m)), as from every other kernel.
//
// Both contractions are mma.sync.m16n8k16 in fp16 with fp32 accumulation: e4m3 values are exact in fp16, so K and V are
// converted without rounding whatever the queries' type is. Query rows are multiplied by the power of two that puts their
// largest element into [2^13, 2^14) (undone in c): fp16 and bf16 are then exact too (down to 2^-38 of the row's largest
// element), fp32 goes in as a sum of two fp16 values, whose products share the instruction (rows g and g + 8 of A). w
// enters as hi + lo fp16 values: with one head per item both ride in one instruction as columns of B (column 0 hi, column 1 lo);
// with several heads the columns are the heads, and lo takes an instruction of its own, which only fp32 queries get: the
// rounding of w alone is at most 2^-11 relative, that of a 16-bit output itself.
// (mma.sync on the codes themselves is no way out: this GPU has no such instruction outside tcgen05, and its emulation
// converts both operands in every call: 860 instructions for a (block, head) of 2 x 2 KiB, against about 400.)
// This kernel serves fp32 queries, blocks of 32 and head sizes 80, 112 and 256; the others go to decode_fp8_tc.cu. It is bound by the
// issue of its instructions: 256 sequences of 1024 tokens x 32 heads, 16-bit queries, 523 us or 4.1 TB/s; fp32, 57 sequences of up
// to 1777 tokens, 12 heads of 80, blocks of 32: 37 us or 2.6 TB/s.
//
// Fragments come from the tiles as they lie in the cache: a 32-bit register of ldmatrix holds four codes of one row,
// (4t .. 4t+3) of 16, which become two fp16 pairs (the contraction index is permuted alike in both
// operands). The rows that ldmatrix is given for K are ordered so that lane t of a quad ends with the logits of tokens
// 4t .. 4t+3: exactly those whose V codes it holds.
//
// Work items, queue and copies are those of single_query.cuh: every warp streams (row, heads of one kv head, chunk of
// blocks) items through a ring of NS stages filled by bulk copies; the scales of the blocks are read by the helper warp
// with the block ids.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "fp8.cuh"

namespace pb {
namespace {

constexpr int kMaxItemHeads = 8;  // query heads of one kv head in an item: the N of the MMA

template <typename T, int D, int B, bool MULTI>
struct Sq8Cfg {
  static constexpr int kTileBytes = D * B;
  static constexpr int kQBytes = D * (int)sizeof(T);
  static constexpr int kQRows = MULTI ? kMaxItemHeads : 1;
  static constexpr int kStageBytes = (2 * kTileBytes + kQRows * kQBytes + 127) / 128 * 128;
  static constexpr int warp_bytes(int ns) { return (ns * (kStageBytes + 16 /*meta*/ + 8 /*scales*/ + 8 /*bar*/) + 127) / 128 * 128; }
};

struct Item8 {
  int row, head, kvh, part, nblk, ntok;
  const int32_t* tbl;
};

constexpr int kQueue8 = 8;   // entries
constexpr int kBatch8 = 4;   // items claimed with one atomic
struct Entry8 {
  int row, head, kvh, part, nblk, ntok, table_kind, tbl_off;
  int ids[32];    // the first 32 block ids of the chunk, with their scales
  float ks[32], vs[32];
};
struct Queue8 {
  Entry8 e[kQueue8];
  int free_at[kQueue8];
  int tail, head, final;
};
__device__ __forceinline__ int ld_shared_now(const int* p) { return *reinterpret_cast<const volatile int*>(p); }

__device__ __forceinline__ void mma_f16_16816(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm_x4(uint32_t* r, uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ uint32_t pack_half2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// (hi, lo) split of two floats: hi = rounded pair, lo = rounded remainders
__device__ __forceinline__ void split_half2(float x, float y, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 hf = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack_half2(x - hf.x, y - hf.y);
}
// Four consecutive elements of a query row in shared memory.
template <typename T> __device__ __forceinline__ void load_q4(const T* p, float* f);
template <> __device__ __forceinline__ void load_q4<float>(const float* p, float* f) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  f[0] = v.x; f[1] = v.y; f[2] = v.z; f[3] = v.w;
}
template <> __device__ __forceinline__ void load_q4<__half>(const __half* p, float* f) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&v.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&v.y));
  f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
}
template <> __device__ __forceinline__ void load_q4<__nv_bfloat16>(const __nv_bfloat16* p, float* f) {
  const uint2 v = *reinterpret_cast<const uint2*>(p);
  f[0] = __uint_as_float(v.x << 16); f[1] = __uint_as_float(v.x & 0xffff0000u);
  f[2] = __uint_as_float(v.y << 16); f[3] = __uint_as_float(v.y & 0xffff0000u);
}

__device__ __forceinline__ const int32_t* table_of(const AttnDev& d, int kind) {
  return kind == 1 ? d.group_tables : kind == 2 ? d.seg_tables : kind == 3 ? d.outer_tables : d.suffix_tables;
}
// The kv head of a query head. A mapping that leaves the cache is recorded and replaced.
__device__ __forceinline__ int kv_head_of(const AttnDev& d, int head) {
  if (!d.head_mapping) return head;
  const int kvh = d.head_mapping[head];
  if (kvh >= 0 && kvh < d.num_kv_heads) return kvh;
  atomicMax(&d.hdr[kHdrStatus], kStatusBadIndex);
  return 0;
}
// Scales of block `blk` (0, 0 for an id outside the cache: the producer replaces and records it).
__device__ __forceinline__ void load_scales(const AttnDev& d, int blk, int kvh, float& ks, float& vs) {
  ks = vs = 0.f;
  if (blk >= 0 && blk < d.num_blocks) {
    const size_t at = (size_t)blk * d.scale_block_stride + (size_t)kvh * d.scale_head_stride;
    ks = d.key_scale[at];
    vs = d.value_scale[at];
  }
}

template <typename T, int D, int B, int WARPS, int NS, bool MULTI>
__global__ void __launch_bounds__((WARPS + 1) * 32, 1) sq8_attn_kernel(const AttnDev d) {
  using C = Sq8Cfg<T, D, B, MULTI>;
  constexpr bool kTwoParts = sizeof(T) == 4;  // fp32: q and w as hi + lo
  constexpr int kQParts = kTwoParts ? 4 : 2;  // registers of q for each 16 elements
  // w is largest at 2^kTop; the reference M is moved when that would pass 2^(kTop + kLag)
  constexpr float kTop = 7.f, kLag = 8.f;
  extern __shared__ __align__(128) uint8_t smem_raw[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kWarpBytes = C::warp_bytes(NS);
  Queue8* wq = reinterpret_cast<Queue8*>(smem_raw + WARPS * kWarpBytes);
  uint8_t* wbase = smem_raw + (warp < WARPS ? warp : 0) * kWarpBytes;
  int4* meta = reinterpret_cast<int4*>(wbase + NS * C::kStageBytes);
  float2* scales = reinterpret_cast<float2*>(wbase + NS * (C::kStageBytes + 16));
  uint64_t* bars = reinterpret_cast<uint64_t*>(wbase + NS * (C::kStageBytes + 16 + 8));

  if (lane == 0 && warp < WARPS) {
#pragma unroll
    for (int s = 0; s < NS; ++s) mbar_init(smem_u32(&bars[s]), 1);
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (threadIdx.x == 0) { wq->tail = 0; wq->head = 0; wq->final = -1; }
  if (threadIdx.x < kQueue8) wq->free_at[threadIdx.x] = threadIdx.x;
  __syncthreads();

  // with a dense kernel in front of it this kernel starts beside it and waits for it at the very end (single_query.cuh)
  if (d.sq_waits_at_start) pdl_wait();
  pdl_trigger();
  // Query heads per item: several only under the usual mapping (head h reads kv head h / (heads / kv heads)), which is
  // device memory and looked at in every call.
  int hpi = 1;
  if constexpr (MULTI) {
    const int share = d.num_heads / d.num_kv_heads;
    bool usual = true;
    for (int h = threadIdx.x; h < d.num_heads; h += (WARPS + 1) * 32) usual = usual && d.head_mapping[h] == h / share;
    if (__syncthreads_and(usual)) hpi = d.gqa_heads;
  }
  const int H = d.num_heads / hpi;  // items per list entry
  const long long n_items = (long long)d.hdr[kHdrNumSq] * H;
  if (warp == WARPS) {
    // ---------------- helper warp: claims items, reads their descriptors, block ids and scales ----------------
    int tail = 0;
    int want = kBatch8;
    bool ok = true;
    while (ok) {
      for (uint32_t spin = 0;; ++spin) {
        bool mine = lane >= want || ld_shared_now(&wq->free_at[(tail + lane) % kQueue8]) == tail + lane;
        if (want < kBatch8) mine = mine && (tail - ld_shared_now(&wq->head) <= 2);
        if (__all_sync(0xffffffffu, mine)) break;
        __nanosleep(64);
        if (spin > (1u << 24)) { ok = false; break; }  // about a second: the consumers are gone
      }
      if (!ok) break;
      int v = 0;
      if (lane == 0) v = atomicAdd(&d.hdr[kHdrSqCounter], want);
      const long long base = (long long)__shfl_sync(0xffffffffu, v, 0) + (long long)gridDim.x * WARPS;
      if (base >= n_items) break;
      const int cnt = (int)min((long long)want, n_items - base);
      if (n_items - (base + cnt) < (long long)gridDim.x * kBatch8) want = kBatch8 / 2;
      int4 a = make_int4(0, 0, 0, 0), b = make_int4(0, 0, 0, 0);
      int head = 0;
      if (lane < cnt) {
        const long long id = base + lane;
        const int sc = (int)(id / H);
        head = (int)(id - (long long)sc * H) * hpi;
        a = *reinterpret_cast<const int4*>(&d.sq_items[sc]);        // row, meta, ntok, part
        b = *(reinterpret_cast<const int4*>(&d.sq_items[sc]) + 1);  // bid[4]
      }
      const int kvh = kv_head_of(d, head);
      int ids[kBatch8];
      float ks[kBatch8], vs[kBatch8];
#pragma unroll
      for (int e = 0; e < kBatch8; ++e) {  // independent loads, all in flight together
        const int m = __shfl_sync(0xffffffffu, a.y, e);
        const int bx = __shfl_sync(0xffffffffu, b.x, e), by = __shfl_sync(0xffffffffu, b.y, e);
        const int bz = __shfl_sync(0xffffffffu, b.z, e), bw = __shfl_sync(0xffffffffu, b.w, e);
        ids[e] = -1;
        if (e < cnt && lane < (m & 0xffff)) {
          if (m & (1 << 17)) ids[e] = (lane == 0) ? bx : (lane == 1) ? by : (lane == 2) ? bz : bw;
          else ids[e] = table_of(d, (m >> 18) & 3)[bx + lane];
        }
      }
#pragma unroll
      for (int e = 0; e < kBatch8; ++e) load_scales(d, ids[e], __shfl_sync(0xffffffffu, kvh, e), ks[e], vs[e]);
#pragma unroll
      for (int e = 0; e < kBatch8; ++e)
        if (e < cnt) {
          Entry8& q = wq->e[(tail + e) % kQueue8];
          q.ids[lane] = ids[e]; q.ks[lane] = ks[e]; q.vs[lane] = vs[e];
        }
      if (lane < cnt) {
        Entry8& q = wq->e[(tail + lane) % kQueue8];
        q.row = a.x; q.head = head; q.kvh = kvh; q.part = a.w; q.nblk = a.y & 0xffff; q.ntok = a.z;
        q.table_kind = (a.y & (1 << 17)) ? -1 : ((a.y >> 18) & 3);
        q.tbl_off = b.x;
      }
      __threadfence_block();  // the slots were seen free (acquire) and are now complete (release)
      __syncwarp();
      tail += cnt;
      if (lane == 0) *reinterpret_cast<volatile int*>(&wq->tail) = tail;
      if (base + cnt >= n_items) break;
    }
    __threadfence_block();
    if (lane == 0) *reinterpret_cast<volatile int*>(&wq->final) = tail;
  } else {
    // ------------------------------ streaming warps ------------------------------
    bool failed = false;
    auto pop = [&](int& bid, float& ks, float& vs) -> Item8 {
      Item8 it = {0, 0, 0, 0, 0, 0, nullptr};
      bid = 0;
      int idx = 0;
      if (lane == 0) idx = atomicAdd(&wq->head, 1);
      idx = __shfl_sync(0xffffffffu, idx, 0);
      for (uint32_t spin = 0;; ++spin) {
        if (ld_shared_now(&wq->tail) > idx) break;
        const int fin = ld_shared_now(&wq->final);
        if (fin >= 0 && idx >= fin) return it;
        __nanosleep(32);
        if (spin > (1u << 25)) {  // about a second without a publisher
          if (lane == 0) atomicMax(&d.hdr[kHdrStatus], kStatusWaitExpired);
          failed = true;
          return it;
        }
      }
      __threadfence_block();
      const Entry8& q = wq->e[idx % kQueue8];
      it.row = q.row; it.head = q.head; it.kvh = q.kvh; it.part = q.part; it.nblk = q.nblk; it.ntok = q.ntok;
      if (q.table_kind >= 0) it.tbl = table_of(d, q.table_kind) + q.tbl_off;
      bid = q.ids[lane]; ks = q.ks[lane]; vs = q.vs[lane];
      __syncwarp();
      if (lane == 0) {
        __threadfence_block();
        *reinterpret_cast<volatile int*>(&wq->free_at[idx % kQueue8]) = idx + kQueue8;
      }
      return it;
    };

    // the first item of every warp of the grid is fixed: item (CTA, warp) of the list
    int cur_bid = 0;
    float cur_ks = 0.f, cur_vs = 0.f;
    Item8 cur;
    {
      const long long id0 = (long long)blockIdx.x * WARPS + warp;
      if (id0 < n_items) {
        const int sc = (int)(id0 / H);
        const int head = (int)(id0 - (long long)sc * H) * hpi;
        const int4 a = *reinterpret_cast<const int4*>(&d.sq_items[sc]);        // row, meta, ntok, part
        const int4 b = *(reinterpret_cast<const int4*>(&d.sq_items[sc]) + 1);  // bid[4]
        cur.row = a.x; cur.head = head; cur.kvh = kv_head_of(d, head);
        cur.part = a.w; cur.nblk = a.y & 0xffff; cur.ntok = a.z;
        cur.tbl = nullptr;
        if (a.y & (1 << 17)) {
          cur_bid = (lane == 0) ? b.x : (lane == 1) ? b.y : (lane == 2) ? b.z : b.w;
        } else {
          cur.tbl = table_of(d, (a.y >> 18) & 3) + b.x;
          cur_bid = (lane < cur.nblk) ? cur.tbl[lane] : -1;
        }
        if (lane >= cur.nblk) cur_bid = -1;
        load_scales(d, cur_bid, cur.kvh, cur_ks, cur_vs);
      } else {
        cur = pop(cur_bid, cur_ks, cur_vs);
      }
    }
    int p_blk = 0;
    uint32_t issued = 0, consumed = 0;
    const uint64_t kv_policy = l2_policy_evict_first();
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(d.key_cache);
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(d.value_cache);
    const uint8_t* qg = reinterpret_cast<const uint8_t*>(d.query);

    // consumer state. Lane (g, t): row g of S (a query head, or with one head part g of w), columns 2t, 2t + 1 of O.
    constexpr int kSteps = D / 16;  // 16-code chunks of a K row = 16-row tiles of V
    const int g = lane >> 2, t = lane & 3;
    uint32_t qa[kSteps][kQParts];
    float oacc[kSteps][4];
    float m_run = -INFINITY, l_run = 0.f, ref = -INFINITY, mul = 0.f;  // m, l, M, c / (power of two of the row)
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f;
#pragma unroll
      for (int i = 0; i < kQParts; ++i) qa[j][i] = 0u;
    }
    // ldmatrix rows. K: matrix m = lane / 8 is (chunk m / 2, n-tile m % 2), its row i token 4 (i / 2) + i % 2 + 2 (m % 2).
    // V: matrix m is rows 8m .. 8m + 7 of 32 rows of the tile.
    const int mi = lane & 7;
    const uint32_t ldm_k = (uint32_t)(((lane >> 4) * B + 4 * (mi >> 1) + (mi & 1) + 2 * ((lane >> 3) & 1)) * 16);
    const uint32_t ldm_v = (uint32_t)(lane * B);

    while (true) {
      // ------------------------------ producer ------------------------------
      while (issued - consumed < (uint32_t)NS && cur.nblk > 0) {
        const int s = issued % NS;
        if (p_blk > 0 && (p_blk & 31) == 0) {  // chunks longer than 32 blocks: next window of ids
          cur_bid = (p_blk + lane < cur.nblk) ? cur.tbl[p_blk + lane] : -1;
          load_scales(d, cur_bid, cur.kvh, cur_ks, cur_vs);
        }
        int blk = __shfl_sync(0xffffffffu, cur_bid, p_blk & 31);
        const float ks = __shfl_sync(0xffffffffu, cur_ks, p_blk & 31), vs = __shfl_sync(0xffffffffu, cur_vs, p_blk & 31);
        if (blk < 0 || blk >= d.num_blocks) {
          if (lane == 0) atomicMax(&d.hdr[kHdrStatus], kStatusBadIndex);
          blk = 0;
        }
        if (lane == 0) {
          const bool first = (p_blk == 0), last = (p_blk == cur.nblk - 1);
          meta[s] = make_int4(cur.row, cur.head | (cur.part << 16), 0,
                              min(B, cur.ntok - p_blk * B) | (first ? 256 : 0) | (last ? 512 : 0));
          scales[s] = make_float2(ks, vs);
          const uint32_t bar = smem_u32(&bars[s]);
          const uint32_t dst = smem_u32(wbase + s * C::kStageBytes);
          const size_t off = (size_t)blk * d.kv_block_stride + (size_t)cur.kvh * d.kv_head_stride;
          mbar_arrive_expect_tx(bar, 2 * C::kTileBytes + (first ? hpi * C::kQBytes : 0));
          bulk_g2s_hint(dst, kc + off, C::kTileBytes, bar, kv_policy);
          bulk_g2s_hint(dst + C::kTileBytes, vc + off, C::kTileBytes, bar, kv_policy);
          if (first)
            bulk_g2s(dst + 2 * C::kTileBytes, qg + ((size_t)cur.row * d.q_stride + (size_t)cur.head * D) * sizeof(T),
                     hpi * C::kQBytes, bar);
        }
        ++issued;
        ++p_blk;
        if (p_blk == cur.nblk) {
          cur = pop(cur_bid, cur_ks, cur_vs);
          p_blk = 0;
        }
      }
      if (consumed == issued) break;
      __syncwarp();

      // ------------------------------ consumer ------------------------------
      const int s = consumed % NS;
      if (!mbar_wait_bounded(smem_u32(&bars[s]), (consumed / NS) & 1)) {
        if (lane == 0) atomicMax(&d.hdr[kHdrStatus], kStatusWaitExpired);
        failed = true;
        break;
      }
      const int4 mt = meta[s];
      const float2 sc = scales[s];
      const int ntok_blk = mt.w & 255;
      const uint8_t* stage = wbase + s * C::kStageBytes;
      const uint32_t st = smem_u32(stage);
      if (mt.w & 256) {  // first block of an item: q as A fragments, fresh accumulators
        // one head: rows 0 and 1 both hold it, for the two parts of w; else row g is head g of the item
        const int qrow = MULTI ? g : 0;
        const bool live = MULTI ? g < hpi : g < 2;
        const T* qs = reinterpret_cast<const T*>(stage + 2 * C::kTileBytes) + (live ? qrow : 0) * D + 4 * t;
        float top = 0.f, odd = 0.f;  // odd: NaN if the row holds NaN or an infinity, whose products could all be -inf
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          float f[4];
          load_q4<T>(qs + c * 16, f);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            top = fmaxf(top, fabsf(f[i]));
            odd = fmaf(f[i], 0.f, odd);
          }
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        odd += __shfl_xor_sync(0xffffffffu, odd, 1);
        odd += __shfl_xor_sync(0xffffffffu, odd, 2);
        const int e = min(max((int)(__float_as_uint(top) >> 23), 20), 254);
        const float up = __uint_as_float((uint32_t)(267 - e) << 23);
        mul = d.scale_log2e * __uint_as_float((uint32_t)(e - 13) << 23) + odd;
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
          float f[4];
          load_q4<T>(qs + c * 16, f);
#pragma unroll
          for (int i = 0; i < 4; ++i) f[i] = live ? f[i] * up : 0.f;
          if constexpr (kTwoParts) {
            split_half2(f[0], f[1], qa[c][0], qa[c][2]);
            split_half2(f[2], f[3], qa[c][1], qa[c][3]);
          } else {
            qa[c][0] = pack_half2(f[0], f[1]);
            qa[c][1] = pack_half2(f[2], f[3]);
          }
        }
        m_run = -INFINITY;
        l_run = 0.f;
        ref = -INFINITY;
#pragma unroll
        for (int j = 0; j < kSteps; ++j) oacc[j][0] = oacc[j][1] = oacc[j][2] = oacc[j][3] = 0.f;
      }
      const float cs = sc.x * mul, lv = __log2f(sc.y);

#pragma unroll
      for (int sub = 0; sub < B / 16; ++sub) {
        const int left = ntok_blk - 16 * sub;  // tokens of this half of the block and behind it
        if (sub > 0 && left <= 0) break;
        float sa[4] = {0.f, 0.f, 0.f, 0.f}, sb[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < kSteps; c += 2) {
          uint32_t kb[4];
          // (an odd number of chunks: the last pair reads its second chunk again)
          const bool pair = c + 1 < kSteps;
          ldsm_x4(kb, st + (pair ? ldm_k : (ldm_k & (16u * B - 1u))) + c * (16 * B) + sub * 256);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (c + u < kSteps) {
              const uint32_t a[4] = {qa[c + u][0], kTwoParts ? qa[c + u][kQParts - 2] : 0u, qa[c + u][1], kTwoParts ? qa[c + u][kQParts - 1] : 0u};
              mma_f16_16816(sa, a, fp8::to_half2(kb[2 * u]), fp8::to_half2_high(kb[2 * u]));
              mma_f16_16816(sb, a, fp8::to_half2(kb[2 * u + 1]), fp8::to_half2_high(kb[2 * u + 1]));
            }
          }
        }
        float lg[4] = {sa[0], sa[1], sb[0], sb[1]};  // tokens 4t .. 4t + 3
        if constexpr (kTwoParts) { lg[0] += sa[2]; lg[1] += sa[3]; lg[2] += sb[2]; lg[3] += sb[3]; }
#pragma unroll
        for (int i = 0; i < 4; ++i) lg[i] = (4 * t + i < left) ? lg[i] * cs : -INFINITY;
        float bm = fmaxf(fmaxf(lg[0], lg[1]), fmaxf(lg[2], lg[3]));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
        const float m_new = fmaxf(m_run, bm);
        const float m_base = m_new == -INFINITY ? 0.f : m_new;  // (nothing but logits of -inf so far)
        l_run *= fast_exp2(m_run - m_base);
        m_run = m_new;
        const bool grow = bm + lv > ref + kLag;  // the reference of the weights moves on jumps of more than 2^kLag
        if (__any_sync(0xffffffffu, grow)) {
          const float alpha = grow ? fast_exp2(ref - (bm + lv)) : 1.f;
          if (grow) ref = bm + lv;
          const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * t), a1 = __shfl_sync(0xffffffffu, alpha, 8 * t + 4);
#pragma unroll
          for (int j = 0; j < kSteps; ++j) { oacc[j][0] *= a0; oacc[j][1] *= a1; oacc[j][2] *= a0; oacc[j][3] *= a1; }
        }
        float w[4];
        const float shift = lv - (ref == -INFINITY ? 0.f : ref) + kTop;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          l_run += fast_exp2(lg[i] - m_base);
          w[i] = fast_exp2(lg[i] + shift);
        }
        uint32_t hi0 = 0u, hi1 = 0u, lo0 = 0u, lo1 = 0u;
        if constexpr (MULTI && !kTwoParts) {
          hi0 = pack_half2(w[0], w[1]);
          hi1 = pack_half2(w[2], w[3]);
        } else {
          split_half2(w[0], w[1], hi0, lo0);
          split_half2(w[2], w[3], hi1, lo1);
          if constexpr (!MULTI) {  // column 0: hi, column 1: lo
            hi0 = g == 0 ? hi0 : g == 1 ? lo0 : 0u;
            hi1 = g == 0 ? hi1 : g == 1 ? lo1 : 0u;
          }
        }
        // codes of tokens beyond the context are not looked at: 0 * NaN would not be 0
        const int keep = left - 4 * t;
        const uint32_t mask = keep >= 4 ? 0xffffffffu : keep <= 0 ? 0u : (1u << (8 * keep)) - 1u;
#pragma unroll
        for (int j = 0; j < kSteps; j += 2) {
          uint32_t va[4];
          const bool pair = j + 1 < kSteps;
          ldsm_x4(va, st + C::kTileBytes + (pair ? ldm_v : (uint32_t)((lane & 15) * B)) + j * (16 * B) + sub * 16);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            if (j + u < kSteps) {
              const uint32_t r0 = va[2 * u] & mask, r1 = va[2 * u + 1] & mask;
              const uint32_t a[4] = {fp8::to_half2(r0), fp8::to_half2(r1), fp8::to_half2_high(r0), fp8::to_half2_high(r1)};
              mma_f16_16816(oacc[j + u], a, hi0, hi1);
              if constexpr (MULTI && kTwoParts) mma_f16_16816(oacc[j + u], a, lo0, lo1);
            }
          }
        }
      }
      __syncwarp();  // stage s may be overwritten from here on
      if (mt.w & 512) {  // last block of the item: the partial, re-based on the exact maximum
        const int it_row = mt.x, it_head = mt.y & 0xffff, it_part = mt.y >> 16;
        float l = l_run;
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        m_run = fp8::told_max(m_run, l);
        // 2^(ref - kTop - m), in two factors: by value scales near 2^-126 or 2^120 one would leave the range of fp32
        const float fix_e = ref == -INFINITY ? 0.f : fminf(fmaxf(rintf(0.5f * (ref - kTop - m_run)), -126.f), 126.f);
        const float fix = ref == -INFINITY ? 0.f : fast_exp2(ref - kTop - m_run - fix_e), fix2 = fp8::pow2(fix_e);
        if constexpr (MULTI) {
          const float f0 = __shfl_sync(0xffffffffu, fix, 8 * t), f1 = __shfl_sync(0xffffffffu, fix, 8 * t + 4);
          const float p0 = __shfl_sync(0xffffffffu, fix2, 8 * t), p1 = __shfl_sync(0xffffffffu, fix2, 8 * t + 4);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int hh = 2 * t + c;
            if (hh < hpi) {
              float* ap = d.acc + partial_slot(d, it_row, it_part, it_head + hh) * D + g;
              const float f = c ? f1 : f0, p = c ? p1 : p0;
#pragma unroll
              for (int j = 0; j < kSteps; ++j) {
                ap[16 * j] = oacc[j][c] * f * p;
                ap[16 * j + 8] = oacc[j][2 + c] * f * p;
              }
            }
          }
          if (t == 0 && g < hpi) d.ml[partial_slot(d, it_row, it_part, it_head + g)] = make_float2(m_run, l);
        } else {
          const size_t slot = partial_slot(d, it_row, it_part, it_head);
          const float f0 = __shfl_sync(0xffffffffu, fix, 0), p0 = __shfl_sync(0xffffffffu, fix2, 0);
          float* ap = d.acc + slot * D + g;
#pragma unroll
          for (int j = 0; j < kSteps; ++j) {
            const float lo = oacc[j][0] + oacc[j][1], hi = oacc[j][2] + oacc[j][3];
            if (t == 0) {
              ap[16 * j] = lo * f0 * p0;
              ap[16 * j + 8] = hi * f0 * p0;
            }
          }
          if (lane == 0) d.ml[slot] = make_float2(m_run, l);
        }
      }
      ++consumed;
    }
    if (failed) {
      // give the copies still in flight one more bounded chance to land before shared memory is released
      for (uint32_t c = consumed + 1; c < issued; ++c)
        (void)mbar_wait_bounded(smem_u32(&bars[c % NS]), (c / NS) & 1);
    }
  }  // streaming warps

  if (!d.sq_waits_at_start) pdl_wait();  // the dense prefix kernel has completed
}

// Streaming warps that fit shared memory with NS stages each, at most 11 (with the helper 384 threads of up to 168 registers).
constexpr int kMaxWarps8 = 11;
template <typename T, int D, int B, int NS, bool MULTI>
constexpr int sq8_warps() {
  const int w = (227 * 1024 - (int)sizeof(Queue8)) / Sq8Cfg<T, D, B, MULTI>::warp_bytes(NS);
  return w > kMaxWarps8 ? kMaxWarps8 : w;
}

template <typename T, int D, int B, bool MULTI>
cudaError_t launch_sq8(const AttnDev& d, cudaStream_t s) {
  constexpr int NS = 4;
  constexpr int WARPS = sq8_warps<T, D, B, NS, MULTI>();
  static_assert(WARPS >= 1, "one warp's stages must fit shared memory");
  constexpr int smem = WARPS * Sq8Cfg<T, D, B, MULTI>::warp_bytes(NS) + (int)sizeof(Queue8);
  auto kfn = sq8_attn_kernel<T, D, B, WARPS, NS, MULTI>;
  cudaError_t e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return launch_kernel(kfn, d.num_sms, (WARPS + 1) * 32, smem, s, true, d);
}

template <typename T, int D, int B>
cudaError_t launch_sq8_shape(const AttnDev& d, cudaStream_t s) {
  if constexpr (fp8::decode_on_tc(sizeof(T) == 2, D, B)) return cudaErrorInvalidValue;  // (never asked for here)
  else return d.gqa_heads > 1 ? launch_sq8<T, D, B, true>(d, s) : launch_sq8<T, D, B, false>(d, s);
}
// All head and block sizes of one type of queries that the tcgen05 kernel does not take.
template <typename T>
cudaError_t launch_sq8_all(const AttnDev& d, int head_size, int block_size, cudaStream_t s) {
#define PB_SQ8(DD) \
  if (head_size == DD) return block_size == 16 ? launch_sq8_shape<T, DD, 16>(d, s) : launch_sq8_shape<T, DD, 32>(d, s);
  PB_SQ8(64) PB_SQ8(80) PB_SQ8(96) PB_SQ8(112) PB_SQ8(128) PB_SQ8(256)
#undef PB_SQ8
  return cudaErrorInvalidValue;
}

}  // namespace
}  // namespace pb
