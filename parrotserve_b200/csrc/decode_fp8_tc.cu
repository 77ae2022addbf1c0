// Single-query attention over the 8-bit cache on tcgen05: the suffix stage for 16-bit queries, block size 16 and head sizes
// 64, 96 and 128. The formulas are those of single_query_fp8.cuh; here the tensor cores take the codes as they are
// (kind::f8f6f4), so that no code passes through a register.
//
// A tile is 128 tokens (8 blocks) of a context. TRANSPOSED products, the cache always as the 128-row operand:
//     S [128 tokens x N] = K . Qp^T       A = K codes [token][d], B = parts of the item's query rows, N columns
//     O [128 d x N]     += V^T . Wp       A = V codes [d][token], B = parts of the weights of the tile's tokens
// so a token is a lane of tensor memory, and a softmax thread owns one token: it adds up the parts' columns, scales, and
// writes the weight's parts back. A part is an e4m3 value, the rounded remainder of those before it, times 16 more each:
//     x = x0 + x1 / 16 + x2 / 256 + x3 / 4096: off by 2^-16 of itself or by half a step of x3, 2^-22 (q is scaled by a
//     power of two to a largest element in [2^7, 2^8), the largest weight of a row lies in [2^8, 2^8.75))
// With up to HMAX heads of one kv head in an item, column (g * kParts + p) * kHeads + h holds part p of head h of the g-th kHeads.
// Operand layouts (no swizzle, K-major, 8 x 16-byte core matrices): V tiles are made of them as they lie in the cache, [d][16 tok];
// the 256-byte chunk rows of the K tiles are put side by side, [d chunk][block][16 tok], by per-thread 16-byte async copies.
//
// Why: through mma.sync a (block, head) of 2 x 2 KiB costs a warp 64 conversions and 24 instructions of the fp16 pipe, some
// 400 instructions in all, and 256 sequences of 1024 tokens x 32 heads ran at 4.1 TB/s, bound by their issue. Here four warps
// spend about 100 instructions each on eight of them: 315 us, 6.8 TB/s, memory is the bound. With several heads per item the bound is
// the chain of a tile through its CTA (Q.K^T, weights, P.V: 2 us with four heads, 3 with eight): 128 sequences of 1024 tokens, 32
// heads over 8, 59 us or 4.5 TB/s; one of 100000 tokens, 64 heads over 8, 65 us or 3.2 TB/s.
//
// Three CTAs an SM with one head per item, so that the copies of one run under the chain of another. With several, two, whose
// heads are shared by two groups of softmax warps: the step from S to the weights is what the chain spends its time on (64 heads
// over 8, 64 sequences of 2048 tokens 94 us with one group, 83 with two).
// Warps 0-3 (and 4-7) softmax and epilogue, behind them one warp claims items and lists their tiles, two copy K (one of them V
// too), one issues the MMAs and one makes the query operands. Every mbarrier wait is bounded; on expiry the CTA records a status,
// drains and returns.
#include <type_traits>

#include "common.cuh"
#include "dense_common.cuh"
#include "fp8.cuh"

namespace pb {
namespace {

using namespace dense;
using fp8::kMinLv;
using fp8::told_max;
using fp8::warp_max;

constexpr int kDescSlots = 8, kItemSlots = 4;  // (how far the lister runs ahead: it waits for three loads in a row per item)
constexpr int kParts = 4;                  // the MMA takes sixteen columns or none: four parts cost what three do
constexpr float kTop = 8.f, kLag = 0.75f;  // the largest weight of a row lies in [2^kTop, 2^(kTop + kLag)) < 448

struct DecDesc {  // a tile
  int32_t blk[8];
  float ks[8], lv[8];
  int32_t nb, ntok;              // blocks and tokens of the tile; nb == 0: no more tiles
  int32_t row, head, part, kvh;  // of its item
  int32_t first, last;
};
struct DecItem {
  int32_t row, head;  // row < 0: no more items
};

template <int D, int HMAX>
struct DecCfg {
  static constexpr int kN = HMAX > 4 ? 32 : 16;       // columns: kParts * HMAX, in sixteens
  static constexpr int kTile = D * 16;                // one K or V tile of a (block, head)
  static constexpr int kStage = 2 * 8 * kTile;        // K, then V
  static constexpr int kGroups = HMAX > 1 ? 2 : 1;    // softmax groups of four warps; each has all tokens and
  static constexpr int kHeads = HMAX / kGroups;       // so many of the heads
  static constexpr int kW0 = 4 * kGroups;             // the first warp behind them
  static constexpr int kThreads = 32 * (kW0 + 5);
  static constexpr int kCtas = HMAX > 1 ? 2 : 3;      // per SM
  static constexpr int kStages = (HMAX == 1 ? 2 : 3) * 128 / D;
  static constexpr int kQSlots = HMAX > 4 ? 1 : 2;    // query operands: of the item at work, and of the next if there is room
  static constexpr int kQ = kN * D, kW = kN * 128;    // operands of one item / one tile
  // rows of V beyond D (the MMA always has 128) are read from what lies behind the tile: kPad bytes behind the last stage
  static constexpr int kPad = (128 - D) * 16;
  static constexpr int kOffW = kStages * kStage + kPad, kOffQ = kOffW + 2 * kW, kOffCtl = kOffQ + kQSlots * kQ;
  static constexpr int kTmem = kN == 32 ? 128 : 64;   // S, S, O, O
};

struct DecCtl {
  DecDesc desc[kDescSlots];
  DecItem item[kItemSlots];
  float mul[2][8];               // per query operand slot and head: scale * log2(e) / (power of two of the row)
  float4 xmax[2][2][4];          // exchange between the softmax warps of a group: per head, the warps' numbers
  float4 left_max[2][2][4], left_sum[2][2][4];  // per group and item: what the warps leave for its epilogue
  float left_ref[2][2][4];
  int left_row[2][2], left_head[2][2], left_part[2][2];
  uint64_t full[8], empty[8];    // stages
  uint64_t desc_full[kDescSlots], desc_empty[kDescSlots], item_full[kItemSlots], item_empty[kItemSlots];
  uint64_t q_full[2], q_empty[2], s_full[2], p_full[2], pv_done[2], exchange[2];
  uint32_t tmem;
  int abort_flag;
};

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* v) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]) : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, const uint32_t* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};"
               ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// The kParts * N columns of parts of a group's N heads, in registers.
template <int N> __device__ __forceinline__ void ld_cols(uint32_t taddr, uint32_t* v) {
  if constexpr (N == 1) tmem_ld4(taddr, v);
  else if constexpr (N == 2) tmem_ld8(taddr, v);
  else tmem_ld16(taddr, v);
}
template <int N> __device__ __forceinline__ void st_cols(uint32_t taddr, const uint32_t* v) {
  if constexpr (N == 1) tmem_st4(taddr, v);
  else if constexpr (N == 2) tmem_st8(taddr, v);
  else tmem_st16(taddr, v);
}

// x -> its parts as codes (low bytes).
__device__ __forceinline__ void parts_of(float x, uint32_t (&p)[kParts]) {
#pragma unroll
  for (int i = 0; i < kParts; ++i) {
    p[i] = fp8::pack2(x, 0.f);
    if (i < kParts - 1) x = (x - fp8::to_float2(p[i]).x) * 16.f;
  }
}
// The same of two numbers (low and second bytes). What two parts leave, 2^-8 of x, needs no more than fp16.
__device__ __forceinline__ void parts_of_two(float x, float y, uint32_t (&p)[kParts]) {
  p[0] = fp8::pack2(x, y);
  float2 a = fp8::to_float2(p[0]);
  x = (x - a.x) * 16.f; y = (y - a.y) * 16.f;
  p[1] = fp8::pack2(x, y);
  a = fp8::to_float2(p[1]);
  __half2 r = __floats2half2_rn((x - a.x) * 16.f, (y - a.y) * 16.f);
  p[2] = fp8::pack2(r);
  const uint32_t b = fp8::to_half2(p[2]);
  r = __hmul2(__hsub2(r, *reinterpret_cast<const __half2*>(&b)), __float2half2_rn(16.f));
  p[3] = fp8::pack2(r);
}
__device__ __forceinline__ float max4(float4 v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }
// Lane h < N leaves v[h] (the same in all lanes) as warp w's number of head h.
template <int N> __device__ __forceinline__ void leave(float4* to, const float (&v)[N], int w, int lane) {
  float mine = v[0];
#pragma unroll
  for (int h = 1; h < N; ++h) mine = lane == h ? v[h] : mine;
  if (lane < N) reinterpret_cast<float*>(to + lane)[w] = mine;
}
// The sum of the parts' columns of a group's head h.
template <int N> __device__ __forceinline__ float join_parts(const uint32_t* c, int h) {
  float sum = __uint_as_float(c[(kParts - 1) * N + h]);
#pragma unroll
  for (int i = kParts - 2; i >= 0; --i) sum = fmaf(sum, 1.f / 16, __uint_as_float(c[i * N + h]));
  return sum;
}

// One claimed item as the lister keeps it (live == false: none).
struct DecClaim {
  int row, head, kvh, part, nblk, ntok, table_kind, tbl_off;
  int bid[4];
  bool live;
};

template <typename T, int D, int HMAX>
__global__ void __launch_bounds__((DecCfg<D, HMAX>::kThreads), (DecCfg<D, HMAX>::kCtas)) decode_fp8_kernel(const AttnDev d) {
  using C = DecCfg<D, HMAX>;
  extern __shared__ __align__(1024) uint8_t smem[];
  DecCtl& ctl = *reinterpret_cast<DecCtl*>(smem + C::kOffCtl);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int* abort_flag = &ctl.abort_flag;
  int32_t* status = &d.hdr[kHdrStatus];
  auto bar = [](uint64_t& b) { return smem_u32(&b); };

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(bar(ctl.full[s]), 64 + 1);  // the threads of the K warps, the copies of V
      mbar_init(bar(ctl.empty[s]), 1);
    }
    for (int i = 0; i < kDescSlots; ++i) {
      mbar_init(bar(ctl.desc_full[i]), 32);
      mbar_init(bar(ctl.desc_empty[i]), 1);
    }
    for (int i = 0; i < kItemSlots; ++i) {
      mbar_init(bar(ctl.item_full[i]), 1);
      mbar_init(bar(ctl.item_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(bar(ctl.q_full[i]), 32);
      mbar_init(bar(ctl.q_empty[i]), 1 + C::kW0);  // the MMAs that read it, the softmax warps (its factors)
      mbar_init(bar(ctl.s_full[i]), 1);
      mbar_init(bar(ctl.p_full[i]), 32 * C::kW0);
      mbar_init(bar(ctl.pv_done[i]), 1);
      mbar_init(bar(ctl.exchange[i]), 4);
    }
    ctl.abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == C::kW0 + 3) tmem_alloc(smem_u32(&ctl.tmem), C::kTmem);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // with a dense kernel in front of it this kernel starts beside it and waits for it at the very end (single_query.cuh)
  if (d.sq_waits_at_start) pdl_wait();
  pdl_trigger();
  int hpi = 1;  // query heads per item (several only under the usual mapping, which is looked at in every call)
  if constexpr (HMAX > 1) {
    const int share = d.num_heads / d.num_kv_heads;
    bool usual = true;
    for (int h = threadIdx.x; h < d.num_heads; h += C::kThreads) usual = usual && d.head_mapping[h] == h / share;
    if (__syncthreads_and(usual)) hpi = d.gqa_heads;
  }
  const uint32_t tmem = ctl.tmem;
  const uint32_t tmem_s = tmem, tmem_o = tmem + 2 * C::kN;
  const uint32_t stage0 = smem_u32(smem);

  if (warp == C::kW0) {
    // ================= lister: items, tiles, V =================
    const int H = d.num_heads / hpi;
    const long long n_items = (long long)d.hdr[kHdrNumSq] * H;
    auto describe = [&](long long id) {
      DecClaim c;
      c.live = id < n_items;
      c.nblk = 0;
      if (c.live) {
        const int sc = (int)(id / H);
        c.head = (int)(id - (long long)sc * H) * hpi;
        const int4 a = *reinterpret_cast<const int4*>(&d.sq_items[sc]);        // row, meta, ntok, part
        const int4 b = *(reinterpret_cast<const int4*>(&d.sq_items[sc]) + 1);  // bid[4]
        c.row = a.x; c.part = a.w; c.nblk = a.y & 0xffff; c.ntok = a.z;
        c.table_kind = (a.y & (1 << 17)) ? -1 : (a.y >> 18) & 3;
        c.tbl_off = b.x;
        c.bid[0] = b.x; c.bid[1] = b.y; c.bid[2] = b.z; c.bid[3] = b.w;
      }
      return c;
    };
    auto window = [&](DecClaim& c, int at) {  // lane l: block id at + l of the item's chunk (0 where there is none)
      if (!c.live || at + lane >= c.nblk) return 0;
      if (c.table_kind < 0) return lane == 0 ? c.bid[0] : lane == 1 ? c.bid[1] : lane == 2 ? c.bid[2] : c.bid[3];
      const int32_t* table = c.table_kind == 1 ? d.group_tables : c.table_kind == 2 ? d.seg_tables
                             : c.table_kind == 3 ? d.outer_tables : d.suffix_tables;
      return (int)table[c.tbl_off + at + lane];
    };
    auto settle = [&](DecClaim& c) {  // the item's kv head
      c.kvh = 0;
      if (!c.live) return;
      c.kvh = d.head_mapping ? d.head_mapping[c.head] : c.head;
      if (c.kvh < 0 || c.kvh >= d.num_kv_heads) {
        atomicMax(status, kStatusBadIndex);
        c.kvh = 0;
      }
    };
    auto scales_of = [&](const DecClaim& c, int at, int& blk, float& ks, float& vs) {
      ks = vs = 0.f;
      if (!c.live || at + lane >= c.nblk) return;
      if (blk < 0 || blk >= d.num_blocks) {
        atomicMax(status, kStatusBadIndex);
        blk = 0;
      }
      const size_t o = (size_t)blk * d.scale_block_stride + (size_t)c.kvh * d.scale_head_stride;
      ks = d.key_scale[o];
      vs = d.value_scale[o];
    };
    auto claim = [&]() { return lane == 0 ? atomicAdd(&d.hdr[kHdrSqCounter], 1) : 0; };
    uint32_t tc = 0, ic = 0;
    bool ok = true;
    DecClaim cur = describe(__shfl_sync(0xffffffffu, claim(), 0));
    settle(cur);
    int ids = window(cur, 0);
    float ks, vs;
    scales_of(cur, 0, ids, ks, vs);
    DecClaim nxt = describe(__shfl_sync(0xffffffffu, claim(), 0));
    while (ok && cur.live) {
      settle(nxt);
      int ids_n = window(nxt, 0);
      const int claimed = claim();
      float ks_n = 0.f, vs_n = 0.f;
      DecClaim after;
      if (ic >= kItemSlots && !wait_or_abort(bar(ctl.item_empty[ic % kItemSlots]), ((ic / kItemSlots) & 1) ^ 1, abort_flag, status)) break;
      if (lane == 0) {
        ctl.item[ic % kItemSlots].row = cur.row;
        ctl.item[ic % kItemSlots].head = cur.head;
        mbar_arrive(bar(ctl.item_full[ic % kItemSlots]));
      }
      ++ic;
      for (int b0 = 0; b0 < cur.nblk; b0 += 8, ++tc) {
        if (b0 > 0 && (b0 & 31) == 0) {  // chunks longer than 32 blocks: the next window
          ids = window(cur, b0);
          scales_of(cur, b0, ids, ks, vs);
        }
        const int nb = min(8, cur.nblk - b0);
        const int r = tc % kDescSlots;
        if (tc >= kDescSlots && !wait_or_abort(bar(ctl.desc_empty[r]), ((tc / kDescSlots) & 1) ^ 1, abort_flag, status)) { ok = false; break; }
        const int src = (b0 & 31) + (lane & 7);
        const int blk = __shfl_sync(0xffffffffu, ids, src);
        const float k1 = __shfl_sync(0xffffffffu, ks, src), v1 = __shfl_sync(0xffffffffu, vs, src);
        DecDesc& e = ctl.desc[r];
        if (lane < 8) {
          e.blk[lane] = blk;
          e.ks[lane] = k1;
          e.lv[lane] = v1 >= fp8::kMinValueScale ? __log2f(v1) : v1 >= 0.f ? -INFINITY : __int_as_float(0x7fc00000);
        }
        if (lane == 0) {
          e.nb = nb;
          e.ntok = min(8 * 16, cur.ntok - b0 * 16);
          e.row = cur.row; e.head = cur.head; e.part = cur.part; e.kvh = cur.kvh;
          e.first = b0 == 0;
          e.last = b0 + 8 >= cur.nblk;
        }
        mbar_arrive(bar(ctl.desc_full[r]));
        if (b0 == 0) {
          scales_of(nxt, 0, ids_n, ks_n, vs_n);
          after = describe(__shfl_sync(0xffffffffu, claimed, 0));
        }
      }
      cur = nxt;
      ids = ids_n;
      ks = ks_n;
      vs = vs_n;
      nxt = after;
    }
    if (ok && !cur.live) {
      // no more items: tell the tile readers and the query warp
      if (tc < kDescSlots || wait_or_abort(bar(ctl.desc_empty[tc % kDescSlots]), ((tc / kDescSlots) & 1) ^ 1, abort_flag, status)) {
        if (lane == 0) ctl.desc[tc % kDescSlots].nb = 0;
        mbar_arrive(bar(ctl.desc_full[tc % kDescSlots]));
      }
      if (ic < kItemSlots || wait_or_abort(bar(ctl.item_empty[ic % kItemSlots]), ((ic / kItemSlots) & 1) ^ 1, abort_flag, status)) {
        if (lane == 0) {
          ctl.item[ic % kItemSlots].row = -1;
          mbar_arrive(bar(ctl.item_full[ic % kItemSlots]));
        }
      }
    }
  } else if (warp == C::kW0 + 1 || warp == C::kW0 + 2) {
    // ===== K: 16-byte async copies, the chunk rows of the tile's blocks side by side. V: bulk copies, by the first warp =====
    const uint8_t* kc = reinterpret_cast<const uint8_t*>(d.key_cache);
    const uint8_t* vc = reinterpret_cast<const uint8_t*>(d.value_cache);
    const uint64_t policy = l2_policy_evict_first();
    bool drain = true;
    uint32_t tc = 0;
    for (;; ++tc) {
      const int s = tc % C::kStages, r = tc % kDescSlots;
      if (!wait_or_abort(bar(ctl.desc_full[r]), (tc / kDescSlots) & 1, abort_flag, status)) break;
      const DecDesc& e = ctl.desc[r];
      const int nb = e.nb;
      if (nb == 0) {
        drain = false;  // (the MMAs wait for all of it)
        break;
      }
      if (tc >= C::kStages && !wait_or_abort(bar(ctl.empty[s]), ((tc / C::kStages) & 1) ^ 1, abort_flag, status)) break;
      if (warp == C::kW0 + 1) {
        if (lane == 0) mbar_arrive_expect_tx(bar(ctl.full[s]), nb * C::kTile);
        __syncwarp();
        if (lane < nb)
          bulk_g2s_hint(stage0 + s * C::kStage + (8 + lane) * C::kTile,
                        vc + (size_t)e.blk[lane] * d.kv_block_stride + (size_t)e.kvh * d.kv_head_stride, C::kTile, bar(ctl.full[s]), policy);
      }
      for (int j = warp - C::kW0 - 1; j < nb; j += 2) {
        const uint8_t* src = kc + (size_t)e.blk[j] * d.kv_block_stride + (size_t)e.kvh * d.kv_head_stride + lane * 16;
        const uint32_t dst = stage0 + s * C::kStage + (lane >> 4) * 2048 + j * 256 + (lane & 15) * 16;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) cp_async16(dst + k * 2 * 2048, src + k * 512);
      }
      cp_async_arrive_noinc(bar(ctl.full[s]));
    }
    cp_async_wait_all();
    if (drain && warp == C::kW0 + 1)  // give copies already issued a bounded chance to land before shared memory goes away
      for (uint32_t c = tc > C::kStages ? tc - C::kStages : 0; c < tc; ++c)
        (void)mbar_wait_bounded(bar(ctl.full[c % C::kStages]), (c / C::kStages) & 1);
  } else if (warp == C::kW0 + 4) {
    // ================= query operands =================
    const uint8_t* qg = reinterpret_cast<const uint8_t*>(d.query);
    for (uint32_t ic = 0;; ++ic) {
      if (!wait_or_abort(bar(ctl.item_full[ic % kItemSlots]), (ic / kItemSlots) & 1, abort_flag, status)) break;
      const int row = ctl.item[ic % kItemSlots].row, head = ctl.item[ic % kItemSlots].head;
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(ctl.item_empty[ic % kItemSlots]));
      if (row < 0) break;
      const int slot = ic % C::kQSlots;
      uint2 raw[HMAX];
#pragma unroll
      for (int h = 0; h < HMAX; ++h)
        raw[h] = (h < hpi && lane < D / 4) ? *reinterpret_cast<const uint2*>(qg + ((size_t)row * d.q_stride + (size_t)(head + h) * D + 4 * lane) * 2)
                                           : make_uint2(0u, 0u);
      if (ic >= C::kQSlots && !wait_or_abort(bar(ctl.q_empty[slot]), ((ic / C::kQSlots) & 1) ^ 1, abort_flag, status)) break;
      uint8_t* qop = smem + C::kOffQ + slot * C::kQ;
#pragma unroll
      for (int h = 0; h < HMAX; ++h) {
        float f[4];
        if constexpr (std::is_same<T, __half>::value) {
          const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw[h].x)), b = __half22float2(*reinterpret_cast<const __half2*>(&raw[h].y));
          f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
        } else {
          f[0] = __uint_as_float(raw[h].x << 16); f[1] = __uint_as_float(raw[h].x & 0xffff0000u);
          f[2] = __uint_as_float(raw[h].y << 16); f[3] = __uint_as_float(raw[h].y & 0xffff0000u);
        }
        float top = 0.f;
        bool odd = false;  // NaN or an infinity: the parts could not say so
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          top = fmaxf(top, fabsf(f[i]));
          odd = odd || !(fabsf(f[i]) <= 3.402823466e38f);
        }
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        odd = __any_sync(0xffffffffu, odd);
        const int e = min(max((int)(__float_as_uint(top) >> 23), 20), 254);
        const float up = __uint_as_float((uint32_t)(261 - e) << 23);  // the largest element into [2^7, 2^8)
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] *= up;
#pragma unroll
        for (int p = 0; p < kParts; ++p) {
          const uint32_t lo = fp8::pack2(f[0], f[1]), hi = fp8::pack2(f[2], f[3]);
          const float2 a = fp8::to_float2(lo), b = fp8::to_float2(hi);
          f[0] = (f[0] - a.x) * 16.f; f[1] = (f[1] - a.y) * 16.f; f[2] = (f[2] - b.x) * 16.f; f[3] = (f[3] - b.y) * 16.f;
          const int n = (h / C::kHeads * kParts + p) * C::kHeads + h % C::kHeads;
          if (lane < D / 4)
            *reinterpret_cast<uint32_t*>(qop + (lane >> 2) * (C::kN * 16) + (n >> 3) * 128 + (n & 7) * 16 + (lane & 3) * 4) = lo | (hi << 16);
        }
        if (lane == 0)
          ctl.mul[slot][h] = odd ? __int_as_float(0x7fc00000) : d.scale_log2e * __uint_as_float((uint32_t)(e - 7) << 23);
      }
      fence_proxy_async_smem();
      mbar_arrive(bar(ctl.q_full[slot]));
    }
  } else if (warp == C::kW0 + 3) {
    // ================= MMA issuer =================
    // S(t + 1) as soon as its tile is there, O(t) as soon as its weights are: whichever comes first.
    constexpr uint32_t kIdesc = (1u << 4) | ((uint32_t)(C::kN >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);  // fp32 += e4m3 . e4m3
    // Descriptors: the operands' addresses (in sixteens of bytes) are added to words made once. (Made anew for every MMA by the one
    // thread that issues them they cost more than the products, 1500 cycles a tile: 128 sequences of 32 heads over 8 took 88 us, 80 so.)
    const uint64_t dk = smem_desc(stage0, 2048, 128, 0), dv = smem_desc(stage0 + 8 * C::kTile, C::kTile, 128, 0);
    const uint64_t dq = smem_desc(smem_u32(smem + C::kOffQ), C::kN * 16, 128, 0), dw = smem_desc(smem_u32(smem + C::kOffW), C::kN * 16, 128, 0);
    const uint32_t k_hi = (uint32_t)(dk >> 32), v_hi = (uint32_t)(dv >> 32), n_hi = (uint32_t)(dq >> 32);
    const uint32_t k_lo = (uint32_t)dk, v_lo = (uint32_t)dv, q_lo = (uint32_t)dq, w_lo = (uint32_t)dw;
    auto word = [](uint32_t hi, uint32_t lo) { return ((uint64_t)hi << 32) | lo; };
    uint32_t qk = 0, pv = 0;           // next tile of either product
    uint32_t qk_item = 0, pv_item = 0;  // items that have begun
    int qk_nb = -1, pv_nb[2] = {0, 0};  // blocks of tile qk (-1: not seen yet), and of the tiles on their way
    bool qk_first = false, qk_last = false, pv_first[2] = {false, false};
    bool ok = true, more = true;
    uint64_t t_start = 0;
    uint32_t spin = 0;
    while (ok && (more || pv < qk)) {
      bool progress = false;
      if (more && qk <= pv + 1) {
        const uint32_t r = qk % kDescSlots, s = qk % C::kStages;
        if (qk_nb < 0) {
          bool there = mbar_test_wait(bar(ctl.desc_full[r]), (qk / kDescSlots) & 1);
          there = __all_sync(0xffffffffu, there);
          if (there) {
            const DecDesc& e = ctl.desc[r];
            qk_nb = e.nb; qk_first = e.first; qk_last = e.last;
            if (qk_nb == 0) more = false;
            progress = true;
          }
        }
        if (qk_nb > 0) {
          const uint32_t item = qk_item + (qk_first ? 1 : 0) - 1;
          bool ready = mbar_test_wait(bar(ctl.full[s]), (qk / C::kStages) & 1);
          if (qk_first) ready = ready && mbar_test_wait(bar(ctl.q_full[item % C::kQSlots]), (item / C::kQSlots) & 1);
          ready = __all_sync(0xffffffffu, ready);
          if (ready) {
            fence_proxy_async_smem();  // K was written by per-thread async copies
            tc_fence_after();
            if (lane == 0) {
              const uint32_t a = k_lo + s * (C::kStage >> 4), b = q_lo + (item % C::kQSlots) * (C::kQ >> 4), to = tmem_s + (qk & 1) * C::kN;
#pragma unroll
              for (int kk = 0; kk < D / 32; ++kk)  // 32 of d: two 16-byte chunks
                mma_f8(to, word(k_hi, a + kk * (2 * 2048 >> 4)), word(n_hi, b + kk * 2 * C::kN), kIdesc, kk > 0 ? 1u : 0u);
              mma_commit(bar(ctl.s_full[qk & 1]));
              if (qk_last) mma_commit(bar(ctl.q_empty[item % C::kQSlots]));
            }
            __syncwarp();
            if (qk & 1) { pv_nb[1] = qk_nb; pv_first[1] = qk_first; } else { pv_nb[0] = qk_nb; pv_first[0] = qk_first; }
            qk_item = item + 1;
            ++qk;
            qk_nb = -1;
            progress = true;
          }
        }
      }
      if (pv < qk) {
        bool ready = mbar_test_wait(bar(ctl.p_full[pv & 1]), (pv >> 1) & 1);
        ready = __all_sync(0xffffffffu, ready);
        if (ready) {
          tc_fence_after();
          const uint32_t r = pv % kDescSlots, s = pv % C::kStages;
          const int nb = (pv & 1) ? pv_nb[1] : pv_nb[0];
          const bool first = (pv & 1) ? pv_first[1] : pv_first[0];
          pv_item += first ? 1 : 0;
          if (lane == 0) {
            const uint32_t a = v_lo + s * (C::kStage >> 4), b = w_lo + (pv & 1) * (C::kW >> 4), to = tmem_o + ((pv_item - 1) & 1) * C::kN;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)  // 32 tokens: two blocks (the softmax threads have cleared what is missing)
              if (2 * kk < nb)
                mma_f8(to, word(v_hi, a + kk * (2 * C::kTile >> 4)), word(n_hi, b + kk * 2 * C::kN), kIdesc, (kk > 0 || !first) ? 1u : 0u);
            mma_commit(bar(ctl.empty[s]));
            mma_commit(bar(ctl.pv_done[pv & 1]));
            mbar_arrive(bar(ctl.desc_empty[r]));
          }
          __syncwarp();
          ++pv;
          progress = true;
        }
      }
      if (progress) {
        spin = 0;
        t_start = 0;
      } else if (__nanosleep(20), (++spin & 255u) == 0) {
        bool give_up = (*abort_flag != 0);
        const uint64_t now = global_timer_ns();
        if (t_start == 0) t_start = now;
        else if (now - t_start > 2000000000ull) give_up = true;
        if (__any_sync(0xffffffffu, give_up)) {
          *abort_flag = 1;
          atomicMax(status, kStatusWaitExpired);
          ok = false;
        }
      }
    }
  } else {
    // ================= softmax (a token per thread) and epilogue (an element d per thread) =================
    constexpr int N = C::kHeads;
    const int g = warp >> 2, quarter = warp & 3, h0 = g * N;  // the group's first head
    const int r = quarter * 32 + lane;
    const uint32_t lane_base = ((uint32_t)(quarter * 32) << 16) + g * kParts * N;  // (and its columns)
    const int blk_of = r >> 4;
    float mul[N], ref[N], l[N], mx[N];
    uint32_t items = 0, x_use = 0;
#pragma unroll
    for (int h = 0; h < N; ++h) { mul[h] = 0.f; ref[h] = -INFINITY; l[h] = 0.f; mx[h] = -INFINITY; }
    // An item's partial: sums and exact maxima of the four warps, O from tensor memory. It waits for the product of the item's last
    // tile, so it is put off until the next item's first weights are on their way (O and what is left of an item have two places).
    bool pending = false;
    uint32_t last_tc = 0;
    auto epilogue = [&](uint32_t item, uint32_t tile) -> bool {
      const int at = item & 1, row = ctl.left_row[g][at], head = ctl.left_head[g][at], part = ctl.left_part[g][at];
      if (!wait_or_abort(bar(ctl.pv_done[tile & 1]), (tile >> 1) & 1, abort_flag, status)) return false;
      tc_fence_after();
      uint32_t o[kParts * N];
      ld_cols<N>(tmem_o + at * C::kN + lane_base, o);
      tmem_wait_ld();
      tc_fence_before();
#pragma unroll
      for (int h = 0; h < N; ++h) {
        if (h0 + h < hpi) {
          const float4 sums = ctl.left_sum[g][at][h];
          const float sum = (sums.x + sums.y) + (sums.z + sums.w);
          const float m = told_max(max4(ctl.left_max[g][at][h]), sum), ref_h = ctl.left_ref[g][at][h];
          const float fix = ref_h == -INFINITY ? 0.f : fast_exp2(ref_h - m);
          const float v = join_parts<N>(o, h);
          const size_t slot = partial_slot(d, row, part, head + h0 + h);
          if (r < D) d.acc[slot * D + r] = v * (fix * (1.f / 256));  // (2^-kTop)
          if (r == 0) d.ml[slot] = make_float2(m, sum * fix);
        }
      }
      return true;
    };
    for (uint32_t tc = 0;; ++tc) {
      const int rr = tc % kDescSlots, s = tc % C::kStages, buf = tc & 1;
      if (!wait_or_abort(bar(ctl.desc_full[rr]), (tc / kDescSlots) & 1, abort_flag, status)) break;
      const DecDesc& e = ctl.desc[rr];
      const int nb = e.nb, ntok = e.ntok, row = e.row, head = e.head, part = e.part;
      const bool first = e.first, last = e.last;
      if (nb == 0) break;
      const float ks = e.ks[blk_of], lv = e.lv[blk_of];
      if (first) {
        const int slot = items % C::kQSlots;
        if (!wait_or_abort(bar(ctl.q_full[slot]), (items / C::kQSlots) & 1, abort_flag, status)) break;
#pragma unroll
        for (int h = 0; h < N; ++h) { mul[h] = ctl.mul[slot][h0 + h]; ref[h] = -INFINITY; l[h] = 0.f; mx[h] = -INFINITY; }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(ctl.q_empty[slot]));
        ++items;
      }
      if (!wait_or_abort(bar(ctl.s_full[buf]), (tc >> 1) & 1, abort_flag, status)) break;
      tc_fence_after();
      uint32_t c[kParts * N];
      ld_cols<N>(tmem_s + buf * C::kN + lane_base, c);
      tmem_wait_ld();
      const bool seen = r < ntok;
      float lg[N], top[N];
#pragma unroll
      for (int h = 0; h < N; ++h) {
        lg[h] = seen ? join_parts<N>(c, h) * (ks * mul[h]) : -INFINITY;
        mx[h] = fmaxf(mx[h], lg[h]);
        top[h] = seen ? lg[h] + fmaxf(lv, kMinLv) : -INFINITY;  // (a block without a scale: no weight, but a reference)
      }
#pragma unroll
      for (int h = 0; h < N; ++h) top[h] = warp_max(top[h]);
      // the tile's maximum, from the four warps
      const int xb = x_use & 1;
      leave(ctl.xmax[g][xb], top, quarter, lane);
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(ctl.exchange[g]));
      if (!wait_or_abort(bar(ctl.exchange[g]), x_use & 1, abort_flag, status)) break;
      ++x_use;
      bool grow = false;
      float alpha[N];
#pragma unroll
      for (int h = 0; h < N; ++h) {
        const float m = max4(ctl.xmax[g][xb][h]);
        alpha[h] = 1.f;
        if (m > ref[h] + kLag) {
          alpha[h] = fast_exp2(ref[h] - m);
          ref[h] = m;
          grow = true;
        }
        l[h] *= alpha[h];
      }
      if (grow && !first) {  // (the same for all warps of the group) the accumulator follows, once the previous tile is in it
        if (!wait_or_abort(bar(ctl.pv_done[buf ^ 1]), ((tc - 1) >> 1) & 1, abort_flag, status)) break;
        tc_fence_after();
        uint32_t o[kParts * N];
        const uint32_t at = tmem_o + ((items - 1) & 1) * C::kN + lane_base;
        ld_cols<N>(at, o);
        tmem_wait_ld();
#pragma unroll
        for (int h = 0; h < N; ++h)
#pragma unroll
          for (int p = 0; p < kParts; ++p) o[p * N + h] = __float_as_uint(__uint_as_float(o[p * N + h]) * alpha[h]);
        st_cols<N>(at, o);
        tmem_wait_st();
      }
      uint8_t* wop = smem + C::kOffW + buf * C::kW + blk_of * (C::kN * 16) + (r & 15);
      const int n0 = g * kParts * N;  // the group's first column
      float w[N];
#pragma unroll
      for (int h = 0; h < N; ++h) {
        const float base = ref[h] == -INFINITY ? 0.f : ref[h];  // (nothing but logits of -inf so far)
        l[h] += fast_exp2(lg[h] - base);
        w[h] = fast_exp2(lg[h] + (lv - base + kTop));
      }
      auto put = [&](int i, uint32_t code) {
        const int n = n0 + i;
        wop[(n >> 3) * 128 + (n & 7) * 16] = (uint8_t)code;
      };
      uint32_t p[kParts];
      if constexpr (N == 1) {
        parts_of(w[0], p);
#pragma unroll
        for (int i = 0; i < kParts; ++i) put(i, p[i]);
      } else {
#pragma unroll
        for (int h = 0; h < N; h += 2) {
          parts_of_two(w[h], w[h + 1], p);
#pragma unroll
          for (int i = 0; i < kParts; ++i) {
            put(i * N + h, p[i]);
            put(i * N + h + 1, p[i] >> 8);
          }
        }
      }
      if ((ntok & 31) && r < D && g == 0) {
        // the last 32 tokens are not all there: clear the codes behind the context (0 * NaN would not be 0)
        if (!wait_or_abort(bar(ctl.full[s]), (tc / C::kStages) & 1, abort_flag, status)) break;
        uint8_t* v = smem + s * C::kStage + 8 * C::kTile + r * 16;
        if (ntok & 15) {
          uint4* cell = reinterpret_cast<uint4*>(v + (ntok >> 4) * C::kTile);
          uint32_t x[4] = {cell->x, cell->y, cell->z, cell->w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = (ntok & 15) - 4 * i;
            x[i] &= n <= 0 ? 0u : n >= 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
          }
          *cell = make_uint4(x[0], x[1], x[2], x[3]);
        }
        if (nb & 1) *reinterpret_cast<uint4*>(v + nb * C::kTile) = make_uint4(0u, 0u, 0u, 0u);
      }
      fence_proxy_async_smem();
      tc_fence_before();
      mbar_arrive(bar(ctl.p_full[buf]));
      if (pending) {
        if (!epilogue(items - 2, tc - 1)) break;
        pending = false;
      }
      if (!last) continue;
      // ---- what the item's epilogue needs is left in shared memory (this phase's exchange orders it) ----
      const int at = (items - 1) & 1;
#pragma unroll
      for (int h = 0; h < N; ++h) {
        mx[h] = warp_max(mx[h]);
#pragma unroll
        for (int o = 16; o >= 1; o >>= 1) l[h] += __shfl_xor_sync(0xffffffffu, l[h], o);
        if (r == 0) ctl.left_ref[g][at][h] = ref[h];
      }
      leave(ctl.left_max[g][at], mx, quarter, lane);
      leave(ctl.left_sum[g][at], l, quarter, lane);
      if (r == 0) {
        ctl.left_row[g][at] = row;
        ctl.left_head[g][at] = head;
        ctl.left_part[g][at] = part;
      }
      pending = true;
      last_tc = tc;
    }
    if (pending && *abort_flag == 0) {  // the last item's
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(ctl.exchange[g]));
      if (wait_or_abort(bar(ctl.exchange[g]), x_use & 1, abort_flag, status)) (void)epilogue(items - 1, last_tc);
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == C::kW0 + 3) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmem);
  }
  if (!d.sq_waits_at_start) pdl_wait();  // the dense prefix kernel has completed
}

template <typename T, int D, int HMAX>
cudaError_t launch_dec(const AttnDev& d, cudaStream_t s) {
  using C = DecCfg<D, HMAX>;
  constexpr int smem = C::kOffCtl + (int)sizeof(DecCtl);
  static_assert(C::kStages <= 8, "stages");
  static_assert((smem + 1024) * C::kCtas <= 228 * 1024, "shared memory budget");
  auto kfn = decode_fp8_kernel<T, D, HMAX>;
  cudaError_t e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  return launch_kernel(kfn, d.num_sms * C::kCtas, C::kThreads, smem, s, true, d);
}

template <typename T>
cudaError_t launch_dec_t(const AttnDev& d, int head_size, cudaStream_t s) {
#define PB_DEC(DD)                                                                            \
  if (head_size == DD)                                                                        \
    return d.gqa_heads == 1 ? launch_dec<T, DD, 1>(d, s) : d.gqa_heads <= 4 ? launch_dec<T, DD, 4>(d, s) : launch_dec<T, DD, 8>(d, s);
  PB_DEC(64) PB_DEC(96) PB_DEC(128)
#undef PB_DEC
  return cudaErrorInvalidValue;
}

}  // namespace

bool decode_fp8_supported(int dtype, int head_size, int block_size) {
  return fp8::decode_on_tc(dtype == PB_F16 || dtype == PB_BF16, head_size, block_size);
}
cudaError_t launch_decode_fp8(const AttnDev& d, int dtype, int head_size, cudaStream_t s) {
  return dtype == PB_F16 ? launch_dec_t<__half>(d, head_size, s) : launch_dec_t<__nv_bfloat16>(d, head_size, s);
}

}  // namespace pb
