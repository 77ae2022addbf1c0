// Prefix and prefill stage over the 8-bit cache: the row-tile pairs of dense_pair.cu (tcgen05 + TMEM), for lone row tiles too.
//
// What the scales do. With (ks, vs) the scales of block b, c = scale * log2(e) and f the factor of the query row (below):
//     lg_t = s_t * ks[b] * c / f         u_t = lg_t + lv[b],  lv = log2(vs)
//     w_t  = 2^(u_t - M + kShift)        l += 2^-lv[b] * sum of the block's w_t          O += w_t v8_t
// with M the lazy reference of max u, so that the weights use fp16's range whatever the scales are. A block with vs = 0, or below 2^kMinLv,
// which counts as 0, gets zeros as V and lv = kMinLv.
//
// What feeds the tensor cores:
//   S_x = Q_x . K^T   kind::f8f6f4 on the codes of K as they are. Q comes as a sum of e4m3 parts, each the rounded remainder of
//                     those before it (3 for fp16, 2 for bf16: 12 and 8 bits), of rows multiplied by the power of two f that
//                     puts their largest element into [2^7, 2^8). A part has 8-bit operands at twice the rate of 16-bit ones.
//                     An element is off by 2^-12 (2^-8 for bf16, whose 8 bits that are) of itself or 2^-10, 2^-17 of the row's
//                     largest. The parts are made once per call by a kernel in front (query_parts_kernel) and come by TMA.
//   O_x += P_x . V    kind::f16: P_x in fp16 from tensor memory, V converted to fp16 (exact) on its way into its ring. A weight is off by
//                     2^-12 of itself for that, what a rounding of the output to fp16 costs (a low part would double the products and does
//                     not fit beside S in tensor memory); the sum l takes it unrounded. Against 64 bits, 64 rows over 4096 tokens, fp16:
//                     2.7e-4 (2-norm, relative), 2.1e-4 with 32-bit weights.
// Converting K like V, on four warps more, kept the SM's instruction caches and the softmax warps' schedulers busy with it: a
// kv tile of 128 rows took 3.0 us.
// What bounds it: the chain of a row tile, S, maximum, exponentials, P.V, and in it the exponentials (a thread spends 2600 of the 6200
// cycles of a kv tile on its 128, of which 2048 are the special-function unit's for the pair). 1024 rows over 16384 tokens, 32
// heads: 398 us, 691 TFLOP/s; 64 rows over 65536: 271 us, 2.0 TB/s of codes.
//
// Warps 0-3 and 4-7: softmax and epilogue of row tile 0 and 1, one thread per row; 8-11 convert V; 12 copies K and asks for
// Q; 13, 14 issue the MMAs of row tile 0 and 1; 15 lists the tiles. Every mbarrier wait is bounded; on expiry the CTA
// records a status, drains and returns.
#include "common.cuh"
#include "dense_common.cuh"
#include "fp8.cuh"

namespace pb {
namespace {

using namespace dense;
using fp8::kMinLv;
using fp8::told_max;
using fp8::warp_max;

constexpr float kShift = 7.f;                            // w <= 2^(kTau + kShift) = 2^15
constexpr int kCodeBytes = kBlkBytes / 2;                // one K or V tile of a (block, head): 2 KiB
constexpr int kPartBytes = 128 * kD;                     // one part of a row tile's Q
constexpr int kRingK = kTileBlocks * kCodeBytes;         // one K slot: 16 KiB of codes
constexpr int kStageBytes = 16384;                       // epilogue staging of one softmax group
constexpr int kConvWarps = 4;                            // converters of V: two blocks of a tile each
constexpr int kDescSlots = 8;
constexpr int kThreads = 512;
constexpr int kGroupThreads = 128;                       // softmax threads of one row tile
constexpr uint32_t kTmemCols = 512;                      // S_0, S_1, O_0, O_1
// The roles in warpgroups, with the registers each keeps (setmaxnreg): two of softmax threads, the converters, the rest. The
// shares sum up to no more than the block is launched with.
constexpr int kRegsLaunch = 128, kRegsSoftmax = 160, kRegsConvert = 96, kRegsIssue = 96;
static_assert(256 * kRegsSoftmax + 128 * kRegsConvert + 128 * kRegsIssue <= kThreads * kRegsLaunch, "register shares");
template <int kRegs> __device__ __forceinline__ void regs_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs> __device__ __forceinline__ void regs_fewer() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

template <typename T> struct QParts { static constexpr int kNum = Pack<T>::kBf16 ? 2 : 3; };

// barriers 0-7: the K and V rings (dense_common.cuh); per row tile x the index is base + x
enum {
  kBarS = 8,         // S_x of a kv tile is in tensor memory
  kBarP = 10,        // P_x of a kv tile is in tensor memory (all 128 rows)
  kBarPV = 12,       // P_x.V of a kv tile has retired: O_x holds it, S_x / P_x may be overwritten
  kBarQ = 14,        // Q_x of a segment has landed
  kBarQFree = 16,    // every Q_x.K^T of a segment has retired: Q_x may be overwritten
  kBarODrained = 18, // the epilogue of a segment has read O_x out of tensor memory
  kBarGroup = 20,    // meeting point of the 128 softmax threads of row tile x (bounded, unlike bar.sync)
  kBarTurn = 22,     // issuer x has issued P_x.V and the next Q_x.K^T of a kv tile (pair items)
  kBarHand = 24,     // (lone row tile) group 1 has left its maxima and sums, and O_1 holds all its tiles
  kNumBars = 25
};

// What the other roles need to know of a kv tile, written by the warp that lists them. A ring of slots, each with a full
// and an empty barrier. Slot t is given back when a V converter has seen tile t's V slot become free: its P.V has retired then, so
// everybody is through with it.
struct TileDesc {
  int32_t blk[kTileBlocks];    // (the complement of the id: a block whose V is zero)
  int32_t nb, ntok, kvh;       // nb == 0: no more tiles
  int32_t row0, head, nrows;   // of the segment, if the tile is its first (else nrows == 0)
  int32_t pad[2];
  float ks[kTileBlocks], lv[kTileBlocks], inv[kTileBlocks];
};
struct TileRing {
  TileDesc desc[kDescSlots];
  uint64_t full[kDescSlots], empty[kDescSlots];
  __device__ __forceinline__ void init() {  // one thread
    for (int i = 0; i < kDescSlots; ++i) {
      mbar_init(smem_u32(&full[i]), 32);
      mbar_init(smem_u32(&empty[i]), 1);
    }
  }
  __device__ __forceinline__ uint32_t full_bar(uint32_t tc) { return smem_u32(&full[tc % kDescSlots]); }
  __device__ __forceinline__ uint32_t empty_bar(uint32_t tc) { return smem_u32(&empty[tc % kDescSlots]); }
  __device__ __forceinline__ uint32_t parity(uint32_t tc) { return (tc / kDescSlots) & 1; }
};

template <typename T> struct Layout {
  static constexpr int kOffQ = 0;                                     // Q_0, Q_1: their parts
  static constexpr int kOffK = 2 * QParts<T>::kNum * kPartBytes;
  static constexpr int kOffV = kOffK + kStages * kRingK;
  static constexpr int kOffStage = kOffV + kStages * kRingBytes;
  static constexpr int kOffBars = kOffStage + 2 * kStageBytes;
  static constexpr int kOffRing = kOffBars + 256;
  static constexpr int kSmemBytes = kOffRing + (int)sizeof(TileRing);
  static_assert(kSmemBytes <= 227 * 1024, "shared memory budget");
};

// ---- query rows as sums of e4m3 parts: a CTA per row and 32 heads, a warp four heads, a lane four elements of each ----
// (A warp per (row, head) had too little on its way to memory: 10714 rows x 32 heads 72 us, 48 so.)
constexpr int kPartsHeads = 4;
template <typename T>
__global__ void __launch_bounds__(256) query_parts_kernel(const AttnDev d) {
  pdl_wait();  // the workspace may still be the kernel's before this one
  pdl_trigger();
  const int lane = threadIdx.x & 31;
  const int row = blockIdx.x, h0 = (blockIdx.y * 8 + (threadIdx.x >> 5)) * kPartsHeads;
  uint2 in[kPartsHeads];
#pragma unroll
  for (int k = 0; k < kPartsHeads; ++k)
    if (h0 + k < d.num_heads)
      in[k] = *reinterpret_cast<const uint2*>(reinterpret_cast<const T*>(d.query) + (size_t)row * d.q_stride + (size_t)(h0 + k) * kD + 4 * lane);
#pragma unroll
  for (int k = 0; k < kPartsHeads; ++k) {
    const int head = h0 + k;
    if (head >= d.num_heads) break;
    const uint2 raw = in[k];
    float f[4];
    if constexpr (Pack<T>::kBf16) {
      f[0] = __uint_as_float(raw.x << 16); f[1] = __uint_as_float(raw.x & 0xffff0000u);
      f[2] = __uint_as_float(raw.y << 16); f[3] = __uint_as_float(raw.y & 0xffff0000u);
    } else {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&raw.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&raw.y));
      f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    }
    float top = 0.f;
    bool odd = false;  // NaN or an infinity: the parts could not say so
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      top = fmaxf(top, fabsf(f[i]));
      odd = odd || !(fabsf(f[i]) <= 3.402823466e38f);
    }
    top = warp_max(top);
    odd = __any_sync(0xffffffffu, odd);
    const int e = min(max((int)(__float_as_uint(top) >> 23), 20), 254);
    const float up = __uint_as_float((uint32_t)(261 - e) << 23);
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] *= up;
#pragma unroll
    for (int p = 0; p < QParts<T>::kNum; ++p) {
      const uint32_t lo = fp8::pack2(f[0], f[1]), hi = fp8::pack2(f[2], f[3]);
      const float2 a = fp8::to_float2(lo), b = fp8::to_float2(hi);
      f[0] -= a.x; f[1] -= a.y; f[2] -= b.x; f[3] -= b.y;
      *reinterpret_cast<uint32_t*>(d.q_parts + (((size_t)p * d.num_heads + head) * d.num_rows + row) * kD + 4 * lane) = lo | (hi << 16);
    }
    if (lane == 0)
      d.q_mul[(size_t)head * d.num_rows + row] = odd ? __int_as_float(0x7fc00000) : d.scale_log2e * __uint_as_float((uint32_t)(e - 7) << 23);
  }
}

// The warp that lists the tiles: block ids, scales and extents of every kv tile of this CTA, as far ahead as the ring allows.
// Four tiles at a time (lane 8 i + j: block j of tile i), and while four are published the scales of the next four and the block
// ids of those behind them are on their way: one after the other, a tile took the two trips to memory, twice what its
// products take. It also asks L2 for the tiles' codes.
__device__ __forceinline__ void list_tiles(const AttnDev& d, SegmentWalker& walk, int lane, TileRing* ring, volatile int* abort_flag,
                                           int32_t* status) {
  const int ti = lane >> 3, j = lane & 7;
  struct Batch {
    int n;                       // tiles; 0: no more
    int blk, nb, ntok, kvh;      // of this lane's tile and block
    int row0, head, nrows;       // of the segment that begins with tile 0 (nrows == 0: none does)
    float ks, vs;
  };
  Segment sg;
  bool have = walk.next(sg);
  int t = have ? sg.t0 : 0;
  auto take_ids = [&](Batch& b) {
    b.n = 0;
    if (!have) return;
    b.n = min(4, sg.t1 - t);
    b.kvh = d.head_mapping ? d.head_mapping[sg.head] : sg.head;
    b.row0 = sg.it.row0;
    b.head = sg.head;
    b.nrows = t == sg.t0 ? sg.it.nrows : 0;
    b.nb = 0;
    b.blk = 0;
    if (ti < b.n) {
      const DenseTileView tv = dense_tile_view(d, sg.it, t + ti);
      b.nb = tv.nb;
      b.ntok = tv.ntok;
      if (j < tv.nb) b.blk = tv.table[j];
    }
    t += b.n;
    if (t == sg.t1) {
      have = walk.next(sg);
      if (have) t = sg.t0;
    }
  };
  auto take_scales = [&](Batch& b) {
    b.ks = b.vs = 0.f;
    if (b.n == 0 || j >= b.nb) return;
    const bool bad_head = b.kvh < 0 || b.kvh >= d.num_kv_heads;
    if (b.blk < 0 || b.blk >= d.num_blocks || bad_head) {
      atomicMax(status, kStatusBadIndex);
      b.blk = 0;
      if (bad_head) b.kvh = 0;
    }
    const size_t at = (size_t)b.blk * d.scale_block_stride + (size_t)b.kvh * d.scale_head_stride;
    b.ks = d.key_scale[at];
    b.vs = d.value_scale[at];
    const size_t tile = (size_t)b.blk * d.kv_block_stride + (size_t)b.kvh * d.kv_head_stride;
    prefetch_l2(reinterpret_cast<const uint8_t*>(d.key_cache) + tile, kBlkBytes / 2);
    prefetch_l2(reinterpret_cast<const uint8_t*>(d.value_cache) + tile, kBlkBytes / 2);
  };
  Batch cur, nxt, after;
  take_ids(cur);
  take_ids(nxt);
  take_scales(cur);
  uint32_t tc = 0;
  bool ok = true;
  while (cur.n > 0) {
    take_scales(nxt);
    take_ids(after);
    for (int i = 0; i < cur.n; ++i, ++tc) {
      if (tc >= kDescSlots && !wait_or_abort(ring->empty_bar(tc), ring->parity(tc) ^ 1, abort_flag, status)) { ok = false; break; }
      TileDesc& e = ring->desc[tc % kDescSlots];
      if (ti == i) {
        const bool none = cur.vs >= 0.f && cur.vs < fp8::kMinValueScale;
        const float lv = none ? kMinLv : cur.vs > 0.f ? __log2f(cur.vs) : __int_as_float(0x7fc00000);
        e.blk[j] = none ? ~cur.blk : cur.blk;  // (the complement: its V is zero)
        e.ks[j] = cur.ks;
        e.lv[j] = lv;
        e.inv[j] = fast_exp2(-lv);
        if (j == 0) {
          e.nb = cur.nb; e.ntok = cur.ntok; e.kvh = cur.kvh;
          e.row0 = cur.row0; e.head = cur.head; e.nrows = i == 0 ? cur.nrows : 0;
        }
      }
      mbar_arrive(ring->full_bar(tc));
    }
    if (!ok) break;
    cur = nxt;
    nxt = after;
  }
  if (ok && (tc < kDescSlots || wait_or_abort(ring->empty_bar(tc), ring->parity(tc) ^ 1, abort_flag, status))) {
    if (lane == 0) ring->desc[tc % kDescSlots].nb = 0;
    mbar_arrive(ring->full_bar(tc));
  }
}

// Converter warp pw of kConvWarps: V of blocks pw and pw + 4 of every kv tile of this CTA. As soon as a block is converted its
// registers take the codes of the next tile's, which arrive while the next slot is waited for. Every thread arrives on the
// slot's full barrier. Operand layout as in the 16-bit kernels: per block [d][16 tok], 32-byte rows, 32-byte swizzle; a lane turns
// a row. Codes behind the item's last token become 0.
__device__ __forceinline__ void convert_v(const AttnDev& d, int pw, int lane, uint8_t* slots, uint32_t bars0, TileRing* ring,
                                          volatile int* abort_flag, int32_t* status) {
  constexpr int kPer = kTileBlocks / kConvWarps;
  const uint8_t* cache = reinterpret_cast<const uint8_t*>(d.value_cache) + lane * 16;
  uint4 v[kPer][4];
  auto fetch_block = [&](const TileDesc& e, uint4 (&to)[4], int j) {
    if (j < e.nb) {
      const int b = e.blk[j];
      const uint4* src = reinterpret_cast<const uint4*>(cache + (size_t)(b < 0 ? ~b : b) * d.kv_block_stride + (size_t)e.kvh * d.kv_head_stride);
#pragma unroll
      for (int k = 0; k < 4; ++k) to[k] = src[k * 32];
    }
  };
  if (!wait_or_abort(ring->full_bar(0), 0, abort_flag, status, 50)) return;
#pragma unroll
  for (int u = 0; u < kPer; ++u) fetch_block(ring->desc[0], v[u], pw + u * kConvWarps);
  for (uint32_t tc = 0;; ++tc) {
    const TileDesc& cur = ring->desc[tc % kDescSlots];
    const int nb = cur.nb;
    if (nb == 0) break;
    const int s = tc & 1;
    if (!wait_or_abort(bars0 + (kBarEmptyV + s) * 8, ((tc >> 1) & 1) ^ 1, abort_flag, status, 50)) break;
    if (pw == 0 && lane == 0 && tc >= 2) mbar_arrive(ring->empty_bar(tc - 2));
    if (!wait_or_abort(ring->full_bar(tc + 1), ring->parity(tc + 1), abort_flag, status, 50)) break;
    const TileDesc& nxt = ring->desc[(tc + 1) % kDescSlots];
    uint8_t* slot = slots + s * kRingBytes;
#pragma unroll
    for (int u = 0; u < kPer; ++u) {
      const int j = pw + u * kConvWarps;
      if (j < nb) {
        const int left = cur.blk[j] < 0 ? 0 : cur.ntok - j * kB;  // tokens of the block that count
        if (left < kB) {
          uint32_t m[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int n = left - 4 * i;
            m[i] = n <= 0 ? 0u : n >= 4 ? 0xffffffffu : (1u << (8 * n)) - 1u;
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) v[u][k] = make_uint4(v[u][k].x & m[0], v[u][k].y & m[1], v[u][k].z & m[2], v[u][k].w & m[3]);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = k * 32 + lane;  // d
          const uint4 w = v[u][k];
          uint8_t* p = slot + j * kBlkBytes + row * 32;
          const int flip = ((row >> 2) & 1) << 4;  // 32-byte swizzle: the halves swap in rows 4..7 of every 8
          *reinterpret_cast<uint4*>(p + flip) = make_uint4(fp8::to_half2(w.x), fp8::to_half2_high(w.x), fp8::to_half2(w.y), fp8::to_half2_high(w.y));
          *reinterpret_cast<uint4*>(p + (flip ^ 16)) = make_uint4(fp8::to_half2(w.z), fp8::to_half2_high(w.z), fp8::to_half2(w.w), fp8::to_half2_high(w.w));
        }
      }
      fetch_block(nxt, v[u], j);
    }
    fence_proxy_async_smem();
    mbar_arrive(bars0 + (kBarFullV + s) * 8);
  }
}

// The warp that copies K and asks for Q. K: per-thread 16-byte async copies, the 256-byte chunk rows of the tile's blocks side by
// side ([d chunk][block][16 tok][16 B]: one no-swizzle operand of up to 128 tokens). Q: with the first tile of a segment, the parts of its
// row tiles, [part][128 rows][128 B] with the 128-byte swizzle; rows beyond the batch read as zero, rows beyond the item are
// other queries whose results are never stored.
template <typename T>
__device__ __forceinline__ void copy_k_and_q(const AttnDev& d, int lane, uint32_t sQ, uint32_t sK, uint32_t bars0, TileRing* ring,
                                             const CUtensorMap* pmap, volatile int* abort_flag, int32_t* status) {
  constexpr int kNum = QParts<T>::kNum;
  const uint8_t* kc = reinterpret_cast<const uint8_t*>(d.key_cache);
  uint32_t segx[2] = {0, 0};
  auto bar = [&](int i) { return bars0 + i * 8; };
  for (uint32_t tc = 0;; ++tc) {
    const int s = tc & 1;
    if (!wait_or_abort(ring->full_bar(tc), ring->parity(tc), abort_flag, status, 50)) break;
    const TileDesc& e = ring->desc[tc % kDescSlots];
    const int nb = e.nb, nrows = e.nrows, row0 = e.row0, head = e.head;  // (read before K is let go: the slot is written anew behind its products)
    if (nb == 0) break;
    if (!wait_or_abort(bar(kBarEmptyK + s), ((tc >> 1) & 1) ^ 1, abort_flag, status, 50)) break;
    for (int j = 0; j < nb; ++j) {
      const int b = e.blk[j];
      const uint8_t* src = kc + (size_t)(b < 0 ? ~b : b) * d.kv_block_stride + (size_t)e.kvh * d.kv_head_stride + lane * 16;
      const uint32_t dst = sK + s * kRingK + (lane >> 4) * (kTileBlocks * 256) + j * 256 + (lane & 15) * 16;
#pragma unroll
      for (int k = 0; k < 4; ++k) cp_async16(dst + k * 2 * (kTileBlocks * 256), src + k * 512);
    }
    cp_async_arrive_noinc(bar(kBarFullK + s));
    if (nrows > 0) {
      const int nsub = nrows > 128 ? 2 : 1;
      bool ok = true;
      for (int x = 0; x < nsub && ok; ++x) {
        if (segx[x] > 0 && !wait_or_abort(bar(kBarQFree + x), (segx[x] - 1) & 1, abort_flag, status, 50)) { ok = false; break; }
        if (lane == 0) {
          mbar_arrive_expect_tx(bar(kBarQ + x), kNum * kPartBytes);
#pragma unroll
          for (int p = 0; p < kNum; ++p)
            tma_load_q(sQ + (x * kNum + p) * kPartBytes, pmap, bar(kBarQ + x), 0, row0 + x * 128, p * d.num_heads + head);
        }
        ++segx[x];
        __syncwarp();
      }
      if (!ok) break;
    }
  }
  cp_async_wait_all();
  for (int x = 0; x < 2; ++x)  // (already complete but when a wait gave up)
    if (segx[x] > 0) (void)mbar_wait_bounded(bar(kBarQ + x), (segx[x] - 1) & 1);
}

// The two passes of one softmax thread over its row of S (128 scores in tensor memory, read in chunks of 32 columns, the next
// chunk in flight while one is worked on; the chunk loops are kept rolled so that the hot code stays small enough for the
// instruction cache). kMasked: only the first `vis` columns count.
// Maximum of the logits with their blocks' offsets; `top` is that of the logits alone. mul: c / f of the row.
template <bool kMasked>
__device__ __forceinline__ float row_max128(uint32_t tmem_s, int vis, const TileDesc& e, float mul, float& top) {
  uint32_t a[32], b[32];
  float mx = -INFINITY;
  auto two_blocks = [&](const uint32_t* v, int c) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float m0 = -INFINITY, m1 = -INFINITY;
      if (!kMasked) {
#pragma unroll
        for (int i = 16 * h; i < 16 * h + 16; i += 4) {
          m0 = max3(m0, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
          m1 = max3(m1, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
        }
      } else {
#pragma unroll
        for (int i = 16 * h; i < 16 * h + 16; i += 2) {
          m0 = fmaxf(m0, 32 * c + i < vis ? __uint_as_float(v[i]) : -INFINITY);
          m1 = fmaxf(m1, 32 * c + i + 1 < vis ? __uint_as_float(v[i + 1]) : -INFINITY);
        }
      }
      const float lg = fmaxf(m0, m1) * (e.ks[2 * c + h] * mul);  // (no visible column: -inf, or NaN, which the maxima drop)
      top = fmaxf(top, lg);
      mx = fmaxf(mx, lg + e.lv[2 * c + h]);
    }
  };
  tmem_ld32(tmem_s, a);
#pragma unroll 1
  for (int c = 0; c < 4; c += 2) {
    tmem_wait_ld();
    tmem_ld32(tmem_s + 32 * (c + 1), b);
    two_blocks(a, c);
    tmem_wait_ld();
    if (c == 0) tmem_ld32(tmem_s + 64, a);
    two_blocks(b, c + 1);
  }
  return mx;
}
// P chunk c (tokens [32c, 32c + 32)) goes to columns [16c, 16c + 16) of the row's S columns, which the chunks read so far
// cover; the chunk in flight lies above them. Returns the row sum (times 2^kShift, relative to M).
template <bool kMasked>
__device__ __forceinline__ float row_exp128(uint32_t tmem_s, int vis, const TileDesc& e, float mul, float m) {
  uint32_t a[32], b[32], pk[16];
  float sum = 0.f;
  auto two_blocks = [&](const uint32_t* v, int c) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float cs = e.ks[2 * c + h] * mul, add = e.lv[2 * c + h] - m + kShift;
      float part[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 16 * h; i < 16 * h + 16; i += 2) {
        float e0 = __uint_as_float(v[i]), e1 = __uint_as_float(v[i + 1]);
        fma_pair(e0, e1, cs, add);
        e0 = fast_exp2(e0);
        e1 = fast_exp2(e1);
        if (kMasked) {
          e0 = (32 * c + i < vis) ? e0 : 0.f;
          e1 = (32 * c + i + 1 < vis) ? e1 : 0.f;
        }
        part[(i >> 1) & 1] += e0 + e1;
        pk[i >> 1] = Pack<__half>::two(e0, e1);
      }
      sum = fmaf(part[0] + part[1], e.inv[2 * c + h], sum);
    }
    tmem_st16(tmem_s + 16 * c, pk);
  };
  tmem_ld32(tmem_s, a);
#pragma unroll 1
  for (int c = 0; c < 4; c += 2) {
    tmem_wait_ld();
    tmem_ld32(tmem_s + 32 * (c + 1), b);
    two_blocks(a, c);
    tmem_wait_ld();
    if (c == 0) tmem_ld32(tmem_s + 64, a);
    two_blocks(b, c + 1);
  }
  return sum;
}

// State of one softmax thread = one query row: reference maximum and sum (base-2 domain), the
// exact maximum seen.
struct RowState {
  float m_run, l_run, m_true;
};

// A lone row tile of a shared prefix is worked on by both softmax groups and issuers: group x takes its kv tiles x, x + 2, ... with
// Q_0, S_x and O_x, and group 0 joins the two O in the epilogue. By one group alone each tile waits for the one before it: S,
// softmax, P.V, 3.4 us against 2.3 (64 rows over 65536 tokens, 32 heads). The last row tiles of prefills stay with group 0:
// they take what a pair takes, and the shares of the CTAs, which count a tile of either as one, stay even (16 prefills of 256 to
// 1024 tokens and 240 decodes over 2048 tokens: 1160 us with both groups, 1015 with one).
// (kSplit: the call has no prefills.)
__device__ __forceinline__ int first_tile(bool pair, bool split, int x, int n) { return (pair || x == 0) ? 0 : split ? 1 : n; }

template <typename T, bool kSplit>
__global__ void __launch_bounds__(kThreads, 1)
dense_fp8_kernel(const AttnDev d, const __grid_constant__ CUtensorMap pmap, const __grid_constant__ CUtensorMap amap,
                 const __grid_constant__ CUtensorMap omap) {
  using L = Layout<T>;
  constexpr int kNum = QParts<T>::kNum;
  extern __shared__ __align__(1024) uint8_t smem[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::kOffBars);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::kOffBars + kNumBars * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::kOffBars + kNumBars * 8 + 8);
  int32_t* status = &d.hdr[kHdrStatus];
  TileRing* tiles = reinterpret_cast<TileRing*>(smem + L::kOffRing);
  const uint32_t bars0 = smem_u32(bars);
  auto bar = [&](int i) { return bars0 + i * 8; };

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar(kBarFullK + s), 32);  // every thread of the warp that copies K arrives
      mbar_init(bar(kBarEmptyK + s), 2);  // one release per MMA issuer
      mbar_init(bar(kBarFullV + s), 32 * kConvWarps);
      mbar_init(bar(kBarEmptyV + s), 2);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(bar(kBarS + x), 1);
      mbar_init(bar(kBarP + x), kGroupThreads);
      mbar_init(bar(kBarPV + x), 1);
      mbar_init(bar(kBarQ + x), 1);
      mbar_init(bar(kBarQFree + x), x == 0 ? 2 : 1);  // (Q_0: both issuers of a lone row tile)
      mbar_init(bar(kBarODrained + x), kGroupThreads);
      mbar_init(bar(kBarTurn + x), 1);
      mbar_init(bar(kBarGroup + x), kGroupThreads);
    }
    mbar_init(bar(kBarHand), kGroupThreads);
    tiles->init();
    *abort_flag = 0;
    mbar_fence_init();
    fence_proxy_async_smem();
  }
  if (warp == 14) tmem_alloc(smem_u32(tmem_slot), kTmemCols);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Everything above overlapped the previous kernel in the stream; from here on its results (new
  // KV in the cache, the work lists) are read. Then let the suffix kernel start on the other SMs.
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem_base = *tmem_slot;

  const uint32_t sQ = smem_u32(smem + L::kOffQ), sK0 = smem_u32(smem + L::kOffK), sV0 = smem_u32(smem + L::kOffV);
  // CTAs beyond the planner's share own no tiles and fall straight through to the teardown. Every role makes its own walker: as
  // one object of them all, made before the roles part, the compiler kept it in local memory.
  auto segments = [&]() { return SegmentWalker(d, blockIdx.x, min(dense_ctas_of(d), (int)gridDim.x)); };
  Segment sg;

  if (warp >= 8 && warp < 8 + kConvWarps) {
    regs_fewer<kRegsConvert>();
    convert_v(d, warp - 8, lane, smem + L::kOffV, bars0, tiles, abort_flag, status);
  } else if (warp >= 12) {
  regs_fewer<kRegsIssue>();  // (one place for the whole warpgroup)
  if (warp == 12) {
    copy_k_and_q<T>(d, lane, sQ, sK0, bars0, tiles, &pmap, abort_flag, status);
  } else if (warp == 15) {
    SegmentWalker walk = segments();
    list_tiles(d, walk, lane, tiles, abort_flag, status);
  } else {
    // ======================= MMA issuer of row tile x =======================
    // The chains and turns of dense_pair.cu: per kv tile i of a segment
    //   P_x.V(i)       once P_x(i) is written and V(i) has landed (i = 0: the last epilogue has drained O_x)
    //   Q_x.K^T(i + 1) once K(i + 1) has landed; it overwrites S_x / P_x, and follows P_x.V(i) in this
    //                  thread's program order, which the tensor pipe keeps
    // and on pair items the two issuers issue in turns. Operands (descriptors built once):
    //   Q_x: [part][row][128 B], 128-byte swizzle            -> SBO 1024 (8-row groups); a k-step: 32 bytes inside the atom
    //   K:   [16-byte d chunk][blk][tok][16 B], no swizzle   -> SBO 128 (8-token groups), LBO 2048 (d chunks)
    //   V:   per block [d][16 tok], 32-byte rows, 32-byte swizzle -> SBO 256 (8-row groups)
    //   P_x: tensor memory, lane = row, tokens packed two per column -> block j = columns [8j, 8j + 8)
    const int x = warp - 13;
    SegmentWalker walk = segments();
    constexpr uint32_t kIdescPV = make_idesc(128, kD, false);
    const uint64_t desc_q = smem_desc(sQ + x * kNum * kPartBytes, 16, 1024, 2), desc_q0 = smem_desc(sQ, 16, 1024, 2);
    const uint64_t desc_k0 = smem_desc(sK0, 2048, 128, 0), desc_k1 = smem_desc(sK0 + kRingK, 2048, 128, 0);
    const uint64_t desc_v0 = smem_desc(sV0, 16, 256, 6), desc_v1 = smem_desc(sV0 + kRingBytes, 16, 256, 6);
    const uint32_t tmem_s = tmem_base + x * 128, tmem_o = tmem_base + 256 + x * 128;
    uint32_t tc = 0, tcx = 0, seg = 0, pairs = 0, turns = 0;  // turns: kv tiles of pair items so far
    bool ok = true;
    while (ok && walk.next(sg)) {
      const int n = sg.t1 - sg.t0;
      const bool pair = sg.it.nrows > 128;
      const bool split = kSplit && !pair;
      const int first = first_tile(pair, split, x, n), step = split ? 2 : 1;
      const uint64_t bq = pair ? desc_q : desc_q0;
      // S_x = Q_x . K(i)^T (the caller has seen K(i) land); lane 0 only
      auto qk_mmas = [&](int i) {
        const int s = (tc + i) & 1;
        // fp32 += e4m3 . e4m3
        const uint32_t idesc = (1u << 4) | ((uint32_t)(dense_tile_view(d, sg.it, sg.t0 + i).nb * (kB / 8)) << 17) | ((uint32_t)(128 >> 4) << 24);
        const uint64_t bk = s ? desc_k1 : desc_k0;
#pragma unroll
        for (int p = 0; p < kNum; ++p)
#pragma unroll
          for (int kk = 0; kk < kD / 32; ++kk)
            mma_f8(tmem_s, bq + ((p * kPartBytes + kk * 32) >> 4), bk + ((kk * 2 * 2048) >> 4), idesc, (p | kk) ? 1u : 0u);
      };
      auto qk_release = [&](int i) {
        mma_commit(bar(kBarS + x));
        mma_commit(bar(kBarEmptyK + ((tc + i) & 1)));
        if (i + step >= n) {  // this issuer's last Q.K^T of the segment
          mma_commit(bar(kBarQFree + (pair ? x : 0)));
          if (x == 0 && !split) mma_commit(bar(kBarQFree));  // (the other issuer does not read Q_0)
        }
      };
      // A wait names its phase by parity alone, so nobody may be two phases away from what it waits for. Ring slots take a release
      // of each issuer for that reason, of a tile that is the other's too, as soon as it has landed.
      auto full_k = [&](int i) { return wait_or_abort(bar(kBarFullK + ((tc + i) & 1)), ((tc + i) >> 1) & 1, abort_flag, status); };
      auto full_v = [&](int i) { return wait_or_abort(bar(kBarFullV + ((tc + i) & 1)), ((tc + i) >> 1) & 1, abort_flag, status); };
      auto pass_k = [&](int i) {
        if (!full_k(i)) return false;
        if (lane == 0) mbar_arrive(bar(kBarEmptyK + ((tc + i) & 1)));
        return true;
      };
      auto pass_v = [&](int i) {
        if (!full_v(i)) return false;
        if (lane == 0) mbar_arrive(bar(kBarEmptyV + ((tc + i) & 1)));
        return true;
      };
      if (!split && !pair && x == 1) {  // nothing for this issuer but its releases
        for (int i = 0; i < n && ok; ++i) ok = pass_k(i) && pass_v(i);
        tc += n;
        ++seg;
        continue;
      }
      if (!wait_or_abort(bar(kBarQ + (pair ? x : 0)), (pair && x == 1 ? pairs : seg) & 1, abort_flag, status)) { ok = false; break; }
      if (split && first >= n && lane == 0) mbar_arrive(bar(kBarQFree));  // (a lone row tile of one kv tile: nothing for this issuer)
      if (split && x == 1 && !pass_k(0)) { ok = false; break; }
      if (first < n) {
        if (!full_k(first)) { ok = false; break; }
        fence_proxy_async_smem();  // K was written by per-thread async copies (generic proxy)
        tc_fence_after();
        if (lane == 0) {
          qk_mmas(first);
          qk_release(first);
        }
        __syncwarp();
      }
      if (split && x == 1 && !pass_v(0)) { ok = false; break; }
      for (int i = first; i < n; i += step, ++tcx) {
        const uint32_t c = tc + i;
        const int s = c & 1;
        const bool more = i + step < n;
        // what arrives early first: V(i), the next K; then P_x(i), which the chain hangs on, and the drained O_x (behind P_x: an
        // issuer without a tile in the last segment knows by it that the segment before that is over)
        if (!full_v(i)) { ok = false; break; }
        if (!split && more && !full_k(i + 1)) { ok = false; break; }
        if (split && i + 1 < n && !pass_k(i + 1)) { ok = false; break; }  // the other issuer's; its slot is for the K after the next
        fence_proxy_async_smem();
        if (!wait_or_abort(bar(kBarP + x), tcx & 1, abort_flag, status)) { ok = false; break; }
        if (i == first && seg > 0 && !wait_or_abort(bar(kBarODrained + x), (seg - 1) & 1, abort_flag, status)) { ok = false; break; }
        if (pair && (x == 1 || turns > 0) &&
            !wait_or_abort(bar(kBarTurn + (x ^ 1)), (x == 1 ? turns : turns - 1) & 1, abort_flag, status)) { ok = false; break; }
        tc_fence_after();
        if (lane == 0) {
          const int nb = dense_tile_view(d, sg.it, sg.t0 + i).nb;
          const uint64_t bv = s ? desc_v1 : desc_v0;
#pragma unroll
          for (int j = 0; j < kTileBlocks; ++j)
            if (j < nb) mma_f16_ts(tmem_o, tmem_s + j * 8, bv + j * (kBlkBytes >> 4), kIdescPV, (i > first || j > 0) ? 1u : 0u);
          if (!split && more) qk_mmas(i + 1);  // behind P_x.V(i) in the pipe: it overwrites S_x / P_x
          if (pair) mbar_arrive(bar(kBarTurn + x));
          // (before the next S is announced: a softmax thread waits for this phase only with its last tile)
          mma_commit(bar(kBarPV + x));
          if (!split && more) qk_release(i + 1);
          mma_commit(bar(kBarEmptyV + s));
        }
        if (pair) ++turns;
        __syncwarp();
        if (split) {
          // the K of this issuer's next tile comes into the slot of this one
          if (more) {
            if (!full_k(i + 2)) { ok = false; break; }
            fence_proxy_async_smem();
            tc_fence_after();
            if (lane == 0) {
              qk_mmas(i + 2);
              qk_release(i + 2);
            }
            __syncwarp();
          }
          if (i + 1 < n && !pass_v(i + 1)) { ok = false; break; }
        }
      }
      if (!ok) break;
      tc += n;
      ++seg;
      if (pair) ++pairs;
    }
  }
  } else {
    regs_more<kRegsSoftmax>();
    SegmentWalker walk = segments();
    // ======================= softmax + epilogue: one thread per row =======================
    const int x = warp >> 2;                      // row tile of this thread's group
    const int r = (warp & 3) * 32 + lane;         // row inside the tile = TMEM lane
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t tmem_s = tmem_base + x * 128 + lane_base;
    const uint32_t tmem_o = tmem_base + 256 + x * 128 + lane_base;
    uint8_t* const stage = smem + L::kOffStage + x * kStageBytes;
    const bool issuer = (r == 0);                 // issues the group's TMA stores
    uint32_t tc = 0, tcx = 0, seg = 0, hands = 0, group_use = 0;  // hands: lone row tiles so far
    bool ok = true, store_pending = false;
    float* const hand = reinterpret_cast<float*>(smem + L::kOffStage + kStageBytes);  // [3][128], in group 1's staging buffer
    auto group_sync = [&]() -> bool {
      mbar_arrive(bar(kBarGroup + x));
      return wait_or_abort(bar(kBarGroup + x), (group_use++) & 1, abort_flag, status);
    };
    // the staging buffer may be written: the TMA store that read it last has done so
    auto stage_begin = [&]() -> bool {
      if (issuer && store_pending) {
        bulk_wait_read();
        store_pending = false;
      }
      return group_sync();
    };
    while (ok && walk.next(sg)) {
      const DnItem& it = sg.it;
      const bool pair = it.nrows > 128;
      const bool split = kSplit && !pair;
      const int first = sg.t0 + first_tile(pair, split, x, sg.t1 - sg.t0), step = split ? 2 : 1;
      const int qrow = (pair ? x * 128 : 0) + r;  // row inside the item
      RowState st = {-INFINITY, 0.f, -INFINITY};
      const float mul = d.q_mul[(size_t)sg.head * d.num_rows + min(it.row0 + qrow, d.num_rows - 1)];
      for (int t = first; t < sg.t1; t += step, ++tcx) {
        const uint32_t tc_t = tc + (t - sg.t0);
        const DenseTileView tv = dense_tile_view(d, it, t);
        // columns this row may attend: all of the tile's tokens, or (causal tile) the first causal0 + row
        const int vis = tv.causal ? min(tv.ntok, tv.causal0 + qrow) : tv.ntok;
        const bool all_valid = __all_sync(0xffffffffu, vis >= kTileTok);
        if (!wait_or_abort(bar(kBarS + x), tcx & 1, abort_flag, status)) { ok = false; break; }
        tc_fence_after();
        // ---- row maximum ----
        if (!wait_or_abort(tiles->full_bar(tc_t), tiles->parity(tc_t), abort_flag, status)) { ok = false; break; }
        const TileDesc& e = tiles->desc[tc_t % kDescSlots];
        float top = -INFINITY;
        const float mx = all_valid ? row_max128<false>(tmem_s, vis, e, mul, top) : row_max128<true>(tmem_s, vis, e, mul, top);
        // Lazy reference maximum: the row keeps its reference m_run until a tile exceeds it by more
        // than 2^kTau; P then holds values up to 2^kTau instead of 1, which fp16/bf16 and the fp32
        // accumulators absorb, and O in TMEM is rescaled only on those rare jumps. (m, l, O) stay
        // mutually consistent, which is all the merge needs.
        st.m_true = fmaxf(st.m_true, top);
        const bool grow = mx > st.m_run + kTau;  // true on the first tile a row sees a token in
        const float alpha = grow ? fast_exp2(st.m_run - mx) : 1.f;
        if (t > first && __any_sync(0xffffffffu, grow && st.l_run > 0.f)) {
          // rescale this warp's O rows in TMEM (the previous tile's P.V, which accumulated into
          // them, retired before this tile's S was produced)
          if (!wait_or_abort(bar(kBarPV + x), (tcx - 1) & 1, abort_flag, status)) { ok = false; break; }
          tc_fence_after();
#pragma unroll 1
          for (int c0 = 0; c0 < kD; c0 += 32) {
            uint32_t o[32];
            tmem_ld32(tmem_o + c0, o);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
            tmem_st32(tmem_o + c0, o);
          }
        }
        st.l_run *= alpha;
        st.m_run = grow ? mx : st.m_run;
        // ---- P = 2^(s - m) into the row's P columns, and the row sum ----
        st.l_run += all_valid ? row_exp128<false>(tmem_s, vis, e, mul, st.m_run) : row_exp128<true>(tmem_s, vis, e, mul, st.m_run);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(bar(kBarP + x));
      }
      if (!ok) break;
      tc += sg.t1 - sg.t0;
      // ---- epilogue: O_x rows -> un-normalised partials, or the finished output rows ----
      if (sg.t1 > first && !wait_or_abort(bar(kBarPV + x), (tcx - 1) & 1, abort_flag, status)) { ok = false; break; }
      tc_fence_after();
      if (!pair) {
        const bool both = split && sg.t1 - sg.t0 > 1;
        if (x == 1) {
          // hand over: O_1 stays where it is, lane for lane beside O_0. The last hand-over has been read by now.
          if (seg > 0 && !wait_or_abort(bar(kBarODrained + 1), (seg - 1) & 1, abort_flag, status)) { ok = false; break; }
          if (!stage_begin()) { ok = false; break; }
          hand[r] = st.m_run;
          hand[128 + r] = st.l_run;
          hand[256 + r] = st.m_true;
          tc_fence_before();
          mbar_arrive(bar(kBarHand));
          ++seg;
          continue;
        }
        if (!wait_or_abort(bar(kBarHand), hands & 1, abort_flag, status)) { ok = false; break; }
        ++hands;
        tc_fence_after();
        if (both) {
          const float m1 = hand[r], l1 = hand[128 + r];
          st.m_true = fmaxf(st.m_true, hand[256 + r]);
          const float m = fmaxf(st.m_run, m1), base = m == -INFINITY ? 0.f : m;
          const float a0 = fast_exp2(st.m_run - base), a1 = fast_exp2(m1 - base);
          uint32_t o[32], q[32];
#pragma unroll 1
          for (int c0 = 0; c0 < kD; c0 += 32) {
            tmem_ld32(tmem_o + c0, o);
            tmem_ld32(tmem_o + 128 + c0, q);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 32; ++i)
              o[i] = __float_as_uint(fmaf(__uint_as_float(q[i]), a1, __uint_as_float(o[i]) * a0));
            tmem_st32(tmem_o + c0, o);
          }
          tmem_wait_st();
          st.l_run = fmaf(l1, a1, st.l_run * a0);
          st.m_run = m;
        }
      }
      st.m_true = told_max(st.m_true, st.l_run);
      const int nrows_x = min(128, it.nrows - (pair ? x * 128 : 0));
      const bool row_ok = r < nrows_x;
      const int row = it.row0 + qrow;
      const size_t slot = partial_slot(d, row_ok ? row : it.row0, dense_part_base(d, it) + sg.part, sg.head);
      // re-base the partial on the exact row maximum; a row that saw no token in this CTA's tiles
      // (causal items) leaves the empty partial (-inf, 0, 0)
      const float fix = (st.m_true == -INFINITY) ? 0.f : fast_exp2(st.m_run - kShift - st.m_true);
      // Finished rows: this CTA holds every kv tile of (item, head) and the rows have no other
      // partial, so O / l IS the attention output; it goes out in the model's type and the merge
      // skips these rows (same test on its side: one dense partial, no suffix, the item's flag).
      const bool direct = dense_direct_ok(d, it) && sg.t0 == 0 && sg.t1 == it.nt;
      const bool by_tma = (nrows_x == 128) && d.acc_tma;
      if (direct) {
        const float inv = (st.l_run > 0.f) ? 1.f / st.l_run : 0.f;
        T* orow = reinterpret_cast<T*>(d.out) + (size_t)(row_ok ? row : it.row0) * d.out_stride + (size_t)sg.head * kD;
#pragma unroll 1
        for (int c0 = 0; c0 < kD; c0 += 64) {
          uint32_t v[64];
          tmem_ld32(tmem_o + c0, v);
          tmem_ld32(tmem_o + c0 + 32, v + 32);
          tmem_wait_ld();
          uint32_t h[32];
#pragma unroll
          for (int i = 0; i < 32; ++i)
            h[i] = Pack<T>::two(__uint_as_float(v[2 * i]) * inv, __uint_as_float(v[2 * i + 1]) * inv);
          if (by_tma) {
            // staging: [128 rows][128 B], 16-byte chunks swizzled by the row; one tiled store per half
            if (!stage_begin()) { ok = false; break; }
            uint8_t* rowp = stage + r * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(rowp + ((i ^ (r & 7)) << 4)) = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
            fence_proxy_async_smem();
            if (!group_sync()) { ok = false; break; }
            if (issuer) {
              tma_store_out(&omap, smem_u32(stage), c0, sg.head, it.row0 + x * 128);
              bulk_commit_group();
              store_pending = true;
            }
          } else if (row_ok) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<uint4*>(orow + c0 + 8 * i) = make_uint4(h[4 * i], h[4 * i + 1], h[4 * i + 2], h[4 * i + 3]);
          }
        }
      } else {
#pragma unroll 1
        for (int c0 = 0; c0 < kD; c0 += 32) {
          uint32_t v[32];
          tmem_ld32(tmem_o + c0, v);
          tmem_wait_ld();
          if (by_tma) {
            // Full row tile: its 128 partial rows are contiguous in the workspace. Staged as
            // [128 rows][32 floats] in the 128-byte-swizzled layout and written by one tiled store;
            // a thread's own stores would touch 32 separate lines per instruction.
            if (!stage_begin()) { ok = false; break; }
            uint8_t* rowp = stage + r * 128;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              *reinterpret_cast<float4*>(rowp + ((i ^ (r & 7)) << 4)) =
                  make_float4(__uint_as_float(v[4 * i]) * fix, __uint_as_float(v[4 * i + 1]) * fix,
                              __uint_as_float(v[4 * i + 2]) * fix, __uint_as_float(v[4 * i + 3]) * fix);
            fence_proxy_async_smem();
            if (!group_sync()) { ok = false; break; }
            if (issuer) {
              const size_t slot0 = partial_slot(d, it.row0 + x * 128, dense_part_base(d, it) + sg.part, sg.head);
              tma_store_acc(&amap, smem_u32(stage), c0, (int)slot0);
              bulk_commit_group();
              store_pending = true;
            }
          } else if (row_ok) {
            float4* dst = reinterpret_cast<float4*>(d.acc + slot * kD + c0);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              dst[i] = make_float4(__uint_as_float(v[4 * i]) * fix, __uint_as_float(v[4 * i + 1]) * fix,
                                   __uint_as_float(v[4 * i + 2]) * fix, __uint_as_float(v[4 * i + 3]) * fix);
          }
        }
        if (ok && row_ok) d.ml[slot] = make_float2(st.m_true, st.l_run * fix);
      }
      if (!ok) break;
      tc_fence_before();
      if (!pair) mbar_arrive(bar(kBarODrained + 1));
      mbar_arrive(bar(kBarODrained + x));
      ++seg;
    }
    if (issuer) bulk_wait_all();  // stores of the last segment have left shared memory and landed
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 14) {
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

// The register shares only add up if the block is launched with kRegsLaunch registers a thread: a build in which it is not must
// not run (the warps that ask for more would wait for good). Asked once per kernel.
template <auto kKernel> cudaError_t check_register_shares() {
  static const cudaError_t verdict = [] {
    cudaFuncAttributes a;
    const cudaError_t e = cudaFuncGetAttributes(&a, reinterpret_cast<const void*>(kKernel));
    if (e != cudaSuccess) return e;
    return a.numRegs == kRegsLaunch ? cudaSuccess : cudaErrorInvalidConfiguration;
  }();
  return verdict;
}

template <typename T, bool kSplit>
cudaError_t launch_dense(const AttnDev& d, const CUtensorMap& pmap, const CUtensorMap& amap, const CUtensorMap& omap, cudaStream_t s) {
  auto kfn = dense_fp8_kernel<T, kSplit>;
  cudaError_t e = cudaFuncSetAttribute(kfn, cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<T>::kSmemBytes);
  if (e == cudaSuccess) e = check_register_shares<dense_fp8_kernel<T, kSplit>>();
  if (e != cudaSuccess) return e;
  return launch_kernel(kfn, d.num_sms, kThreads, Layout<T>::kSmemBytes, s, true, d, pmap, amap, omap);
}

template <typename T>
cudaError_t launch_t(const AttnDev& d, const CUtensorMap& pmap, const CUtensorMap& amap, const CUtensorMap& omap, cudaStream_t s) {
  const dim3 grid((unsigned)d.num_rows, (unsigned)((d.num_heads + 8 * kPartsHeads - 1) / (8 * kPartsHeads)));
  const cudaError_t e = launch_kernel(query_parts_kernel<T>, grid, 256, 0, s, true, d);
  if (e != cudaSuccess) return e;
  return d.num_segments == 0 ? launch_dense<T, true>(d, pmap, amap, omap, s) : launch_dense<T, false>(d, pmap, amap, omap, s);
}

}  // namespace

cudaError_t launch_dense_fp8(const AttnDev& d, int dtype, const CUtensorMap& pmap, const CUtensorMap& amap, const CUtensorMap& omap,
                             cudaStream_t s) {
  return dtype == PB_F16 ? launch_t<__half>(d, pmap, amap, omap, s) : launch_t<__nv_bfloat16>(d, pmap, amap, omap, s);
}

}  // namespace pb
