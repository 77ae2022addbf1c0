// Fill of the 8-bit paged cache, and rows out of it again.
//
// The scale of a (block, head) depends on all tokens that the call brings to the block, and a scale that grows changes the
// block's other cells, so a block has one owner per call: the window (16 consecutive entries of slot_mapping) that holds the
// first of its tokens. Which tokens those are, member[offset] = the last token of the list with that slot, a window finds in
// one of two ways. Up to kScanTokens tokens it reads the whole list. Beyond, a table with an entry per slot says so, written
// by a kernel in front (fp8_link). The table lives in scratch that nobody clears: an entry counts only if it names a token
// of this call whose slot is that slot, and every slot that has a token has been written.
//
// A tile of 16 tokens x 64 elements is spread over a warp as 4 tokens x 8 elements a lane: rows are read and written in 128-byte
// runs, K in 8-byte pieces, and V, whose codes lie the other way round ([d][token]), after a transposition in registers (4 x 4
// bytes inside a lane, then 4 x 4 words between four lanes) as 16 bytes a lane.
//
// Bound by memory where it is large: fill and gather of a batch with 16 prefills and 240 decodes (9.4k rows, 32 heads of 128, bf16)
// 135 us, 3.6 TB/s of the 6.5 a copy reaches; what is lost lies in the latency of short CTAs and in the conversions of the gather.
// Small calls are bound by latency: slots, scales and rows, store: 5 us each.
//
// Reference counterpart of the unquantised fill: reshape_and_cache_kernel (3rdparty/vllm/csrc/cache_kernels.cu:142-182).
#include "common.cuh"
#include "fp8.cuh"

namespace pb {
namespace {

__device__ __forceinline__ long long slot_at(const void* slots, int is64, long long t) {
  return is64 ? reinterpret_cast<const long long*>(slots)[t] : (long long)reinterpret_cast<const int*>(slots)[t];
}

struct Fp8Rows {  // what the fill and the gather walk; strides in elements
  uint8_t* key;
  uint8_t* value;
  uint8_t* kcache;
  uint8_t* vcache;
  float* kscale;
  float* vscale;
  const void* slots;
  int* member;
  long long tokens, key_stride, value_stride, kbs, khs, sbs, shs, num_blocks;
  int is64, heads, head_size;
};

__global__ void __launch_bounds__(256) fp8_link_kernel(const Fp8Rows a, const int B) {
  pdl_wait();  // the scratch may still be the kernel's before this one
  pdl_trigger();
  const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
  if (t >= a.tokens) return;
  const long long slot = slot_at(a.slots, a.is64, t);
  if (slot < 0 || slot >= a.num_blocks * B) return;
  int* entry = a.member + slot;
  int seen = *reinterpret_cast<volatile int*>(entry);
  while (true) {  // ends: the entry only changes to tokens of this slot, and among them only to later ones
    if (seen >= (int)t && seen < a.tokens && slot_at(a.slots, a.is64, seen) == slot) return;
    const int was = atomicCAS(entry, seen, (int)t);
    if (was == seen) return;
    seen = was;
  }
}

// Rows and cells are read with ordinary loads: these kernels begin while the one before them may still write what they read, which the
// read-only path does not allow. (In this form, so that stores to other places do not hold them up.)
__device__ __forceinline__ uint4 load16(const void* p) {
  uint4 v;
  asm volatile("ld.global.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
__device__ __forceinline__ uint2 load8(const void* p) {
  uint2 v;
  asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// Eight consecutive elements of a row, as they come.
template <typename T> struct Raw8 {
  static constexpr int kVecs = sizeof(T) / 2;
  uint4 v[kVecs];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) v[i] = load16(p + 16 * i);
  }
  __device__ __forceinline__ void floats(float* f) const {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) unpack16<T>(v[i], f + i * ElemTraits<T>::kVec);
  }
  // Running maximum of magnitudes as bits, which order like the numbers (two 16-bit ones side by side).
  __device__ __forceinline__ void top_bits(uint32_t& m) const {
#pragma unroll
    for (int i = 0; i < kVecs; ++i) {
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) m = sizeof(T) == 2 ? __vmaxu2(m, w[k] & 0x7fff7fffu) : max(m, w[k] & 0x7fffffffu);
    }
  }
};
// The larger magnitude in such bits, as a float (an infinity or NaN stays one).
template <typename T> __device__ __forceinline__ float top_of(uint32_t m);
template <> __device__ __forceinline__ float top_of<float>(uint32_t m) { return __uint_as_float(m); }
template <> __device__ __forceinline__ float top_of<__half>(uint32_t m) { return __half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16))); }
template <> __device__ __forceinline__ float top_of<__nv_bfloat16>(uint32_t m) { return __uint_as_float(max(m & 0xffffu, m >> 16) << 16); }

__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

template <typename T> __device__ __forceinline__ void store8(uint8_t* p, const float* f) {
  constexpr int kVec = ElemTraits<T>::kVec;
#pragma unroll
  for (int j = 0; j < 8; j += kVec) {
    uint4 v;
    T* o = reinterpret_cast<T*>(&v);
#pragma unroll
    for (int i = 0; i < kVec; ++i) o[i] = from_float<T>(f[j + i]);
    *reinterpret_cast<uint4*>(p + j * sizeof(T)) = v;
  }
}

// 4 x 4 bytes: byte i of w[j] and byte j of w[i] change places.
__device__ __forceinline__ void transpose4(uint32_t (&w)[4]) {
  const uint32_t a = __byte_perm(w[0], w[1], 0x5140), b = __byte_perm(w[2], w[3], 0x5140);
  const uint32_t c = __byte_perm(w[0], w[1], 0x7362), e = __byte_perm(w[2], w[3], 0x7362);
  w[0] = __byte_perm(a, b, 0x5410); w[1] = __byte_perm(a, b, 0x7632);
  w[2] = __byte_perm(c, e, 0x5410); w[3] = __byte_perm(c, e, 0x7632);
}
// Lane (g, dg) = (lane / 8, lane % 8) of a 16 x 64 tile: codes of tokens 4 g .. 4 g + 3 at elements 8 dg .. 8 dg + 7 (tok[j]: token
// 4 g + j) <-> the codes of all 16 tokens at elements 8 dg + 2 g and 8 dg + 2 g + 1 (row[0], row[1]).
__device__ __forceinline__ void tokens_to_rows(const uint2 (&tok)[4], uint4 (&row)[2], int g) {
  uint32_t lo[4] = {tok[0].x, tok[1].x, tok[2].x, tok[3].x}, hi[4] = {tok[0].y, tok[1].y, tok[2].y, tok[3].y};
  transpose4(lo);  // lo[k]: tokens 4 g .. at element k; hi[k]: at element 4 + k
  transpose4(hi);
  const bool g1 = g & 2, g0 = g & 1;
  uint32_t x[4], y[4];  // elements 4 (g / 2) + k: x of token groups 0, 1 (that with the parity of g), y of 2, 3
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, g1 ? lo[k] : hi[k], 16);
    x[k] = g1 ? got : lo[k];
    y[k] = g1 ? hi[k] : got;
  }
#pragma unroll
  for (int k = 0; k < 2; ++k) {  // elements 2 g + k
    const uint32_t gx = __shfl_xor_sync(0xffffffffu, g0 ? x[k] : x[k + 2], 8), gy = __shfl_xor_sync(0xffffffffu, g0 ? y[k] : y[k + 2], 8);
    const uint32_t mx = g0 ? x[k + 2] : x[k], my = g0 ? y[k + 2] : y[k];
    row[k] = g0 ? make_uint4(gx, mx, gy, my) : make_uint4(mx, gx, my, gy);
  }
}
__device__ __forceinline__ void rows_to_tokens(const uint4 (&row)[2], uint2 (&tok)[4], int g) {
  const bool g1 = g & 2, g0 = g & 1;
  uint32_t x[4], y[4];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const uint32_t sx = g0 ? row[k].x : row[k].y, sy = g0 ? row[k].z : row[k].w;
    const uint32_t gx = __shfl_xor_sync(0xffffffffu, sx, 8), gy = __shfl_xor_sync(0xffffffffu, sy, 8);
    const uint32_t mx = g0 ? row[k].y : row[k].x, my = g0 ? row[k].w : row[k].z;
    x[k] = g0 ? gx : mx; x[k + 2] = g0 ? mx : gx;
    y[k] = g0 ? gy : my; y[k + 2] = g0 ? my : gy;
  }
  uint32_t lo[4], hi[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t got = __shfl_xor_sync(0xffffffffu, g1 ? x[k] : y[k], 16);
    lo[k] = g1 ? got : x[k];
    hi[k] = g1 ? y[k] : got;
  }
  transpose4(lo);
  transpose4(hi);
#pragma unroll
  for (int j = 0; j < 4; ++j) tok[j] = make_uint2(lo[j], hi[j]);
}

constexpr int kWarps = 8;
constexpr int kScanTokens = 1024;  // (the table's kernel is a launch more: 5 us)

// Codes that a block holds already, under its grown scale. (Under a scale of 0 they all stood for 0, whatever they are.)
__device__ __forceinline__ uint32_t requantised(uint32_t w, float held, float inv) {
  if (held == 0.f) return 0u;
  const float2 a = fp8::to_float2(w), b = fp8::to_float2(w >> 16);
  return fp8::pack4(fp8::scaled(__fmul_rn(a.x, held), inv), fp8::scaled(__fmul_rn(a.y, held), inv),
                    fp8::scaled(__fmul_rn(b.x, held), inv), fp8::scaled(__fmul_rn(b.y, held), inv));
}
// 0xff in the bytes of the tokens 4 w .. 4 w + 3 that are in `mask`.
__device__ __forceinline__ uint32_t byte_mask(uint32_t mask, int w) {
  const uint32_t m = (mask >> (4 * w)) & 15u;
  return ((m & 1u) | ((m & 2u) << 7) | ((m & 4u) << 14) | ((m & 8u) << 21)) * 255u;
}

// The K or the V tile of one (block, head), by a warp. member: its tokens per offset (-1: none), mask: the offsets that have one.
template <typename T, int D, int B>
__device__ __forceinline__ void fill_tile(const uint8_t* rows, size_t row_bytes, uint8_t* tile, float* scale, const int* member,
                                          uint32_t mask, bool is_value, int lane) {
  constexpr int kPasses = (D / 8 + 7) / 8, kSubs = B / 16;
  // Rows wait in registers for the scale where 64 hold them, else they are read twice.
  constexpr bool kHold = kSubs * kPasses * 16 * (int)sizeof(T) / 2 <= 64;
  const int g = lane >> 3, dg = lane & 7;
  Raw8<T> raw[kHold ? kSubs : 1][kHold ? kPasses : 1][4];
  auto fetch = [&](Raw8<T>& to, int sub, int p, int j) {
    const int m = member[sub * 16 + 4 * g + j], c = p * 8 + dg;
    to.clear();
    if (m >= 0 && c < D / 8) to.load(rows + (size_t)m * row_bytes + c * 8 * sizeof(T));
  };
  const float held = (mask & 1u) ? 0.f : *scale;  // a block that gets its first token begins anew
  uint32_t bits = 0;
#pragma unroll
  for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      if (kHold) {
#pragma unroll
        for (int j = 0; j < 4; ++j) fetch(raw[kHold ? sub : 0][kHold ? p : 0][j], sub, p, j);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) fetch(raw[0][0][j], sub, p, j);
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[0][0][j].top_bits(bits);
      }
    }
  if (kHold) {
#pragma unroll
    for (int sub = 0; sub < kSubs; ++sub)
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int j = 0; j < 4; ++j) raw[kHold ? sub : 0][kHold ? p : 0][j].top_bits(bits);
  }
  float top = top_of<T>(bits);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = __uint_as_float(max(__float_as_uint(top), __shfl_xor_sync(0xffffffffu, __float_as_uint(top), o)));
  const bool odd = !is_finite(top);  // NaN or an infinity among them: the others' maximum is looked for one by one
  if (odd) {
    top = 0.f;
#pragma unroll 1
    for (int i = 0; i < kSubs * kPasses * 4; ++i) {
      Raw8<T> one;
      fetch(one, i / (4 * kPasses), (i >> 2) % kPasses, i & 3);
      float f[8];
      one.floats(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, is_finite(f[k]) ? fabsf(f[k]) : 0.f);
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    top = fmaxf(top, 448.f * fp8::kMinValueScale);  // (tiles with smaller scales may be read as zeros, which NaN is not)
  }
  const float now = fmaxf(held, fp8::scale_for(top));
  const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
  const bool grown = !(mask & 1u) && now > held;
#pragma unroll
  for (int sub = 0; sub < kSubs; ++sub) {
    const uint32_t sub_mask = (mask >> (16 * sub)) & 0xffffu;
    if (sub_mask == 0 && !grown) continue;
#pragma unroll
    for (int p = 0; p < kPasses; ++p) {
      const int c = p * 8 + dg;
      uint2 tok[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!kHold) fetch(raw[0][0][j], sub, p, j);
        float f[8];
        raw[kHold ? sub : 0][kHold ? p : 0][j].floats(f);
        if (odd) {
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = fp8::scaled(f[k], inv);
        } else {
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = __fmul_rn(f[k], inv);
        }
        tok[j] = make_uint2(fp8::pack4(f[0], f[1], f[2], f[3]), fp8::pack4(f[4], f[5], f[6], f[7]));
      }
      if (!is_value) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int off = 4 * g + j;
          uint2* at = reinterpret_cast<uint2*>(tile + ((c >> 1) * B + sub * 16 + off) * 16 + 8 * (c & 1));
          if (c >= D / 8) continue;
          if ((sub_mask >> off) & 1u) *at = tok[j];
          else if (grown) *at = make_uint2(requantised(at->x, held, inv), requantised(at->y, held, inv));
        }
      } else {
        uint4 row[2];
        tokens_to_rows(tok, row, g);
        if (c < D / 8) {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint4* at = reinterpret_cast<uint4*>(tile + (c * 8 + 2 * g + k) * B + sub * 16);
            if (sub_mask != 0xffffu) {
              uint4 old = *at;
              if (grown) old = make_uint4(requantised(old.x, held, inv), requantised(old.y, held, inv), requantised(old.z, held, inv), requantised(old.w, held, inv));
              const uint32_t m0 = byte_mask(sub_mask, 0), m1 = byte_mask(sub_mask, 1), m2 = byte_mask(sub_mask, 2), m3 = byte_mask(sub_mask, 3);
              row[k] = make_uint4((row[k].x & m0) | (old.x & ~m0), (row[k].y & m1) | (old.y & ~m1), (row[k].z & m2) | (old.z & ~m2),
                                  (row[k].w & m3) | (old.w & ~m3));
            }
            *at = row[k];
          }
        }
      }
    }
  }
  __syncwarp();  // every lane has read the scale
  if (lane == 0 && now != held) *scale = now;
  if (lane == 0 && now == held && (mask & 1u)) *scale = now;  // (0: what the block's last owner left is void)
}

// One token alone in its block, under kRowHeads heads from h0 (nh of them are there): lanes 0-15 take its K rows, 16-31 its V rows.
// Returns the tiles that are left to fill_tile, two bits a head: those of heads where a scale has to grow under other tokens, or with a NaN or an
// infinity.
constexpr int kRowHeads = 4;
template <typename T, int D, int B>
__device__ __forceinline__ uint32_t fill_rows(const Fp8Rows& a, long long blk, int h0, int nh, int m, int off, int lane) {
  constexpr int kPer = (D / 8 + 15) / 16;
  const int v = lane >> 4, l = lane & 15;
  const uint8_t* row = (v ? a.value : a.key) + ((size_t)m * (v ? a.value_stride : a.key_stride) + (size_t)h0 * D) * sizeof(T);
  uint8_t* tile = (v ? a.vcache : a.kcache) + (size_t)blk * a.kbs + (size_t)h0 * a.khs;
  float* scale = (v ? a.vscale : a.kscale) + (size_t)blk * a.sbs + (size_t)h0 * a.shs;
  Raw8<T> raw[kRowHeads][kPer];
  float held[kRowHeads];
#pragma unroll
  for (int h = 0; h < kRowHeads; ++h) {
    held[h] = (h < nh && off != 0) ? scale[(size_t)h * a.shs] : 0.f;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      raw[h][p].clear();
      if (h < nh && p * 16 + l < D / 8) raw[h][p].load(row + (h * D + (p * 16 + l) * 8) * sizeof(T));
    }
  }
  uint32_t left = 0;
#pragma unroll
  for (int h = 0; h < kRowHeads; ++h) {
    uint32_t bits = 0;
#pragma unroll
    for (int p = 0; p < kPer; ++p) raw[h][p].top_bits(bits);
    float top = top_of<T>(bits);
#pragma unroll
    for (int o = 8; o >= 1; o >>= 1) top = __uint_as_float(max(__float_as_uint(top), __shfl_xor_sync(0xffffffffu, __float_as_uint(top), o)));
    const float now = fmaxf(held[h], fp8::scale_for(top));
    if (__any_sync(0xffffffffu, !is_finite(top) || (off != 0 && now > held[h]))) {
      left |= 3u << (2 * h);
      continue;
    }
    if (h >= nh) continue;
    const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
#pragma unroll
    for (int p = 0; p < kPer; ++p) {
      const int c = p * 16 + l;
      if (c >= D / 8) continue;
      float f[8];
      raw[h][p].floats(f);
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] = __fmul_rn(f[k], inv);
      const uint2 w = make_uint2(fp8::pack4(f[0], f[1], f[2], f[3]), fp8::pack4(f[4], f[5], f[6], f[7]));
      uint8_t* t = tile + (size_t)h * a.khs;
      if (v == 0) {
        *reinterpret_cast<uint2*>(t + ((c >> 1) * B + off) * 16 + 8 * (c & 1)) = w;
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) t[(c * 8 + k) * B + off] = (uint8_t)((k < 4 ? w.x : w.y) >> (8 * (k & 3)));
      }
    }
    if (l == 0) scale[(size_t)h * a.shs] = now;  // (behind the shuffles: every lane has read it)
  }
  return left;
}

// CTAs an SM: four where the rows of a tile take 32 registers, two where they take 64, three where they are read twice. (Left to
// itself the compiler takes up to 210 registers: 930 rows of fp32, heads of 80, blocks of 32, 41 us against 19. The bounds spill: 24 to 40
// bytes a thread in 16-bit tiles of 16 tokens x 80 to 128 and of 32 x 64, as much in fp32 ones of 16 x 64 and 32 x 80 to 112, 120 to 128 in fp32
// of 256. They were chosen by time, the other bounds of a shape were not tried one by one.)
template <typename T, int D, int B> constexpr int kRowWords = (B / 16) * ((D / 8 + 7) / 8) * 16 * (int)sizeof(T) / 2;
template <typename T, int D, int B> constexpr int kFillCtas = kRowWords<T, D, B> <= 32 ? 4 : kRowWords<T, D, B> <= 64 ? 2 : 3;

// A CTA: 16 consecutive entries of slot_mapping, the blocks whose first token is among them, and one head or a few. A warp
// takes one (block, head) at a time.
template <typename T, int D, int B>
__global__ void __launch_bounds__(kWarps * 32, kFillCtas<T, D, B>) fp8_fill_kernel(const Fp8Rows a, const int heads_per_cta) {
  __shared__ int member[16][B];
  __shared__ int first[16], many[16], lone[16], n_many, n_lone;  // (the blocks of this window with several tokens, and with one)
  __shared__ long long block_of[16];
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t0 = (long long)blockIdx.x * 16;
  if (warp == 0) {
    const long long t = t0 + lane, slot = lane < 16 && t < a.tokens ? slot_at(a.slots, a.is64, t) : -1;
    const long long blk = slot >= 0 && slot < a.num_blocks * B ? slot / B : -1;
    const unsigned same = __match_any_sync(0xffffffffu, blk);
    if (lane < 16) {
      block_of[lane] = __ffs(same) - 1 == lane ? blk : -1;  // a block stands at its first entry
      first[lane] = 0x7fffffff;
    }
  }
  if (!a.member)
    for (int i = threadIdx.x; i < 16 * B; i += kWarps * 32) member[0][i] = -1;
  __syncthreads();
  if (a.member) {
    for (int idx = threadIdx.x; idx < 16 * B; idx += kWarps * 32) {
      const int i = idx / B, off = idx % B;
      const long long blk = block_of[i];
      int m = -1;
      if (blk >= 0) {
        m = a.member[blk * B + off];
        if (m < 0 || m >= a.tokens || slot_at(a.slots, a.is64, m) != blk * B + off) m = -1;
      }
      member[i][off] = m;
      if (m >= 0) atomicMin(&first[i], m);
    }
  } else {
    for (int t = threadIdx.x; t < (int)a.tokens; t += kWarps * 32) {
      const long long slot = slot_at(a.slots, a.is64, t);
      if (slot < 0) continue;
      const long long blk = slot / B;
#pragma unroll 4
      for (int i = 0; i < 16; ++i)
        if (block_of[i] == blk) {
          atomicMax(&member[i][(int)(slot - blk * B)], t);
          atomicMin(&first[i], t);
        }
    }
  }
  __syncthreads();
  if (warp == 0) {
    const bool mine = lane < 16 && block_of[lane & 15] >= 0 && first[lane & 15] >= t0 && first[lane & 15] < t0 + 16;
    int count = 0;
    if (mine)
      for (int off = 0; off < B; ++off) count += member[lane][off] >= 0;
    const unsigned ones = __ballot_sync(0xffffffffu, mine && count == 1), others = __ballot_sync(0xffffffffu, mine && count != 1);
    const unsigned before = (1u << lane) - 1u;
    if (mine && count == 1) lone[__popc(ones & before)] = lane;
    if (mine && count != 1) many[__popc(others & before)] = lane;
    if (lane == 0) {
      n_lone = __popc(ones);
      n_many = __popc(others);
    }
  }
  __syncthreads();
  const int h0 = blockIdx.y * heads_per_cta, nh = min(heads_per_cta, a.heads - h0);
  // The K and V tiles of the many, block by block and head by head, then the lone ones four heads at a time; what the latter
  // leave over is done behind them.
  const int tile_tasks = n_many * nh * 2, row_tasks = (nh + kRowHeads - 1) / kRowHeads, n_tasks = tile_tasks + n_lone * row_tasks;
  for (int idx = warp; idx < n_tasks; idx += kWarps) {
    int e, h, heads = 0;
    uint32_t left;  // bit 2 k + v: the K (v = 0) or V tile of head h + k
    if (idx < tile_tasks) {
      e = many[(idx >> 1) / nh]; h = h0 + (idx >> 1) % nh;
      left = 1u << (idx & 1);
    } else {
      const int i = idx - tile_tasks;
      e = lone[i / row_tasks]; h = h0 + i % row_tasks * kRowHeads;
      heads = min(kRowHeads, h0 + nh - h);
    }
    const long long blk = block_of[e];
    const int m = lane < B ? member[e][lane] : -1;
    const uint32_t mask = __ballot_sync(0xffffffffu, m >= 0);
    if (heads > 0) {
      const int off = __ffs(mask) - 1;
      left = fill_rows<T, D, B>(a, blk, h, heads, __shfl_sync(0xffffffffu, m, off), off, lane);
    }
    for (; left; left &= left - 1) {
      const int v = (__ffs(left) - 1) & 1, hh = h + ((__ffs(left) - 1) >> 1);
      fill_tile<T, D, B>((v ? a.value : a.key) + (size_t)hh * D * sizeof(T), (size_t)(v ? a.value_stride : a.key_stride) * sizeof(T),
                         (v ? a.vcache : a.kcache) + (size_t)blk * a.kbs + (size_t)hh * a.khs,
                         (v ? a.vscale : a.kscale) + (size_t)blk * a.sbs + (size_t)hh * a.shs, member[e], mask, v == 1, lane);
    }
  }
}

// A CTA: `win` (at most kMaxWin) consecutive entries of slot_mapping, cut into runs of consecutive slots inside 16 tokens of a block,
// and one head or a few. A warp takes the K or V rows of one (run, head) at a time. (V of a lone token costs the DRAM sectors
// of the whole tile however it is read.)
constexpr int kMaxWin = 256;
template <typename T, int D, int B>
__global__ void __launch_bounds__(kWarps * 32) fp8_gather_kernel(const Fp8Rows a, const int win, const int heads_per_cta) {
  constexpr int kPasses = (D / 8 + 7) / 8;
  __shared__ long long slot_of[kMaxWin];
  __shared__ int run_start[kMaxWin + 1], n_runs_s;
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long t0 = (long long)blockIdx.x * win;
  if ((int)threadIdx.x < win) {
    const long long t = t0 + threadIdx.x, slot = t < a.tokens ? slot_at(a.slots, a.is64, t) : -1;
    slot_of[threadIdx.x] = slot >= 0 && slot < a.num_blocks * B ? slot : -1;
  }
  __syncthreads();
  if (warp == 0) {
    int n = 0;
    for (int b = 0; b < win; b += 32) {
      const int i = b + lane;
      const bool live = i < win;
      const long long s = live ? slot_of[i] : -1;
      const bool starts = live && (i == 0 || s < 0 || s % 16 == 0 || slot_of[i - 1] != s - 1);
      const unsigned all = __ballot_sync(0xffffffffu, starts);
      if (starts) run_start[n + __popc(all & ((1u << lane) - 1u))] = i;
      n += __popc(all);
    }
    if (lane == 0) {
      run_start[n] = win;
      n_runs_s = n;
    }
  }
  __syncthreads();
  const int h0 = blockIdx.y * heads_per_cta, nh = min(heads_per_cta, a.heads - h0), n_runs = n_runs_s;
  const int g = lane >> 3, dg = lane & 7;
  for (int idx = warp; idx < n_runs * nh * 2; idx += kWarps) {
    const bool is_value = idx & 1;
    const int h = h0 + (idx >> 1) % nh, run = (idx >> 1) / nh;
    const int start = run_start[run], len = run_start[run + 1] - start;
    const long long slot = slot_of[start];
    if (slot < 0) continue;
    const long long blk = slot / B;
    const int off0 = (int)(slot % 16), sub = (int)(slot % B) / 16;
    const uint8_t* tile = (is_value ? a.vcache : a.kcache) + (size_t)blk * a.kbs + (size_t)h * a.khs;
    const float scale = (is_value ? a.vscale : a.kscale)[(size_t)blk * a.sbs + (size_t)h * a.shs];
    const size_t stride = (size_t)(is_value ? a.value_stride : a.key_stride) * sizeof(T);
    uint8_t* rows = (is_value ? a.value : a.key) + (size_t)(t0 + start) * stride + (size_t)h * D * sizeof(T);
    uint2 tok[kPasses][4];
    if (!is_value) {
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int c = p * 8 + dg, i = 4 * g + j;
          tok[p][j] = make_uint2(0u, 0u);
          if (c < D / 8 && i >= off0 && i < off0 + len)
            tok[p][j] = load8(tile + ((c >> 1) * B + sub * 16 + i) * 16 + 8 * (c & 1));
        }
    } else {
      uint4 row[kPasses][2];
#pragma unroll
      for (int p = 0; p < kPasses; ++p)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c = p * 8 + dg;
          row[p][k] = make_uint4(0u, 0u, 0u, 0u);
          if (c < D / 8) row[p][k] = load16(tile + (c * 8 + 2 * g + k) * B + sub * 16);
        }
#pragma unroll
      for (int p = 0; p < kPasses; ++p) rows_to_tokens(row[p], tok[p], g);
    }
#pragma unroll
    for (int p = 0; p < kPasses; ++p)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int c = p * 8 + dg, i = 4 * g + j;
        if (c >= D / 8 || i < off0 || i >= off0 + len) continue;
        const uint32_t w[4] = {tok[p][j].x, tok[p][j].x >> 16, tok[p][j].y, tok[p][j].y >> 16};
        float f[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 x = fp8::to_float2(w[k]);
          f[2 * k] = x.x * scale;
          f[2 * k + 1] = x.y * scale;
        }
        store8<T>(rows + (size_t)(i - off0) * stride + c * 8 * sizeof(T), f);
      }
  }
}

int bind_rows(const pb_fp8_cache* c, const void* key, const void* value, const void* slots, int32_t is64, int64_t tokens,
              int64_t key_stride, int64_t value_stride, int32_t dtype, Fp8Rows* a) {
  if (!c) return PB_ERR_INVALID_ARG;
  const int rc = check_fp8_cache(c);
  if (rc != PB_OK) return rc;
  if (dtype != PB_F32 && dtype != PB_F16 && dtype != PB_BF16) return PB_ERR_UNSUPPORTED;
  if (tokens < 0 || tokens > 0x7fffffff) return PB_ERR_INVALID_ARG;
  if (tokens == 0) return PB_OK;
  if (!key || !value || !slots) return PB_ERR_INVALID_ARG;
  const int vec = dtype == PB_F32 ? 4 : 8;
  if ((reinterpret_cast<uintptr_t>(key) & 15u) || (reinterpret_cast<uintptr_t>(value) & 15u) || key_stride % vec || value_stride % vec)
    return PB_ERR_INVALID_ARG;
  if (tokens > 1 && (key_stride < (int64_t)c->num_kv_heads * c->head_size || value_stride < (int64_t)c->num_kv_heads * c->head_size))
    return PB_ERR_INVALID_ARG;
  a->key = static_cast<uint8_t*>(const_cast<void*>(key)); a->value = static_cast<uint8_t*>(const_cast<void*>(value));
  a->kcache = static_cast<uint8_t*>(c->key_cache); a->vcache = static_cast<uint8_t*>(c->value_cache);
  a->kscale = c->key_scale; a->vscale = c->value_scale;
  a->slots = slots; a->is64 = is64; a->member = nullptr;
  a->tokens = tokens; a->key_stride = key_stride; a->value_stride = value_stride;
  a->kbs = c->kv_block_stride; a->khs = c->kv_head_stride; a->sbs = c->scale_block_stride; a->shs = c->scale_head_stride;
  a->num_blocks = c->num_blocks; a->heads = c->num_kv_heads; a->head_size = c->head_size;
  return PB_OK;
}

// Whether the tiles of a [blocks, heads] grid lie apart: neighbours by the smaller stride, and their rows by the larger one. (Grids whose
// rows interleave without a collision are not looked for: no view of a cache is one.)
bool lie_apart(int64_t blocks, int64_t block_stride, int64_t heads, int64_t head_stride, int64_t tile) {
  if (blocks <= 1) return heads <= 1 || head_stride >= tile;
  if (heads <= 1) return block_stride >= tile;
  const bool heads_inside = head_stride <= block_stride;
  const int64_t inner = heads_inside ? head_stride : block_stride, count = heads_inside ? heads : blocks;
  return inner >= tile && (heads_inside ? block_stride : head_stride) >= (count - 1) * inner + tile;
}

int fail(cudaError_t e) {
  set_cuda_error(e);
  return PB_ERR_LAUNCH;
}

// Heads per CTA, of `windows` windows: as many CTAs as keep the SMs busy, and what they share read as seldom as that allows, up to
// four (fill and gather of 9.4k rows x 32 heads, with at most 1 / 2 / 3 / 4 / 6 / 8 heads: 205 / 155 / 146 / 139 / 142 / 143 us).
int heads_per_cta(long long windows, int heads) {
  const long long spare = windows * heads / ((long long)sm_count() * 8);
  return (int)(spare < 1 ? 1 : spare > 4 ? 4 : spare);
}

template <typename T, int D, int B>
cudaError_t launch_fill(const Fp8Rows& a, cudaStream_t s) {
  const unsigned windows = (unsigned)((a.tokens + 15) / 16);
  const int hpc = heads_per_cta(windows, a.heads);
  return launch_kernel(fp8_fill_kernel<T, D, B>, dim3(windows, (unsigned)((a.heads + hpc - 1) / hpc)), kWarps * 32, 0, s, true, a, hpc);
}
template <typename T, int D, int B>
cudaError_t launch_gather(const Fp8Rows& a, cudaStream_t s) {
  // (short windows for few rows, long ones where runs are cut less often by them)
  int win = kMaxWin;
  while (win > 16 && a.tokens * a.heads < (long long)sm_count() * 4 * win) win /= 4;
  const unsigned windows = (unsigned)((a.tokens + win - 1) / win);
  const int hpc = heads_per_cta(windows, a.heads);
  return launch_kernel(fp8_gather_kernel<T, D, B>, dim3(windows, (unsigned)((a.heads + hpc - 1) / hpc)), kWarps * 32, 0, s, true, a, win, hpc);
}

template <typename T, int D>
cudaError_t launch_d(const Fp8Rows& a, int block_size, bool fill, cudaStream_t s) {
  if (block_size == 16) return fill ? launch_fill<T, D, 16>(a, s) : launch_gather<T, D, 16>(a, s);
  return fill ? launch_fill<T, D, 32>(a, s) : launch_gather<T, D, 32>(a, s);
}
template <typename T>
cudaError_t launch_t(const Fp8Rows& a, int block_size, bool fill, cudaStream_t s) {
  switch (a.head_size) {
    case 64: return launch_d<T, 64>(a, block_size, fill, s);
    case 80: return launch_d<T, 80>(a, block_size, fill, s);
    case 96: return launch_d<T, 96>(a, block_size, fill, s);
    case 112: return launch_d<T, 112>(a, block_size, fill, s);
    case 128: return launch_d<T, 128>(a, block_size, fill, s);
    case 256: return launch_d<T, 256>(a, block_size, fill, s);
    default: return cudaErrorInvalidValue;
  }
}
cudaError_t launch_rows(const Fp8Rows& a, int dtype, int block_size, bool fill, cudaStream_t s) {
  return dtype == PB_F16    ? launch_t<__half>(a, block_size, fill, s)
         : dtype == PB_BF16 ? launch_t<__nv_bfloat16>(a, block_size, fill, s)
                            : launch_t<float>(a, block_size, fill, s);
}

}  // namespace
}  // namespace pb

extern "C" {

size_t pb_fp8_fill_workspace_bytes(int64_t num_tokens, int64_t num_blocks, int32_t block_size) {
  if (num_tokens <= pb::kScanTokens || num_blocks < 0 || block_size <= 0 || num_blocks > (int64_t)1 << 40) return 0;
  return (size_t)num_blocks * block_size * sizeof(int32_t);
}

int pb_fp8_reshape_and_cache(const pb_fp8_cache* cache, const void* key, const void* value, const void* slot_mapping,
                             int32_t slot_is_i64, int64_t num_tokens, int64_t key_stride, int64_t value_stride,
                             int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
  pb::Fp8Rows a;
  const int rc = pb::bind_rows(cache, key, value, slot_mapping, slot_is_i64, num_tokens, key_stride, value_stride, dtype, &a);
  if (rc != PB_OK || num_tokens == 0) return rc;
  // blocks or heads that share memory would be written by several owners
  if (!pb::lie_apart(cache->num_blocks, cache->kv_block_stride, cache->num_kv_heads, cache->kv_head_stride, (int64_t)cache->head_size * cache->block_size) ||
      !pb::lie_apart(cache->num_blocks, cache->scale_block_stride, cache->num_kv_heads, cache->scale_head_stride, 1))
    return PB_ERR_INVALID_ARG;
  const size_t need = pb_fp8_fill_workspace_bytes(num_tokens, cache->num_blocks, cache->block_size);
  if (need > 0 && (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) || workspace_bytes < need)) return PB_ERR_WORKSPACE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaSuccess;
  if (num_tokens > pb::kScanTokens) {
    a.member = static_cast<int*>(workspace);
    e = pb::launch_kernel(pb::fp8_link_kernel, dim3((unsigned)((num_tokens + 255) / 256)), 256, 0, s, true, a, (int)cache->block_size);
  }
  if (e == cudaSuccess) e = pb::launch_rows(a, dtype, cache->block_size, true, s);
  return e == cudaSuccess ? PB_OK : pb::fail(e);
}

int pb_fp8_gather_cached_kv(const pb_fp8_cache* cache, void* key, void* value, const void* slot_mapping,
                            int32_t slot_is_i64, int64_t num_tokens, int64_t key_stride, int64_t value_stride,
                            int32_t dtype, void* stream) {
  pb::Fp8Rows a;
  const int rc = pb::bind_rows(cache, key, value, slot_mapping, slot_is_i64, num_tokens, key_stride, value_stride, dtype, &a);
  if (rc != PB_OK || num_tokens == 0) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = pb::launch_rows(a, dtype, cache->block_size, false, s);
  return e == cudaSuccess ? PB_OK : pb::fail(e);
}

}  // extern "C"
