// Fill of the 8-bit paged cache, and rows out of it again.
//
// The scale of a (block, head) depends on all tokens that the call brings to the block, and a scale that grows changes the
// block's other cells, so a block has one owner per call: the window (16 consecutive entries of slot_mapping) that holds the
// first of its tokens. Which tokens those are says a table with an entry per slot, written by a kernel in front (fp8_link):
//     member[slot] = the last token of the list with that slot
// The table lives in scratch that nobody clears: an entry counts only if it names a token of this call whose slot is that
// slot, and every slot that has a token has been written.
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

// Eight consecutive elements of a row as floats.
template <typename T> __device__ __forceinline__ void load8(const uint8_t* p, float* f);
template <> __device__ __forceinline__ void load8<float>(const uint8_t* p, float* f) {
  unpack16<float>(*reinterpret_cast<const uint4*>(p), f);
  unpack16<float>(*reinterpret_cast<const uint4*>(p + 16), f + 4);
}
template <> __device__ __forceinline__ void load8<__half>(const uint8_t* p, float* f) { unpack16<__half>(*reinterpret_cast<const uint4*>(p), f); }
template <> __device__ __forceinline__ void load8<__nv_bfloat16>(const uint8_t* p, float* f) {
  unpack16<__nv_bfloat16>(*reinterpret_cast<const uint4*>(p), f);
}
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

// Eight codes of token `off` of a tile: elements 16 c + 8 half .. + 7.
template <int B> __device__ __forceinline__ uint2 load_codes(const uint8_t* tile, bool is_value, int off, int c, int half) {
  if (!is_value) return *reinterpret_cast<const uint2*>(tile + (c * B + off) * 16 + 8 * half);
  uint32_t w[2] = {0u, 0u};
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j >> 2] |= (uint32_t)tile[(size_t)(16 * c + 8 * half + j) * B + off] << (8 * (j & 3));
  return make_uint2(w[0], w[1]);
}
template <int B> __device__ __forceinline__ void store_codes(uint8_t* tile, bool is_value, int off, int c, int half, uint2 v) {
  if (!is_value) { *reinterpret_cast<uint2*>(tile + (c * B + off) * 16 + 8 * half) = v; return; }
#pragma unroll
  for (int j = 0; j < 8; ++j) tile[(size_t)(16 * c + 8 * half + j) * B + off] = (uint8_t)((j < 4 ? v.x : v.y) >> (8 * (j & 3)));
}

constexpr int kFillWarps = 4;

// A CTA: 16 consecutive entries of slot_mapping, the blocks whose first token is among them, and one head or a few. A warp
// takes the K or the V tile of one (block, head): lane (i, half) = (lane % 16, lane / 16) holds eight elements of token i at a time.
template <typename T, int B>
__global__ void __launch_bounds__(kFillWarps * 32) fp8_fill_kernel(const Fp8Rows a, const int heads_per_cta) {
  __shared__ int member[16][B];
  __shared__ long long block_of[16];  // -1: not this window's block
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  {
    constexpr int kPer = B / 8;  // member entries per thread: eight threads a token
    const int i = threadIdx.x >> 3, sub = threadIdx.x & 7;
    const long long t = (long long)blockIdx.x * 16 + i;
    const long long slot = t < a.tokens ? slot_at(a.slots, a.is64, t) : -1;
    const bool live = slot >= 0 && slot < a.num_blocks * B;
    const long long blk = live ? slot / B : -1;
    int first = 0x7fffffff;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const int off = sub * kPer + k;
      int m = -1;
      if (live) {
        m = a.member[blk * B + off];
        if (m < 0 || m >= a.tokens || slot_at(a.slots, a.is64, m) != blk * B + off) m = -1;
      }
      member[i][off] = m;
      if (m >= 0) first = min(first, m);
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
    if (sub == 0) block_of[i] = live && first == (int)t ? blk : -1;
  }
  __syncthreads();
  const unsigned owned = __ballot_sync(0xffffffffu, lane < 16 && block_of[lane & 15] >= 0);
  const int n_own = __popc(owned), h0 = blockIdx.y * heads_per_cta, nh = min(heads_per_cta, a.heads - h0);
  const int i = lane & 15, half = lane >> 4, chunks = a.head_size / 16;
  for (int idx = warp; idx < n_own * nh * 2; idx += kFillWarps) {
    const bool is_value = idx & 1;
    const int h = h0 + (idx >> 1) % nh;
    const int e = __fns(owned, 0, (idx >> 1) / nh + 1);
    const long long blk = block_of[e];
    const uint8_t* rows = (is_value ? a.value : a.key) + (size_t)h * a.head_size * sizeof(T);
    const size_t row_bytes = (size_t)(is_value ? a.value_stride : a.key_stride) * sizeof(T);
    uint8_t* tile = (is_value ? a.vcache : a.kcache) + (size_t)blk * a.kbs + (size_t)h * a.khs;
    float* scale = (is_value ? a.vscale : a.kscale) + (size_t)blk * a.sbs + (size_t)h * a.shs;
    const float held = member[e][0] >= 0 ? 0.f : *scale;  // a block that gets its first token begins anew
    float top = 0.f;
#pragma unroll
    for (int sub = 0; sub < B / 16; ++sub) {
      const int m = member[e][sub * 16 + i];
      if (m < 0) continue;
      for (int c = 0; c < chunks; ++c) {
        float f[8];
        load8<T>(rows + (size_t)m * row_bytes + (16 * c + 8 * half) * sizeof(T), f);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(f[j]) <= 3.402823466e38f ? fabsf(f[j]) : 0.f);
      }
    }
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    const float now = fmaxf(held, fp8::scale_for(top));
    const float inv = now > 0.f ? __frcp_rn(now) : 0.f;
    const bool grown = held > 0.f && now > held;
#pragma unroll
    for (int sub = 0; sub < B / 16; ++sub) {
      const int off = sub * 16 + i, m = member[e][off];
      if (m < 0 && !grown) continue;
      for (int c = 0; c < chunks; ++c) {
        float f[8];
        if (m >= 0) {
          load8<T>(rows + (size_t)m * row_bytes + (16 * c + 8 * half) * sizeof(T), f);
        } else {
          const uint2 v = load_codes<B>(tile, is_value, off, c, half);
          const uint32_t w[4] = {v.x, v.x >> 16, v.y, v.y >> 16};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 x = fp8::to_float2(w[j]);
            f[2 * j] = __fmul_rn(x.x, held);
            f[2 * j + 1] = __fmul_rn(x.y, held);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = fp8::scaled(f[j], inv);
        store_codes<B>(tile, is_value, off, c, half, make_uint2(fp8::pack4(f[0], f[1], f[2], f[3]), fp8::pack4(f[4], f[5], f[6], f[7])));
      }
    }
    __syncwarp();  // every lane has read the scale
    if (lane == 0) *scale = now;
  }
}

// A warp: 16 entries of slot_mapping, the K or the V rows of one head.
template <typename T, int B>
__global__ void __launch_bounds__(kFillWarps * 32) fp8_gather_kernel(const Fp8Rows a) {
  pdl_wait();
  pdl_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = lane & 15, half = lane >> 4;
  const long long t = (long long)blockIdx.x * 16 + i;
  const int idx = blockIdx.y * kFillWarps + warp;
  if (idx >= 2 * a.heads || t >= a.tokens) return;
  const bool is_value = idx & 1;
  const int h = idx >> 1;
  const long long slot = slot_at(a.slots, a.is64, t);
  if (slot < 0 || slot >= a.num_blocks * B) return;
  const long long blk = slot / B;
  const int off = (int)(slot - blk * B);
  const uint8_t* tile = (is_value ? a.vcache : a.kcache) + (size_t)blk * a.kbs + (size_t)h * a.khs;
  const float scale = (is_value ? a.vscale : a.kscale)[(size_t)blk * a.sbs + (size_t)h * a.shs];
  uint8_t* row = is_value ? a.value + ((size_t)t * a.value_stride + (size_t)h * a.head_size) * sizeof(T)
                          : a.key + ((size_t)t * a.key_stride + (size_t)h * a.head_size) * sizeof(T);
  for (int c = 0; c < a.head_size / 16; ++c) {
    const uint2 v = load_codes<B>(tile, is_value, off, c, half);
    const uint32_t w[4] = {v.x, v.x >> 16, v.y, v.y >> 16};
    float f[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 x = fp8::to_float2(w[j]);
      f[2 * j] = x.x * scale;
      f[2 * j + 1] = x.y * scale;
    }
    store8<T>(row + (16 * c + 8 * half) * sizeof(T), f);
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

int fail(cudaError_t e) {
  set_cuda_error(e);
  return PB_ERR_LAUNCH;
}

template <int B>
cudaError_t launch_fill(const Fp8Rows& a, int dtype, cudaStream_t s) {
  const unsigned windows = (unsigned)((a.tokens + 15) / 16);
  const int hpc = 2;
  const dim3 grid(windows, (unsigned)((a.heads + hpc - 1) / hpc));
  auto kfn = dtype == PB_F16 ? fp8_fill_kernel<__half, B> : dtype == PB_BF16 ? fp8_fill_kernel<__nv_bfloat16, B> : fp8_fill_kernel<float, B>;
  return launch_kernel(kfn, grid, kFillWarps * 32, 0, s, true, a, hpc);
}
template <int B>
cudaError_t launch_gather(const Fp8Rows& a, int dtype, cudaStream_t s) {
  const dim3 grid((unsigned)((a.tokens + 15) / 16), (unsigned)((2 * a.heads + kFillWarps - 1) / kFillWarps));
  auto kfn = dtype == PB_F16 ? fp8_gather_kernel<__half, B> : dtype == PB_BF16 ? fp8_gather_kernel<__nv_bfloat16, B> : fp8_gather_kernel<float, B>;
  return launch_kernel(kfn, grid, kFillWarps * 32, 0, s, true, a);
}

}  // namespace
}  // namespace pb

extern "C" {

size_t pb_fp8_fill_workspace_bytes(int64_t num_tokens, int64_t num_blocks, int32_t block_size) {
  if (num_tokens < 0 || num_blocks < 0 || block_size <= 0 || num_blocks > (int64_t)1 << 40) return 0;
  return (size_t)num_blocks * block_size * sizeof(int32_t);
}

int pb_fp8_reshape_and_cache(const pb_fp8_cache* cache, const void* key, const void* value, const void* slot_mapping,
                             int32_t slot_is_i64, int64_t num_tokens, int64_t key_stride, int64_t value_stride,
                             int32_t dtype, void* workspace, size_t workspace_bytes, void* stream) {
  pb::Fp8Rows a;
  const int rc = pb::bind_rows(cache, key, value, slot_mapping, slot_is_i64, num_tokens, key_stride, value_stride, dtype, &a);
  if (rc != PB_OK || num_tokens == 0) return rc;
  if (!workspace || (reinterpret_cast<uintptr_t>(workspace) & 15u) ||
      workspace_bytes < pb_fp8_fill_workspace_bytes(num_tokens, cache->num_blocks, cache->block_size))
    return PB_ERR_WORKSPACE;
  a.member = static_cast<int*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t e = pb::launch_kernel(pb::fp8_link_kernel, dim3((unsigned)((num_tokens + 255) / 256)), 256, 0, s, true, a, (int)cache->block_size);
  if (e != cudaSuccess) return pb::fail(e);
  e = cache->block_size == 16 ? pb::launch_fill<16>(a, dtype, s) : pb::launch_fill<32>(a, dtype, s);
  return e == cudaSuccess ? PB_OK : pb::fail(e);
}

int pb_fp8_gather_cached_kv(const pb_fp8_cache* cache, void* key, void* value, const void* slot_mapping,
                            int32_t slot_is_i64, int64_t num_tokens, int64_t key_stride, int64_t value_stride,
                            int32_t dtype, void* stream) {
  pb::Fp8Rows a;
  const int rc = pb::bind_rows(cache, key, value, slot_mapping, slot_is_i64, num_tokens, key_stride, value_stride, dtype, &a);
  if (rc != PB_OK || num_tokens == 0) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const cudaError_t e = cache->block_size == 16 ? pb::launch_gather<16>(a, dtype, s) : pb::launch_gather<32>(a, dtype, s);
  return e == cudaSuccess ? PB_OK : pb::fail(e);
}

}  // extern "C"
