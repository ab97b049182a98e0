// Attention of a sequence's new tokens, drafted as a tree or following each other, over its paged cache.
//
// For new token i of n of a sequence of L tokens, head h reading kv head h / group:
// o_i = sum_j softmax_j(scale q_i . k_j) v_j over the context (j < L - n) and the new tokens that i sees:
// those of its tree's bits, or without a tree itself and those before.  Codes of 8 bits enter the sums as they
// are: a key's scale multiplies its score, a value's scale its weight.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sfe_cache.hpp"
#include "sfe_internal.hpp"

namespace sfe {
namespace {

template <int TYPE>
__device__ __forceinline__ float kept_value(const char* row, int d) {
  if constexpr (TYPE == kCacheE4m3) return __builtin_amdgcn_cvt_f32_fp8((int)(uint8_t)row[d], 0);
  else if constexpr (TYPE == kCacheInt8) return (float)(int8_t)row[d];
  else if constexpr (TYPE == kCacheBf16) return (float)reinterpret_cast<const __bf16*>(row)[d];
  else return (float)reinterpret_cast<const _Float16*>(row)[d];
}

// A wave a packed row: a lane takes a key's score, then two channels of the values' sum.
template <typename T, int TYPE>
__global__ __launch_bounds__(64) void sfe_cache_attn_kernel(CacheAttnArgs a, int64_t first) {
  const CacheArgs& c = a.c;
  const int64_t unit = first + blockIdx.x;
  const int kvh = (int)(unit % c.kv_heads), lane = (int)threadIdx.x;
  const CacheTile tile = c.tiles[unit / c.kv_heads];
  const int length = c.lengths[tile.seq];
  const int64_t part = (int64_t)Kept<TYPE>::kSize * c.dim << c.shift;
  for (int r = tile.at; r < tile.at + tile.count; ++r) {
    const int token = r / a.group, head = kvh * a.group + r - token * a.group;
    const T* q = reinterpret_cast<const T*>(a.q.data + (tile.first + token) * a.q.row + head * a.q.head);
    const int64_t context = (int64_t)length - tile.n, me = context + token;
    const uint64_t bits = a.tree ? a.tree[tile.first + token] : 0;
    float m = -INFINITY, l = 0.0f, o[2] = {0.0f, 0.0f};
    const int64_t end = me < 0 ? 0 : (a.tree ? length : me + 1);
    for (int64_t j0 = 0; j0 < end; j0 += 64) {
      const int64_t j = j0 + lane, draft = j - context;
      const int64_t page = j < end ? page_of(c, tile.seq, j) : -1;
      const bool see = page >= 0 && (draft < 0 || !a.tree || (draft < 64 && (bits >> draft & 1)));
      const char* record = c.data + (page * c.kv_heads + kvh) * c.record;
      const int slot = (int)(j & ((1 << c.shift) - 1));
      float s = -INFINITY, vs = 1.0f;
      if (see) {
        s = 0.0f;
        for (int d = 0; d < c.dim; ++d) s += (float)q[d] * kept_value<TYPE>(record + (int64_t)Kept<TYPE>::kSize * slot * c.dim, d);
        if (cache_coded(TYPE)) {
          const float* scales = reinterpret_cast<const float*>(record + 2 * part);
          s *= scales[slot];
          vs = scales[(1 << c.shift) + slot];
        }
        s *= a.scale_log2;
      }
      float top = s;
      for (int d = 32; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor(top, d));
      const float nm = fmaxf(m, top);
      const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - nm);
      m = nm;
      const float p = see ? __builtin_amdgcn_exp2f(s - m) : 0.0f;
      float sum = p;
      for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d);
      l = l * f + sum;
      o[0] *= f, o[1] *= f;
      for (int i = 0; i < 64; ++i) {
        if (!__shfl((int)see, i)) continue;
        const float w = __shfl(p, i) * __shfl(vs, i);
        const char* values = c.data + (__shfl(page, i) * c.kv_heads + kvh) * c.record + part +
                             (int64_t)Kept<TYPE>::kSize * __shfl(slot, i) * c.dim;
        for (int e = 0; e < 2; ++e)
          if (lane + 64 * e < c.dim) o[e] += w * kept_value<TYPE>(values, lane + 64 * e);
      }
    }
    T* out = reinterpret_cast<T*>(const_cast<char*>(a.o.data) + (tile.first + token) * a.o.row + head * a.o.head);
    for (int e = 0; e < 2; ++e)
      if (lane + 64 * e < c.dim) out[lane + 64 * e] = (T)(l != 0.0f ? o[e] / l : 0.0f);
  }
}

template <typename T, int TYPE>
hipError_t run(const CacheAttnArgs& a, hipStream_t stream) {
  return for_launches((int64_t)a.c.n_tiles * a.c.kv_heads, 64, [&](int64_t first, unsigned blocks) {
    sfe_cache_attn_kernel<T, TYPE><<<dim3(blocks), dim3(64), 0, stream>>>(a, first);
    return hipGetLastError();
  });
}

}  // namespace

hipError_t launch_cache_attn(const CacheAttnArgs& a, int type, int dtype, hipStream_t stream) {
  switch (type) {
    case kCacheBf16: return run<__bf16, kCacheBf16>(a, stream);
    case kCacheF16: return run<_Float16, kCacheF16>(a, stream);
    case kCacheE4m3: return dtype == kOpBf16 ? run<__bf16, kCacheE4m3>(a, stream) : run<_Float16, kCacheE4m3>(a, stream);
    default: return dtype == kOpBf16 ? run<__bf16, kCacheInt8>(a, stream) : run<_Float16, kCacheInt8>(a, stream);
  }
}

}  // namespace sfe
