// Attention over the paged 4-bit cache: softmax(scale q K^T) V for sequences of any lengths.
//
// With a stored value = code * step + offset per group of 32 channels, a score is
//   q . k = sum_groups step_g (q_g . code_g) + offset_g (sum of q_g),
// and the running maximum and sum of an online softmax need one pass over the keys.
#include "kvcache.cuh"

namespace fopt {
namespace kv {
namespace {

struct AttnArgs {
  uint16_t* o;
  const uint16_t* q;
  Cache cache;
  const int32_t* table;
  const int32_t* q_start;
  const int32_t* kv_len;
  int32_t* err;
  int batch, tokens, width, hq, group;
  float scale;
  int causal;
};

// Sequence b's query range and key count, cut to what the arguments allow.
__device__ __forceinline__ void sequence(const AttnArgs& a, int b, int& q0, int& q1, int& keys) {
  const int s0 = a.q_start[b], s1 = a.q_start[b + 1], n = a.kv_len[b];
  q0 = min(max(s0, 0), a.tokens);
  q1 = min(max(s1, q0), a.tokens);
  const int64_t room = (int64_t)a.width * a.cache.page_size;
  keys = (int)min((int64_t)max(n, 0), room);
  if (q0 != s0 || q1 != s1) atomicExch(a.err, kBadStart);
  if (keys != n) atomicExch(a.err, kBadLength);
}

// A warp per (query token, query head): lane l holds channels l, l + 32, ... (one of each group).
template <int NG>
__global__ void __launch_bounds__(256) rows_kernel(AttnArgs a) {
  constexpr int D = NG * kGroup;
  const int lane = threadIdx.x & 31;
  const int b = blockIdx.y, h = blockIdx.z, hk = h / a.group;
  int q0, q1, keys;
  sequence(a, b, q0, q1, keys);
  for (int j = blockIdx.x * 8 + (threadIdx.x >> 5); j < q1 - q0; j += gridDim.x * 8) {
    const int64_t at = ((int64_t)(q0 + j) * a.hq + h) * D;
    const int seen = a.causal ? min(keys, keys - (q1 - q0) + j + 1) : keys;
    float q[NG], acc[NG] = {}, m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g) q[g] = __uint_as_float((uint32_t)a.q[at + g * kGroup + lane] << 16) * a.scale;
    for (int i = 0; i < seen; ++i) {
      const int slot = (int)fdiv(a.cache.by_page, (uint32_t)i);
      const int page = a.table[(int64_t)b * a.width + slot];
      const bool there = page >= 0 && page < a.cache.pages;
      if (!there) atomicExch(a.err, kBadPage);
      const int64_t row = ((int64_t)(there ? page : 0) * a.cache.heads + hk) * a.cache.page_size + (i - slot * a.cache.page_size);
      float s = 0.0f, v[NG];
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        const uint32_t km = a.cache.k_scale[row * NG + g], vm = a.cache.v_scale[row * NG + g];
        const int ke = ((lane >> 3) * NG + g) * 8 + (lane & 7), ve = ((lane >> 2) * NG + g) * 4 + (lane & 3);
        const int kc = (int)(raw_nibble(a.cache.k, row * D + ke) ^ 8) - 8;
        const int vc = (int)(raw_nibble(a.cache.v, row * D + ve) ^ 8) - 8;
        const float k = fmaf((float)kc, __uint_as_float(km << 16), __uint_as_float(km & 0xffff0000u));
        v[g] = there ? fmaf((float)vc, __uint_as_float(vm << 16), __uint_as_float(vm & 0xffff0000u)) : 0.0f;
        s = there ? fmaf(q[g], k, s) : 0.0f;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
      const float top = fmaxf(m, s), keep = expf(m - top), p = expf(s - top);
      m = top;
      l = fmaf(l, keep, p);
#pragma unroll
      for (int g = 0; g < NG; ++g) acc[g] = fmaf(acc[g], keep, p * v[g]);
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      const float y = seen > 0 ? acc[g] / l : 0.0f;
      a.o[at + g * kGroup + lane] = (uint16_t)(f32_to_bf16w(__float_as_uint(y)) >> 16);
    }
  }
}

}  // namespace
}  // namespace kv
}  // namespace fopt

using namespace fopt;

extern "C" fopt_status fopt_cache_attention(fopt_ctx* ctx, void* o, const void* q, const fopt_paged_cache* cache,
                                            const int32_t* table, const int32_t* q_start, const int32_t* kv_len,
                                            int32_t batch, int32_t tokens, int32_t table_width, int32_t hq, float scale,
                                            int32_t causal) {
  return kv::checked_call(ctx, [&] {
    kv::AttnArgs a{};
    a.cache = kv::checked(cache, "fopt_cache_attention");
    require(batch >= 0 && tokens >= 0, "fopt_cache_attention: a negative count");
    require(table_width > 0, "fopt_cache_attention: an empty page table");
    require(hq > 0 && hq % cache->heads == 0, "fopt_cache_attention: query heads must be a multiple of the cache's heads");
    require(std::isfinite(scale), "fopt_cache_attention: the scale must be finite");
    require((int64_t)tokens * (hq / cache->heads) <= INT32_MAX, "fopt_cache_attention: too many query rows");
    if (ctx && (batch == 0 || tokens == 0)) return;
    require(o && q && table && q_start && kv_len, "fopt_cache_attention: null argument");
    require(((uintptr_t)o | (uintptr_t)q) % 16 == 0, "fopt_cache_attention: q and o must be 16-byte aligned");
    require(ctx != nullptr, "null context");
    DeviceGuard guard(ctx);
    a.o = (uint16_t*)o;
    a.q = (const uint16_t*)q;
    a.table = table;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.err = ctx->dev_err;
    a.batch = batch;
    a.tokens = tokens;
    a.width = table_width;
    a.hq = hq;
    a.group = hq / cache->heads;
    a.scale = scale;
    a.causal = causal != 0;
    const dim3 grid((unsigned)std::min(64, (tokens + 7) / 8), (unsigned)batch, (unsigned)hq);
    switch (cache->head_dim) {
      case 64: kv::rows_kernel<2><<<grid, 256, 0, ctx->stream>>>(a); break;
      case 128: kv::rows_kernel<4><<<grid, 256, 0, ctx->stream>>>(a); break;
      default: kv::rows_kernel<8><<<grid, 256, 0, ctx->stream>>>(a); break;
    }
    launched(ctx, "cache attention");
  });
}
