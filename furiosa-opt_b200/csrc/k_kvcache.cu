// Rotary positions, and the moves into and out of the paged 4-bit key / value cache.
//
// Rotation of a pair (a, b) by angle w = position * inv_freq: (a cos w - b sin w, b cos w + a sin w). The
// angle is kept in 2^-64 turns as an integer: position * turn modulo 2^64 is the reduced angle, exact
// for any position, where a product in f32 would be off by position * 2^-24 radians. Its sine and cosine
// are taken in f64 (sincospi) and rounded to f32 once per (token, pair), shared by all heads of the
// token through shared memory: at 32 heads that is one f64 evaluation per 64 rotated values.
//
// Quantising a group of 32 channels x: step s = bf16((max - min) / 15), offset z = bf16(min + 8 s),
// code = rint((x - z) / s) in [-8, 7]. The division is the IEEE one: bf16 inputs make exact halves
// common, and those must go to even rather than to where a reciprocal's error sends them.
//
// All three kernels move every byte once and compute little; they are bound by memory on prompts and by
// latency on single tokens.
#include "kvcache.cuh"

namespace fopt {
namespace kv {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float bf(uint32_t low16) { return __uint_as_float(low16 << 16); }

template <bool F32>
struct Elem;
template <>
struct Elem<true> {
  using T = float;
  static __device__ __forceinline__ float load(const T* p) { return *p; }
  static __device__ __forceinline__ void store(T* p, float v) { *p = v; }
};
template <>
struct Elem<false> {
  using T = uint16_t;
  static __device__ __forceinline__ float load(const T* p) { return bf(*p); }
  static __device__ __forceinline__ void store(T* p, float v) {
    *p = (uint16_t)(f32_to_bf16w(__float_as_uint(v)) >> 16);
  }
};

// N consecutive values (N = 4 or 8), as whole vectors where the address allows.
template <bool F32, int N>
__device__ __forceinline__ void load_n(const typename Elem<F32>::T* p, bool vec, float* v) {
  if (!vec) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = Elem<F32>::load(p + i);
    return;
  }
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) *(float4*)(v + 4 * i) = ((const float4*)p)[i];
  } else {
    uint32_t w[N / 2];
    if constexpr (N == 8) *(uint4*)w = *(const uint4*)p;
    else *(uint2*)w = *(const uint2*)p;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      v[2 * i] = bf(w[i] & 0xffffu);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }
}

template <bool F32>
__device__ __forceinline__ void store_8(typename Elem<F32>::T* p, const float* v) {
  if constexpr (F32) {
    ((float4*)p)[0] = *(const float4*)v;
    ((float4*)p)[1] = *(const float4*)(v + 4);
  } else {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bf16x2_rule(v[2 * i], v[2 * i + 1]);
    *(uint4*)p = *(uint4*)w;
  }
}

template <typename T>
__device__ __forceinline__ void copy_8(T* to, const T* from) {
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) ((uint4*)to)[i] = ((const uint4*)from)[i];
}

// (cos, sin) of the first `n` tokens' pairs, from their positions, into shared memory [token][pair].
__device__ __forceinline__ void angles(float2* cs, const Rope& r, const int32_t* positions, int n) {
  for (int k = threadIdx.x; k < n * r.pairs; k += kThreads) {
    const int t = k / r.pairs, p = k - t * r.pairs;
    // half turns in [-1, 1): the 64-bit product as a signed fraction
    const double half = (double)(long long)((unsigned long long)(long long)positions[t] * r.turn[p]) * 0x1p-63;
    double s, c;
    sincospi(half, &s, &c);
    cs[k] = make_float2((float)(c * r.magnitude), (float)(s * r.magnitude));
  }
}

__device__ __forceinline__ float turned_first(float a, float b, float2 cs) {
  return __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
}
__device__ __forceinline__ float turned_second(float a, float b, float2 cs) {
  return __fadd_rn(__fmul_rn(b, cs.x), __fmul_rn(a, cs.y));
}

// ---- rotary ----
struct RotaryArgs {
  void* out;
  const void* x;
  const int32_t* positions;
  int64_t x_stride, out_stride;
  int tokens, heads, dim;
  int units;         // per head: 8-channel chunks (pairs of them for HALF) when vectorised, pairs or channels if not
  FastDiv by_units;
};

// TB tokens a block: their angles first, then all their heads' units.
template <bool F32, bool VEC, int TB>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a, const __grid_constant__ Rope r) {
  using E = Elem<F32>;
  extern __shared__ float2 cs[];
  const int t0 = blockIdx.x * TB, n = min(TB, a.tokens - t0);
  angles(cs, r, a.positions + t0, n);
  __syncthreads();
  const int per_token = a.heads * a.units;
  for (int k = threadIdx.x; k < per_token; k += kThreads) {
    const int h = (int)fdiv(a.by_units, (uint32_t)k), u = k - h * a.units;
#pragma unroll
    for (int t = 0; t < TB; ++t) {
      if (t >= n) break;
      const auto* x = (const typename E::T*)a.x + (int64_t)(t0 + t) * a.x_stride + (int64_t)h * a.dim;
      auto* o = (typename E::T*)a.out + (int64_t)(t0 + t) * a.out_stride + (int64_t)h * a.dim;
      const float2* c = cs + t * r.pairs;
      if constexpr (VEC) {
        float v[8], w[8], y[8];
        if (r.interleaved) {
          if (4 * u < r.pairs) {
            load_n<F32, 8>(x + 8 * u, true, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              y[2 * i] = turned_first(v[2 * i], v[2 * i + 1], c[4 * u + i]);
              y[2 * i + 1] = turned_second(v[2 * i], v[2 * i + 1], c[4 * u + i]);
            }
            store_8<F32>(o + 8 * u, y);
          } else {
            copy_8(o + 8 * u, x + 8 * u);
          }
        } else if (8 * u < r.pairs) {
          load_n<F32, 8>(x + 8 * u, true, v);
          load_n<F32, 8>(x + 8 * u + r.pairs, true, w);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            y[i] = turned_first(v[i], w[i], c[8 * u + i]);
            w[i] = turned_second(v[i], w[i], c[8 * u + i]);
          }
          store_8<F32>(o + 8 * u, y);
          store_8<F32>(o + 8 * u + r.pairs, w);
        } else {  // past the rotated channels: units count on in whole chunks
          copy_8(o + 8 * u + r.pairs, x + 8 * u + r.pairs);
        }
      } else if (u < r.pairs) {
        const int i = r.interleaved ? 2 * u : u, j = r.interleaved ? 2 * u + 1 : u + r.pairs;
        const float p = E::load(x + i), q = E::load(x + j);
        E::store(o + i, turned_first(p, q, c[u]));
        E::store(o + j, turned_second(p, q, c[u]));
      } else {
        o[u + r.pairs] = x[u + r.pairs];
      }
    }
  }
}

// ---- append ----
struct AppendArgs {
  Cache cache;
  const void* k;
  const void* v;
  const int32_t* slots;
  const int32_t* positions;
  int64_t k_stride, v_stride;
  int32_t* err;
  int tokens;
  int k_vec, v_vec, pair_vec;  // whole-vector loads of k, of v, and of the other half of k's pairs
};

constexpr float kLargest = 0x1p100f;

__device__ __forceinline__ float storable(float x) { return x == x ? fminf(fmaxf(x, -kLargest), kLargest) : 0.0f; }

// (step, offset) of a group from its extremes, as the cache's word.
__device__ __forceinline__ uint32_t group_scale(float lo, float hi) {
  const uint32_t s = f32_to_bf16w(__float_as_uint(__fdiv_rn(__fsub_rn(hi, lo), 15.0f)));
  const uint32_t z = f32_to_bf16w(__float_as_uint(__fadd_rn(lo, __fmul_rn(8.0f, __uint_as_float(s)))));
  return s >> 16 | z;
}
__device__ __forceinline__ uint32_t code_of(float x, uint32_t scale) {
  const float s = __uint_as_float(scale << 16), z = __uint_as_float(scale & 0xffff0000u);
  const float c = s > 0.0f ? rintf(__fdiv_rn(__fsub_rn(x, z), s)) : 0.0f;
  return (uint32_t)(int)fminf(fmaxf(c, -8.0f), 7.0f) & 15u;
}

// A quad of threads per key row, thread i with channels 32 j + 8 i .. + 7 of every group j (its share of
// the image's [D % 32 / 8, D / 32, D % 8] is contiguous); eight threads per value row, thread g with
// channels 32 j + 4 g .. + 3. A group's extremes then take two or three shuffles.
template <bool F32, int NG, int TB>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a, const __grid_constant__ Rope r) {
  using E = Elem<F32>;
  constexpr int D = NG * kGroup;
  extern __shared__ float2 cs[];
  const int t0 = blockIdx.x * TB, n = min(TB, a.tokens - t0), heads = a.cache.heads;
  if (r.pairs) {
    angles(cs, r, a.positions + t0, n);
    __syncthreads();
  }
  const int capacity = a.cache.pages * a.cache.page_size;
  const int lane = threadIdx.x & 31, warp0 = threadIdx.x & ~31;

  const int k_items = n * heads * 4;
  for (int base = warp0; base < k_items; base += kThreads) {
    const int item = min(base + lane, k_items - 1);  // lanes past the end repeat the last item, unstored
    const int row = item >> 2, i = item & 3, t = row / heads, h = row - t * heads;
    const int slot = a.slots[t0 + t];
    const auto* x = (const typename E::T*)a.k + (int64_t)(t0 + t) * a.k_stride + h * D;
    const float2* c = cs + t * r.pairs;
    uint32_t words[NG], scales[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const int d = j * kGroup + i * 8;
      float v[8];
      load_n<F32, 8>(x + d, a.k_vec, v);
      if (d < 2 * r.pairs) {
        if (r.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            if (d + e < 2 * r.pairs) {
              const float2 w = c[(d + e) >> 1];
              const float p = v[e], q = v[e + 1];
              v[e] = turned_first(p, q, w);
              v[e + 1] = turned_second(p, q, w);
            }
          }
        } else if (a.pair_vec) {  // the chunk and its pairs' other halves are whole chunks
          const bool first = d < r.pairs;
          const int p0 = first ? d : d - r.pairs;
          float w[8];
          load_n<F32, 8>(x + (first ? d + r.pairs : p0), true, w);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            v[e] = first ? turned_first(v[e], w[e], c[p0 + e]) : turned_second(w[e], v[e], c[p0 + e]);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int p = d + e;
            if (p < r.pairs) v[e] = turned_first(v[e], E::load(x + p + r.pairs), c[p]);
            else if (p < 2 * r.pairs) v[e] = turned_second(E::load(x + p - r.pairs), v[e], c[p - r.pairs]);
          }
        }
      }
      float lo = INFINITY, hi = -INFINITY;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = storable(v[e]);
        lo = fminf(lo, v[e]);
        hi = fmaxf(hi, v[e]);
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      scales[j] = group_scale(lo, hi);
      words[j] = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) words[j] |= code_of(v[e], scales[j]) << (4 * e);
    }
    if (base + lane >= k_items || slot < 0) continue;
    if (slot >= capacity) {
      atomicExch(a.err, kBadSlot);
      continue;
    }
    const int64_t to = row_of(a.cache, slot, h);
    uint32_t* codes = (uint32_t*)(a.cache.k + to * (D / 2)) + i * NG;
    uint32_t* scale = a.cache.k_scale + to * NG;
    if constexpr (NG == 2) *(uint2*)codes = make_uint2(words[0], words[1]);
#pragma unroll
    for (int j = 0; j + 3 < NG; j += 4) *(uint4*)(codes + j) = make_uint4(words[j], words[j + 1], words[j + 2], words[j + 3]);
#pragma unroll
    for (int j = 0; j < NG; ++j)
      if ((j & 3) == i) scale[j] = scales[j];
  }

  const int v_items = n * heads * 8;
  for (int base = warp0; base < v_items; base += kThreads) {
    const int item = min(base + lane, v_items - 1);
    const int row = item >> 3, g = item & 7, t = row / heads, h = row - t * heads;
    const int slot = a.slots[t0 + t];
    const auto* x = (const typename E::T*)a.v + (int64_t)(t0 + t) * a.v_stride + h * D;
    uint32_t words[NG / 2], scales[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      float v[4];
      load_n<F32, 4>(x + j * kGroup + g * 4, a.v_vec, v);
      float lo = INFINITY, hi = -INFINITY;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = storable(v[e]);
        lo = fminf(lo, v[e]);
        hi = fmaxf(hi, v[e]);
      }
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      }
      scales[j] = group_scale(lo, hi);
      uint32_t w = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) w |= code_of(v[e], scales[j]) << (4 * e);
      if (j & 1) words[j >> 1] |= w << 16;
      else words[j >> 1] = w;
    }
    if (base + lane >= v_items || slot < 0) continue;
    if (slot >= capacity) {
      atomicExch(a.err, kBadSlot);
      continue;
    }
    const int64_t to = row_of(a.cache, slot, h);
    uint32_t* codes = (uint32_t*)(a.cache.v + to * (D / 2)) + g * (NG / 2);
    uint32_t* scale = a.cache.v_scale + to * NG;
    if constexpr (NG == 2) codes[0] = words[0];
    if constexpr (NG == 4) *(uint2*)codes = make_uint2(words[0], words[1]);
    if constexpr (NG == 8) *(uint4*)codes = make_uint4(words[0], words[1], words[2], words[3]);
#pragma unroll
    for (int j = 0; j < NG; ++j)
      if (j == g) scale[j] = scales[j];
  }
}

// ---- read ----
// A thread per 32-bit word of codes: 8 neighbouring channels of a key, or 4 of each of two groups of a value.
template <bool F32, int NG>
__global__ void __launch_bounds__(kThreads) read_kernel(Cache cache, void* out_k, void* out_v, const int32_t* slots,
                                                        int n, int32_t* err) {
  using E = Elem<F32>;
  constexpr int D = NG * kGroup, W = D / 8;
  const int capacity = cache.pages * cache.page_size;
  const int64_t total = (int64_t)n * cache.heads * W;
  for (int64_t f = blockIdx.x * (int64_t)kThreads + threadIdx.x; f < 2 * total; f += (int64_t)gridDim.x * kThreads) {
    const bool value = f >= total;
    const int64_t q = value ? f - total : f;
    const int w = (int)(q % W);
    const int64_t row = q / W;
    const int64_t token = row / cache.heads;
    const int h = (int)(row - token * cache.heads), slot = slots[token];
    if (slot < 0) continue;
    if (slot >= capacity) {
      atomicExch(err, kBadSlot);
      continue;
    }
    const int64_t from = row_of(cache, slot, h);
    const uint32_t codes = ((const uint32_t*)((value ? cache.v : cache.k) + from * (D / 2)))[w];
    const uint32_t* scale = (value ? cache.v_scale : cache.k_scale) + from * NG;
    auto* o = (typename E::T*)(value ? out_v : out_k) + row * D;
    float y[8];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      // word w holds group w % NG (a key's), or groups 2 (w % (NG / 2)) and the next (a value's)
      const uint32_t m = scale[value ? 2 * (w % (NG / 2)) + half : w % NG];
      const float s = __uint_as_float(m << 16), z = __uint_as_float(m & 0xffff0000u);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = (int)(codes << (28 - 16 * half - 4 * e)) >> 28;
        y[4 * half + e] = fmaf((float)c, s, z);
      }
    }
    if (!value) {
      store_8<F32>(o + (w % NG) * kGroup + (w / NG) * 8, y);
    } else {
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        auto* to = o + (2 * (w % (NG / 2)) + half) * kGroup + (w / (NG / 2)) * 4;
        if constexpr (F32) *(float4*)to = *(float4*)(y + 4 * half);
        else
          *(uint2*)to = make_uint2(bf16x2_rule(y[4 * half], y[4 * half + 1]), bf16x2_rule(y[4 * half + 2], y[4 * half + 3]));
      }
    }
  }
}

bool aligned16(const void* p, int64_t stride_elems, int elem_bytes) {
  return (uintptr_t)p % 16 == 0 && stride_elems * elem_bytes % 16 == 0;
}

template <bool F32, int TB>
void launch_append(fopt_ctx* ctx, const AppendArgs& a, const Rope& r, int dim) {
  const int grid = (a.tokens + TB - 1) / TB;
  const size_t smem = (size_t)TB * r.pairs * sizeof(float2);
  switch (dim) {
    case 64: append_kernel<F32, 2, TB><<<grid, kThreads, smem, ctx->stream>>>(a, r); break;
    case 128: append_kernel<F32, 4, TB><<<grid, kThreads, smem, ctx->stream>>>(a, r); break;
    default: append_kernel<F32, 8, TB><<<grid, kThreads, smem, ctx->stream>>>(a, r); break;
  }
  launched(ctx, "cache append");
}

template <bool F32, bool VEC>
void launch_rotary(fopt_ctx* ctx, const RotaryArgs& a, const Rope& r, bool wide) {
  // four tokens share a block's angles once there are blocks enough for the SMs
  if (wide)
    rotary_kernel<F32, VEC, 4><<<(a.tokens + 3) / 4, kThreads, 4 * r.pairs * sizeof(float2), ctx->stream>>>(a, r);
  else
    rotary_kernel<F32, VEC, 1><<<a.tokens, kThreads, r.pairs * sizeof(float2), ctx->stream>>>(a, r);
  launched(ctx, "rotary");
}

}  // namespace
}  // namespace kv
}  // namespace fopt

using namespace fopt;

extern "C" {

fopt_status fopt_rope_create(const double* inv_freq, int32_t n_pairs, fopt_rope_layout layout, double magnitude,
                             fopt_rope** out) {
  try {
    if (out) *out = nullptr;
    require(inv_freq && out, "fopt_rope_create: null argument");
    require(n_pairs > 0 && n_pairs <= kv::kMaxPairs, "fopt_rope_create: 1 to 128 pairs");
    require(layout == FOPT_ROPE_HALF || layout == FOPT_ROPE_INTERLEAVED, "fopt_rope_create: unknown layout");
    require(std::isfinite(magnitude), "fopt_rope_create: the magnitude must be finite");
    auto r = std::make_unique<fopt_rope>();
    r->r = kv::Rope{};
    for (int i = 0; i < n_pairs; ++i) {
      require(std::isfinite(inv_freq[i]), "fopt_rope_create: frequencies must be finite");
      // turns per position in an extended double (64 bits of mantissa), the whole turns dropped
      long double turns = (long double)inv_freq[i] / 6.283185307179586476925286766559005768L;
      turns -= floorl(turns);
      long double scaled = turns * 18446744073709551616.0L;  // 2^64
      r->r.turn[i] = scaled >= 18446744073709551615.5L ? 0ull : (unsigned long long)roundl(scaled);
    }
    r->r.magnitude = magnitude;
    r->r.pairs = n_pairs;
    r->r.interleaved = layout == FOPT_ROPE_INTERLEAVED;
    *out = r.release();
    return FOPT_OK;
  } catch (const Fail& f) {
    g_noctx_err = f.msg;
    return f.code;
  } catch (const std::exception& e) {
    g_noctx_err = e.what();
    return FOPT_ERR_INVALID;
  }
}

fopt_status fopt_rope_free(fopt_rope* rope) {
  delete rope;
  return FOPT_OK;
}

fopt_status fopt_rotary(fopt_ctx* ctx, void* out, const void* x, fopt_dtype dtype, const int32_t* positions,
                        const fopt_rope* rope, int32_t tokens, int32_t heads, int32_t head_dim, int64_t x_stride,
                        int64_t out_stride) {
  return kv::checked_call(ctx, [&] {
    require(rope != nullptr, "fopt_rotary: null argument");
    require(dtype == FOPT_BF16 || dtype == FOPT_F32, "fopt_rotary: bf16 or f32 values");
    require(tokens >= 0 && heads > 0 && head_dim > 0, "fopt_rotary: empty heads");
    const kv::Rope& r = rope->r;
    require(2 * r.pairs <= head_dim, "fopt_rotary: more rotated channels than the head has");
    const int64_t row = (int64_t)heads * head_dim;
    require(row <= INT32_MAX, "fopt_rotary: a token's heads past 2^31 elements");
    require(x_stride >= row && out_stride >= row, "fopt_rotary: a token stride below heads * head_dim");
    require(out != x || x_stride == out_stride, "fopt_rotary: in place needs equal strides");
    if (ctx && tokens == 0) return;
    require(out && x && positions, "fopt_rotary: null argument");
    require(ctx != nullptr, "null context");
    DeviceGuard guard(ctx);
    const bool f32 = dtype == FOPT_F32;
    const int sz = f32 ? 4 : 2;
    const int tail = out == x ? 0 : head_dim - 2 * r.pairs;  // in place, the channels past the pairs stay
    const bool vec = head_dim % 8 == 0 && (2 * r.pairs) % 8 == 0 && (r.interleaved || r.pairs % 8 == 0) &&
                     kv::aligned16(x, x_stride, sz) && kv::aligned16(out, out_stride, sz);
    const int units = vec ? (r.interleaved ? 2 * r.pairs : r.pairs) / 8 + tail / 8 : r.pairs + tail;
    kv::RotaryArgs a{out, x, positions, x_stride, out_stride, tokens, heads, head_dim, units, make_fastdiv((uint32_t)units)};
    const bool wide = tokens >= 4 * 148;
    if (f32) vec ? kv::launch_rotary<true, true>(ctx, a, r, wide) : kv::launch_rotary<true, false>(ctx, a, r, wide);
    else vec ? kv::launch_rotary<false, true>(ctx, a, r, wide) : kv::launch_rotary<false, false>(ctx, a, r, wide);
  });
}

fopt_status fopt_cache_append(fopt_ctx* ctx, const fopt_paged_cache* cache, const void* k, const void* v,
                              fopt_dtype dtype, int64_t k_stride, int64_t v_stride, const int32_t* slots,
                              const int32_t* positions, const fopt_rope* rope, int32_t tokens) {
  return kv::checked_call(ctx, [&] {
    kv::AppendArgs a{};
    a.cache = kv::checked(cache, "fopt_cache_append");
    require(dtype == FOPT_BF16 || dtype == FOPT_F32, "fopt_cache_append: bf16 or f32 keys and values");
    require(tokens >= 0, "fopt_cache_append: a negative token count");
    const int dim = cache->head_dim;
    const int64_t row = (int64_t)cache->heads * dim;
    require(row <= INT32_MAX / 16, "fopt_cache_append: too many heads");
    require(k_stride >= row && v_stride >= row, "fopt_cache_append: a token stride below heads * head_dim");
    static const kv::Rope none{};
    const kv::Rope& r = rope ? rope->r : none;
    require(2 * r.pairs <= dim, "fopt_cache_append: more rotated channels than the head has");
    if (ctx && tokens == 0) return;
    require(k && v && slots && (positions || !rope), "fopt_cache_append: null argument");
    require(ctx != nullptr, "null context");
    DeviceGuard guard(ctx);
    const bool f32 = dtype == FOPT_F32;
    a.k = k;
    a.v = v;
    a.slots = slots;
    a.positions = positions;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.err = ctx->dev_err;
    a.tokens = tokens;
    a.k_vec = kv::aligned16(k, k_stride, f32 ? 4 : 2);
    a.v_vec = kv::aligned16(v, v_stride, f32 ? 4 : 2);
    a.pair_vec = a.k_vec && r.pairs % 8 == 0;
    const bool wide = tokens >= 4 * 148;  // as in the rotation
    if (f32) wide ? kv::launch_append<true, 4>(ctx, a, r, dim) : kv::launch_append<true, 1>(ctx, a, r, dim);
    else wide ? kv::launch_append<false, 4>(ctx, a, r, dim) : kv::launch_append<false, 1>(ctx, a, r, dim);
  });
}

fopt_status fopt_cache_read(fopt_ctx* ctx, void* out_k, void* out_v, fopt_dtype dtype, const fopt_paged_cache* cache,
                            const int32_t* slots, int32_t n) {
  return kv::checked_call(ctx, [&] {
    const kv::Cache c = kv::checked(cache, "fopt_cache_read");
    require(dtype == FOPT_BF16 || dtype == FOPT_F32, "fopt_cache_read: bf16 or f32 values");
    require(n >= 0, "fopt_cache_read: a negative slot count");
    if (ctx && n == 0) return;
    require(out_k && out_v && slots, "fopt_cache_read: null argument");
    require(((uintptr_t)out_k | (uintptr_t)out_v) % 16 == 0, "fopt_cache_read: outputs must be 16-byte aligned");
    require(ctx != nullptr, "null context");
    DeviceGuard guard(ctx);
    const int dim = cache->head_dim;
    const int64_t blocks = (2 * (int64_t)n * c.heads * (dim / 8) + kv::kThreads - 1) / kv::kThreads;
    const int grid = (int)std::min<int64_t>(blocks, 148 * 32);
    auto go = [&](auto kernel) {
      kernel<<<grid, kv::kThreads, 0, ctx->stream>>>(c, out_k, out_v, slots, n, ctx->dev_err);
      launched(ctx, "cache read");
    };
    if (dtype == FOPT_F32)
      dim == 64 ? go(kv::read_kernel<true, 2>) : dim == 128 ? go(kv::read_kernel<true, 4>) : go(kv::read_kernel<true, 8>);
    else
      dim == 64 ? go(kv::read_kernel<false, 2>) : dim == 128 ? go(kv::read_kernel<false, 4>) : go(kv::read_kernel<false, 8>);
  });
}

}  // extern "C"
