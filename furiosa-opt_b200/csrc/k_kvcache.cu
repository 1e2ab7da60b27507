// Rotary positions, and the moves into and out of the paged 4-bit key / value cache.
//
// Rotation of a pair (a, b) by angle w = position * inv_freq: (a cos w - b sin w, b cos w + a sin w). The
// angle is kept in 2^-64 turns as an integer: position * turn modulo 2^64 is the reduced angle, exact
// for any position, where a product in f32 would be off by position * 2^-24 radians. Its sine and cosine
// are taken in f64 (sincospi) and rounded to f32 once per (token, pair), shared by all heads of the
// token through shared memory: at 32 heads that is one f64 evaluation per 64 rotated values.
//
// Quantising a group of 32 channels x: step s = bf16((max - min) / 15), offset z = bf16(min + 8 s),
// code = rint((x - z) / s) in [-8, 7], the quotient rounded as IEEE division rounds it: bf16 inputs make exact halves
// common, and those must go to even rather than to where a reciprocal's error sends them.
//
// What bounds them, on inputs that come from HBM: the rotation memory (16.3 us for 4096 tokens of 32 heads of 128 in
// bf16, 67 MB: 4.1 TB/s, 0.63 of a copy's rate; 12.4 us where L2 still holds them), the append instructions (16.4 us for
// 4096 tokens of 8 heads of 128, 21 MB, where memory would take 3.3; 14.6 from L2), the read the values' stores, which
// fill half a line each (12.3 us for 4608 such slots; 10.3 from L2), single tokens the launch (4.3 us each).
#include "kvcache.cuh"

namespace fopt {
namespace kv {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ float bf(uint32_t low16) { return __uint_as_float(low16 << 16); }

// x, a subnormal as a zero of its sign.
__device__ __forceinline__ float flushed(float x) {
  float y;
  asm("mul.ftz.f32 %0, %1, 0f3F800000;" : "=f"(y) : "f"(x));
  return y;
}
// bf16x2_rule without its selects, for halves that are not NaN.
__device__ __forceinline__ uint32_t bf16x2_of(float lo, float hi) {
  uint32_t w;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(flushed(hi)), "f"(flushed(lo)));
  return w;
}

template <bool F32>
struct Elem;
template <>
struct Elem<true> {
  using T = float;
  static __device__ __forceinline__ float value(T v) { return v; }
  static __device__ __forceinline__ void store(T* p, float v) { *p = v; }
};
template <>
struct Elem<false> {
  using T = uint16_t;
  static __device__ __forceinline__ float value(T v) { return bf(v); }
  static __device__ __forceinline__ void store(T* p, float v) { *p = v == v ? (uint16_t)bf16x2_of(v, 0.0f) : 0x7fc0; }
};

// Stores N values (4 or 8). The selects of bf16x2_rule cost more than all else in these kernels, so they are left
// to the words that need them: 0 x + sum is NaN if any x is NaN (or infinite, which the rule rounds alike).
template <bool F32, int N>
__device__ __forceinline__ void store_n(typename Elem<F32>::T* p, const float* v) {
  uint32_t w[F32 ? N : N / 2];
  if constexpr (F32) {
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v[i]);
  } else {
    uint32_t sum = 0;
#pragma unroll
    for (int i = 0; i < N / 2; ++i) {
      w[i] = bf16x2_of(v[2 * i], v[2 * i + 1]);
      asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(sum) : "r"(w[i]), "r"(0u));
    }
    if ((sum & 0x7fff7fffu) != 0) {  // zeros, else NaN
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = bf16x2_rule(v[2 * i], v[2 * i + 1]);
    }
  }
  if constexpr (sizeof(w) == 8) *(uint2*)p = *(const uint2*)w;
#pragma unroll
  for (int i = 0; i < (int)sizeof(w) / 16; ++i) ((uint4*)p)[i] = ((const uint4*)w)[i];
}

// N values (4 or 8) as they are in memory, moved in whole vectors where the address allows.
template <bool F32, int N = 8>
struct Raw {
  static constexpr int kWords = F32 ? N : N / 2;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const void* p) {
    if constexpr (kWords == 2) *(uint2*)w = *(const uint2*)p;
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) ((uint4*)w)[i] = ((const uint4*)p)[i];
  }
  __device__ __forceinline__ void store(void* p) const {
    if constexpr (kWords == 2) *(uint2*)p = *(const uint2*)w;
#pragma unroll
    for (int i = 0; i < kWords / 4; ++i) ((uint4*)p)[i] = ((const uint4*)w)[i];
  }
  __device__ __forceinline__ void put(int i, typename Elem<F32>::T v) {
    if constexpr (F32) w[i] = __float_as_uint(v);
    else w[i / 2] = i % 2 ? (w[i / 2] & 0xffffu) | (uint32_t)v << 16 : v;
  }
  __device__ __forceinline__ void load(const typename Elem<F32>::T* p, bool vec) {
    if (vec) return load((const void*)p);
#pragma unroll
    for (int i = 0; i < N; ++i) put(i, p[i]);
  }
  __device__ __forceinline__ void values(float* v) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (F32) v[i] = __uint_as_float(w[i]);
      else v[i] = i % 2 ? __uint_as_float(w[i / 2] & 0xffff0000u) : bf(w[i / 2] & 0xffffu);
    }
  }
};

// (cos, sin) of the first `n` tokens' pairs, from their positions, into shared memory: [token][pair], or, for threads
// that take 2^shift neighbouring pairs each, [token][two of a thread's pairs][thread][pair of the two], since lanes
// that read 64 bytes apart share banks (which made the rotation of 4096 tokens of 32 heads of 128 take 16.5 us, not 12.4, from L2).
__device__ __forceinline__ void angles(float2* cs, const Rope& r, const int32_t* positions, int n, int shift) {
  // by a plain address: lanes that differ in it take turns at the constant bank
  const unsigned long long* turn = r.turn;
  asm("" : "+l"(turn));
  for (int k = threadIdx.x; k < n * r.pairs; k += kThreads) {
    const int t = k / r.pairs, p = k - t * r.pairs;
    // half turns in [-1, 1): the 64-bit product as a signed fraction
    const double half = (double)(long long)((unsigned long long)(long long)positions[t] * turn[p]) * 0x1p-63;
    double s, c;
    sincospi(half, &s, &c);
    const int to = shift ? t * r.pairs + ((((p & ((1 << shift) - 1)) >> 1) * (r.pairs >> shift) + (p >> shift)) << 1 | (p & 1)) : k;
    cs[to] = make_float2((float)(c * r.magnitude), (float)(s * r.magnitude));
  }
}
// N of them from the place of the first two, with `units` threads' pairs between.
template <int N>
__device__ __forceinline__ void load_angles(float2* c, const float2* at, int units) {
#pragma unroll
  for (int i = 0; i < N / 2; ++i) *(float4*)(c + 2 * i) = *(const float4*)(at + 2 * i * units);
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
  int each;          // tokens a block
  int units;         // per head: 8-channel chunks (pairs of them for HALF) when vectorised, pairs or channels if not
  FastDiv by_units, by_heads;
};

// A block has `each` tokens. With vectors their units are one range, of which a thread has AHEAD at a time, a block's
// threads apart, on their way while the angles are computed (the sines take about as long as the loads). Without,
// most time goes into addresses, so a thread takes the same unit of kOnes tokens: 5878 tokens of 21 heads of 96 with
// 35 pairs in bf16 take 22.7 us, bound by instructions (from L2; 45 as one range, 35 token after token).
constexpr int kOnes = 4;
template <bool F32, bool VEC, int AHEAD>
__global__ void __launch_bounds__(kThreads) rotary_kernel(RotaryArgs a, const __grid_constant__ Rope r) {
  using E = Elem<F32>;
  using T = typename E::T;
  extern __shared__ __align__(16) float2 cs[];
  const int t0 = blockIdx.x * a.each, n = min(a.each, a.tokens - t0);
  if constexpr (!VEC) {
    angles(cs, r, a.positions + t0, n, 0);
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < (uint32_t)(a.heads * a.units); k += kThreads) {
      const int h = (int)fdiv(a.by_units, k), u = (int)k - h * a.units;
      const bool pair = u < r.pairs;
      const int i = !pair ? u + r.pairs : r.interleaved ? 2 * u : u, j = !pair ? i : r.interleaved ? i + 1 : u + r.pairs;
      const T* from = (const T*)a.x + t0 * a.x_stride + (int64_t)h * a.dim;
      T* to = (T*)a.out + t0 * a.out_stride + (int64_t)h * a.dim;
      T p[kOnes], q[kOnes];
#pragma unroll
      for (int t = 0; t < kOnes; ++t) {
        if (t >= n) continue;
        p[t] = from[t * a.x_stride + i];
        q[t] = from[t * a.x_stride + j];
      }
#pragma unroll
      for (int t = 0; t < kOnes; ++t) {
        if (t >= n) continue;
        if (pair) {
          const float2 c = cs[t * r.pairs + u];
          const float x = E::value(p[t]), y = E::value(q[t]);
          E::store(to + t * a.out_stride + i, turned_first(x, y, c));
          E::store(to + t * a.out_stride + j, turned_second(x, y, c));
        } else {
          to[t * a.out_stride + i] = p[t];
        }
      }
    }
    return;
  }
  const uint32_t total = n * a.heads * a.units;  // a token's are below 2^31
  const int shift = r.interleaved ? 2 : 3;
  bool turned = false;
  for (uint32_t k0 = threadIdx.x; !turned || k0 < total; k0 += kThreads * AHEAD) {
    T* to[AHEAD];
    const float2* c[AHEAD];
    bool rotated[AHEAD];
    Raw<F32> v[AHEAD], w[AHEAD];  // the unit's values and, of pairs that lie apart, the second ones
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const uint32_t k = k0 + i * kThreads;
      if (k >= total) continue;
      const int row = (int)fdiv(a.by_units, k), u = (int)k - row * a.units;
      const int t = (int)fdiv(a.by_heads, (uint32_t)row), h = row - t * a.heads;
      rotated[i] = r.interleaved ? 4 * u < r.pairs : 8 * u < r.pairs;
      // past the rotated channels units count on in whole chunks
      const int64_t at = (int64_t)h * a.dim + (r.interleaved || rotated[i] ? 8 * u : 8 * u + r.pairs);
      const T* from = (const T*)a.x + (t0 + t) * a.x_stride + at;
      to[i] = (T*)a.out + (t0 + t) * a.out_stride + at;
      c[i] = cs + t * r.pairs + 2 * u;
      v[i].load(from);
      if (rotated[i] && !r.interleaved) w[i].load(from + r.pairs);
    }
    if (!turned) {
      angles(cs, r, a.positions + t0, n, shift);
      __syncthreads();
      turned = true;
    }
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (k0 + i * kThreads >= total) continue;
      if (!rotated[i]) {
        v[i].store(to[i]);
        continue;
      }
      float x[8], y[8], z[8];
      float2 k[8];
      v[i].values(x);
      if (r.interleaved) {
        load_angles<4>(k, c[i], r.pairs >> 2);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[2 * e] = turned_first(x[2 * e], x[2 * e + 1], k[e]);
          y[2 * e + 1] = turned_second(x[2 * e], x[2 * e + 1], k[e]);
        }
      } else {
        load_angles<8>(k, c[i], r.pairs >> 3);
        w[i].values(z);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          y[e] = turned_first(x[e], z[e], k[e]);
          z[e] = turned_second(x[e], z[e], k[e]);
        }
        store_n<F32, 8>(to[i] + r.pairs, z);
      }
      store_n<F32, 8>(to[i], y);
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
  int32_t* bad;
  int tokens;
  int each;          // tokens a block
  FastDiv by_heads;
  int k_vec, v_vec;  // whole-vector loads of k and of v
  int pair_vec;      // a thread's eight channels are of whole pairs or of none, the other halves' too and read as vectors
};

constexpr float kLargest = 0x1p100f;
constexpr float kSmallStep = 0x1p-100f;  // remainders of smaller steps may underflow

__device__ __forceinline__ float storable(float x) { return x == x ? fminf(fmaxf(x, -kLargest), kLargest) : 0.0f; }

// (step, offset) of a group from its extremes, as the cache's word. For a range d that is not tiny, q + (d - 15 q) / 15
// with q = d / 15 to an ulp is the quotient to 2^-46, and no quotient of a 24-bit number by 15 is nearer than 2^-29 to
// the middle of two neighbours: it rounds as the division does.
__device__ __forceinline__ uint32_t group_scale(float lo, float hi) {
  const float d = __fsub_rn(hi, lo);
  constexpr float r15 = 1.0f / 15.0f;
  float s = __fmul_rn(d, r15);
  s = d >= kSmallStep ? __fmaf_rn(__fmaf_rn(-s, 15.0f, d), r15, s) : __fdiv_rn(d, 15.0f);
  const uint32_t step = bf16x2_of(s, 0.0f);
  return bf16x2_of(__uint_as_float(step << 16), __fadd_rn(lo, __fmul_rn(8.0f, __uint_as_float(step << 16))));
}
__device__ __forceinline__ uint32_t code_of(float x, uint32_t scale) {
  const float s = __uint_as_float(scale << 16), z = __uint_as_float(scale & 0xffff0000u);
  const float c = s > 0.0f ? rintf(__fdiv_rn(__fsub_rn(x, z), s)) : 0.0f;
  return (uint32_t)(int)fminf(fmaxf(c, -8.0f), 7.0f) & 15u;
}

// The codes without a division for each, by the correction step of Markstein's division (IBM J. Res. Dev. 34, 1990):
// with t = x - z and r = 1 / s to an ulp, q = t r is off by less than 2^-22 of itself; the remainder t - q s is exact
// (s has 8 bits, so it is a multiple of 2^-30 of the binade of t and below 2^-20 of it), and q + (t - q s) r is t / s to
// 2^-45 before its rounding. Where t / s is a half, that rounds to it; where it is not, t differs from that multiple of
// half a step by its own last place at least, which is more than half a last place of the half (again as s has 8 bits):
// so the sum lies on the right side, as the division's rounded quotient does. No quotient passes 2^20: a range that is
// not zero is at least 2^-23 of the values. A step below 2^-100, whose remainders could underflow, takes the division.
struct Steps {
  float s, z, r;
  __device__ __forceinline__ explicit Steps(uint32_t scale) {
    s = __uint_as_float(scale << 16);
    z = __uint_as_float(scale & 0xffff0000u);
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
    if (s == 0.0f) r = 0.0f;  // no step: codes of zero
  }
  __device__ __forceinline__ bool small() const { return s > 0.0f && s < kSmallStep; }
  // 0x4b400000 + code
  __device__ __forceinline__ uint32_t code(float x) const {
    const float t = __fsub_rn(x, z), q = __fmul_rn(t, r), c = __fmaf_rn(__fmaf_rn(-q, s, t), r, q);
    return __float_as_uint(__fadd_rn(fminf(fmaxf(c, -8.0f), 7.0f), 0x1.8p23f));
  }
};

// A thread per two 32-bit words of codes, D / 16 neighbouring lanes to a row. Word i * NG + j of a key is channels
// 32 j + 8 i .. + 7; a thread has 16 neighbouring channels, its group's two threads lie NG apart. Word
// g * (NG / 2) + j of a value is channels 4 g .. + 3 of groups 2 j and 2 j + 1; a thread has 8 neighbouring channels
// of both, and their four threads lie NG / 2 apart. Extremes cross by shuffles. Instructions bound this kernel on
// prompts; shuffles, scales and addresses are a large part of them, so a thread has as many values as that allows:
// 14.6 us for 4096 tokens of 8 heads of 128 in bf16 from L2, where a thread per word with the tokens of its block one after
// the other took 18 us, and all groups' channels to four and eight threads a row, with a division a value, 27 us.
template <bool F32, int NG>
__global__ void __launch_bounds__(kThreads) append_kernel(AppendArgs a, const __grid_constant__ Rope r) {
  constexpr int D = NG * kGroup, W = D / 16;
  constexpr uint32_t kAll = 0xffffffffu;
  extern __shared__ __align__(16) float2 cs[];
  const int t0 = blockIdx.x * a.each, n = min(a.each, a.tokens - t0), heads = a.cache.heads;
  const int keys = n * heads * W, items = 2 * keys;
  const int lane = threadIdx.x & 31;
  bool turned = false;
  for (int base = threadIdx.x & ~31; !turned || base < items; base += kThreads) {
    // lanes past the end repeat the last item, unstored
    const int item = min(base + lane, items - 1), w = item % W;
    const bool value = item >= keys, live = base + lane < items;
    const int row = (item - (value ? keys : 0)) / W, t = (int)fdiv(a.by_heads, (uint32_t)row), h = row - t * heads;
    const int d = value ? (w % (NG / 2)) * 2 * kGroup + (w / (NG / 2)) * 8 : (w % NG) * kGroup + (w / NG) * 16;
    const auto* from = (const typename Elem<F32>::T*)(value ? a.v : a.k) + (t0 + t) * (value ? a.v_stride : a.k_stride) + h * D + d;
    const int slot = a.slots[t0 + t];
    // v[i]: the eight values of word i. A key's are neighbours; a value's are four of each of its groups.
    Raw<F32> v[2], y[2];
    if (value) {
      Raw<F32> one, two;
      one.load(from, a.v_vec);
      two.load(from + kGroup, a.v_vec);
      constexpr int half = Raw<F32>::kWords / 2;
#pragma unroll
      for (int i = 0; i < half; ++i) {
        v[0].w[i] = one.w[i];
        v[0].w[half + i] = two.w[i];
        v[1].w[i] = one.w[half + i];
        v[1].w[half + i] = two.w[half + i];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[i].load(from + 8 * i, a.k_vec);
        const int c = d + 8 * i;
        if (c >= 2 * r.pairs || r.interleaved) continue;
        // the other values of the pairs; a first half's with their signs turned, for it takes -sin of them
        if (a.pair_vec) {
          y[i].load(from + 8 * i + (c < r.pairs ? r.pairs : -r.pairs));
          const uint32_t sign = c < r.pairs ? (F32 ? 0x80000000u : 0x80008000u) : 0u;
#pragma unroll
          for (int e = 0; e < Raw<F32>::kWords; ++e) y[i].w[e] ^= sign;
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int p = c + e;
            y[i].put(e, from[p - d + (p < r.pairs ? r.pairs : p < 2 * r.pairs ? -r.pairs : 0)]);
          }
        }
      }
    }
    if (!turned) {
      // values do not wait for the angles: items go from keys to values, so a warp without keys now has none later
      if (r.pairs) {
        angles(cs, r, a.positions + t0, n, !a.pair_vec ? 0 : r.interleaved ? 2 : 3);
        if (base < keys) asm volatile("barrier.cta.sync 1, %0;" ::"n"(kThreads) : "memory");
        else asm volatile("barrier.cta.arrive 1, %0;" ::"n"(kThreads) : "memory");
      }
      turned = true;
    }
    float f[2][8];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      v[i].values(f[i]);
      const int c = d + 8 * i;
      if (value || c >= 2 * r.pairs) continue;
      const float2* k = cs + t * r.pairs;
      float2 turn[8];
      if (r.interleaved) {
        if (a.pair_vec) {
          load_angles<4>(turn, k + (c >> 3) * 2, r.pairs >> 2);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) turn[e] = k[min((c >> 1) + e, r.pairs - 1)];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if ((c >> 1) + e < r.pairs) {
            const float p = f[i][2 * e], q = f[i][2 * e + 1];
            f[i][2 * e] = turned_first(p, q, turn[e]);
            f[i][2 * e + 1] = turned_second(p, q, turn[e]);
          }
        }
      } else {
        float other[8];
        y[i].values(other);
        if (a.pair_vec) {
          load_angles<8>(turn, k + ((c < r.pairs ? c : c - r.pairs) >> 3) * 2, r.pairs >> 3);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[i][e] = __fadd_rn(__fmul_rn(f[i][e], turn[e].x), __fmul_rn(other[e], turn[e].y));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const int p = c + e;
            if (p < r.pairs) f[i][e] = turned_first(f[i][e], other[e], k[p]);
            else if (p < 2 * r.pairs) f[i][e] = turned_second(other[e], f[i][e], k[p - r.pairs]);
          }
        }
      }
    }
    // extremes of the first and of the last four of both words
    float lo[2], hi[2];
    auto extremes = [&] {
#pragma unroll
      for (int z = 0; z < 2; ++z) {
        lo[z] = hi[z] = f[0][4 * z];
#pragma unroll
        for (int e = 1; e < 8; ++e) {
          lo[z] = fminf(lo[z], f[e / 4][4 * z + e % 4]);
          hi[z] = fmaxf(hi[z], f[e / 4][4 * z + e % 4]);
        }
      }
    };
    extremes();
    float total[2] = {0.0f, 0.0f};  // NaN if a value is (or if infinities meet, which the extremes show)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      total[0] += f[0][e];
      total[1] += f[1][e];
    }
    if (!(fminf(lo[0], lo[1]) >= -kLargest && fmaxf(hi[0], hi[1]) <= kLargest && total[0] == total[0] && total[1] == total[1])) {
#pragma unroll
      for (int e = 0; e < 16; ++e) f[e / 8][e % 8] = storable(f[e / 8][e % 8]);
      extremes();
    }
    // A value's two neighbours take a group each: what each has of the other's changes hands.
    const bool upper = value && (w & (NG / 2));
    const float gl = __shfl_xor_sync(kAll, upper ? lo[0] : lo[1], NG / 2), gu = __shfl_xor_sync(kAll, upper ? hi[0] : hi[1], NG / 2);
    float l = fminf(upper ? lo[1] : lo[0], value ? gl : lo[1]), u = fmaxf(upper ? hi[1] : hi[0], value ? gu : hi[1]);
    l = fminf(l, __shfl_xor_sync(kAll, l, NG));
    u = fmaxf(u, __shfl_xor_sync(kAll, u, NG));
    const uint32_t mine = group_scale(l, u), theirs = __shfl_xor_sync(kAll, mine, NG / 2);
    const uint32_t scale0 = value && upper ? theirs : mine, scale1 = value && !upper ? theirs : mine;
    const Steps s0(scale0), s1(scale1);
    uint32_t word[2] = {0, 0};
    if (s0.small() || s1.small()) {
#pragma unroll
      for (int e = 0; e < 16; ++e) word[e / 8] |= code_of(f[e / 8][e % 8], e & 4 ? scale1 : scale0) << (4 * (e % 8));
    } else {
      // the sum of code + 8 at each place, and of the constants that come with them
#pragma unroll
      for (int e = 0; e < 16; ++e) word[e / 8] += (e & 4 ? s1 : s0).code(f[e / 8][e % 8]) << (4 * (e % 8));
#pragma unroll
      for (int i = 0; i < 2; ++i) word[i] = (word[i] - (0x4b400000u - 8u) * 0x11111111u) ^ 0x88888888u;
    }
    if (!live || slot < 0) continue;
    if (slot >= a.cache.pages * a.cache.page_size) {
      atomicExch(a.bad, kBadSlot);
      continue;
    }
    const int64_t to = row_of(a.cache, slot, h);
    uint32_t* codes = (uint32_t*)((value ? a.cache.v : a.cache.k) + to * (D / 2));
    uint32_t* scales = (value ? a.cache.v_scale : a.cache.k_scale) + to * NG;
    const int pitch = value ? NG / 2 : NG, j = w % pitch;
    codes += (w - j) * 2 + j;
    codes[0] = word[0];
    codes[pitch] = word[1];
    if (w >= pitch) continue;
    if (value) *(uint2*)(scales + 2 * j) = make_uint2(scale0, scale1);
    else scales[j] = scale0;
  }
}

// ---- read ----
// A thread per word, as they are stored: 8 neighbouring channels of a key, or 4 of each of two groups of a value.
// Slots and heads are one range, so that few heads fill blocks too. (10.3 us for 4608 slots of 8 heads of 128 from L2 to
// bf16, with one, two, four or eight words of a thread on their way.)
template <bool F32, int NG>
__global__ void __launch_bounds__(kThreads) read_kernel(Cache cache, void* out_k, void* out_v, const int32_t* slots,
                                                        int64_t rows, FastDiv by_heads, int32_t* bad) {
  using E = Elem<F32>;
  constexpr int D = NG * kGroup, W = D / 8;
  const int w = threadIdx.x % W;
  const int64_t row = (int64_t)blockIdx.x * (kThreads / W) + threadIdx.x / W;
  if (row >= rows) return;
  const int at = (int)fdiv(by_heads, (uint32_t)row), head = (int)row - at * cache.heads, slot = slots[at];
  if (slot >= cache.pages * cache.page_size) atomicExch(bad, kBadSlot);
  if (slot < 0 || slot >= cache.pages * cache.page_size) return;
  const bool value = blockIdx.y;
  const int64_t from = row_of(cache, slot, head);
  const uint32_t code = __ldg((const uint32_t*)((value ? cache.v : cache.k) + from * (D / 2)) + w);
  const uint32_t* s = (value ? cache.v_scale : cache.k_scale) + from * NG;
  uint2 scale;
  if (value) scale = __ldg((const uint2*)s + w % (NG / 2));
  else scale.x = scale.y = __ldg(s + w % NG);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t q = e < 4 ? scale.x : scale.y;
    // 2^23 + code + 8, as the four bits with their highest turned over
    const float c = __uint_as_float((code >> (4 * e) & 15u) ^ 0x4b000008u) - (0x1p23f + 8.0f);
    y[e] = fmaf(c, __uint_as_float(q << 16), __uint_as_float(q & 0xffff0000u));
  }
  auto* to = (typename E::T*)(value ? out_v : out_k) + row * D;
  if (!value) {
    store_n<F32, 8>(to + (w % NG) * kGroup + (w / NG) * 8, y);
  } else {
    to += (w % (NG / 2)) * 2 * kGroup + (w / (NG / 2)) * 4;
    store_n<F32, 4>(to, y);
    store_n<F32, 4>(to + kGroup, y + 4);
  }
}

bool aligned16(const void* p, int64_t stride_elems, int elem_bytes) {
  return (uintptr_t)p % 16 == 0 && stride_elems * elem_bytes % 16 == 0;
}

template <bool F32>
void launch_append(fopt_ctx* ctx, AppendArgs a, const Rope& r, int dim) {
  // tokens enough to occupy a block's threads, but not so many that SMs go without
  const int rows = 2 * a.cache.heads * (dim / 16);
  a.each = std::max(1, std::min(kThreads / rows, a.tokens / sm_count(ctx)));
  a.by_heads = make_fastdiv((uint32_t)a.cache.heads);
  const int grid = (a.tokens + a.each - 1) / a.each;
  const size_t smem = (size_t)a.each * r.pairs * sizeof(float2);
  switch (dim) {
    case 64: append_kernel<F32, 2><<<grid, kThreads, smem, ctx->stream>>>(a, r); break;
    case 128: append_kernel<F32, 4><<<grid, kThreads, smem, ctx->stream>>>(a, r); break;
    default: append_kernel<F32, 8><<<grid, kThreads, smem, ctx->stream>>>(a, r); break;
  }
  launched(ctx, "cache append");
}

template <bool F32, bool VEC>
void launch_rotary(fopt_ctx* ctx, RotaryArgs a, const Rope& r) {
  constexpr int kAhead = 2;
  // tokens enough to occupy a block's threads kAhead times over (12 us for 14598 tokens of 3 heads of 128 in bf16 from L2,
  // against 19 with two tokens a block), but not so many that SMs go without
  const int64_t per_token = (int64_t)a.heads * a.units, sms = sm_count(ctx);
  const int64_t fill = VEC ? std::min<int64_t>(kThreads * kAhead / per_token, 2048 / r.pairs) : kOnes;
  a.each = (int)std::max<int64_t>(1, std::min(fill, a.tokens / (2 * sms)));
  rotary_kernel<F32, VEC, kAhead><<<(a.tokens + a.each - 1) / a.each, kThreads, a.each * r.pairs * sizeof(float2), ctx->stream>>>(a, r);
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
    kv::RotaryArgs a{out, x, positions, x_stride, out_stride, tokens, heads, head_dim, 1, units, make_fastdiv((uint32_t)units),
                     make_fastdiv((uint32_t)heads)};
    if (f32) vec ? kv::launch_rotary<true, true>(ctx, a, r) : kv::launch_rotary<true, false>(ctx, a, r);
    else vec ? kv::launch_rotary<false, true>(ctx, a, r) : kv::launch_rotary<false, false>(ctx, a, r);
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
    a.bad = ctx->bad_index();
    a.tokens = tokens;
    a.k_vec = kv::aligned16(k, k_stride, f32 ? 4 : 2);
    a.v_vec = kv::aligned16(v, v_stride, f32 ? 4 : 2);
    a.pair_vec = r.interleaved ? r.pairs % 4 == 0 : a.k_vec && r.pairs % 8 == 0;
    f32 ? kv::launch_append<true>(ctx, a, r, dim) : kv::launch_append<false>(ctx, a, r, dim);
  });
}

fopt_status fopt_cache_read(fopt_ctx* ctx, void* out_k, void* out_v, fopt_dtype dtype, const fopt_paged_cache* cache,
                            const int32_t* slots, int32_t n) {
  return kv::checked_call(ctx, [&] {
    const kv::Cache c = kv::checked(cache, "fopt_cache_read");
    require(dtype == FOPT_BF16 || dtype == FOPT_F32, "fopt_cache_read: bf16 or f32 values");
    require(n >= 0, "fopt_cache_read: a negative slot count");
    require((int64_t)n * c.heads <= INT32_MAX, "fopt_cache_read: slots times heads past 2^31");
    if (ctx && n == 0) return;
    require(out_k && out_v && slots, "fopt_cache_read: null argument");
    require(((uintptr_t)out_k | (uintptr_t)out_v) % 16 == 0, "fopt_cache_read: outputs must be 16-byte aligned");
    require(ctx != nullptr, "null context");
    DeviceGuard guard(ctx);
    const int dim = cache->head_dim;
    const int64_t rows = (int64_t)n * c.heads;
    auto go = [&](auto kernel) {
      const int64_t each = kv::kThreads / (dim / 8);
      kernel<<<dim3((unsigned)((rows + each - 1) / each), 2), kv::kThreads, 0, ctx->stream>>>(
          c, out_k, out_v, slots, rows, make_fastdiv((uint32_t)c.heads), ctx->bad_index());
      launched(ctx, "cache read");
    };
    if (dtype == FOPT_F32)
      dim == 64 ? go(kv::read_kernel<true, 2>) : dim == 128 ? go(kv::read_kernel<true, 4>) : go(kv::read_kernel<true, 8>);
    else
      dim == 64 ? go(kv::read_kernel<false, 2>) : dim == 128 ? go(kv::read_kernel<false, 4>) : go(kv::read_kernel<false, 8>);
  });
}

}  // extern "C"
