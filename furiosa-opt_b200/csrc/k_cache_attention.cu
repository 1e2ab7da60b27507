// Attention over the paged 4-bit cache: softmax(scale q K^T) V for sequences of any lengths.
//
// With a stored value = code * step + offset per group of 32 channels, a score is
//   q . k = sum_groups step (q_g . code_g) + offset (sum of q_g)
// and an output  o = sum_tokens (p step) code + p offset, so the products run on the codes themselves
// (small integers, exact in f16) with f32 sums, and the scales enter on [token x row] numbers, 32 times
// fewer than the channels. One pass over the keys with a running maximum and sum.
//
// tokens_kernel: the products are mma.sync m16n8k16 (f16 in, f32 sums) with the TOKENS as the 16 rows and 8
// query rows (the query heads of one key head, of one or more tokens) as the 8 columns. A single token's
// queries fill 4 to 8 of 128 rows of a tcgen05 tile and would need the codes expanded through shared memory;
// here a lane turns the words that it loaded into fragments in registers. What bounds it is the cache's
// bytes; the instructions of the expansion (about one per code) come next.
//   * K operand: lane (g, i) = (lane / 4, lane % 4) takes the 16-byte (D = 128) run of token g that the
//     layout [D % 32 / 8, D / 32, D % 8] puts at i: word j is 8 channels of group j, which make its operand
//     registers of two k16 steps; q's fragments are permuted to match. (x & 0x00f000f0) ^ 0x64806480 is
//     f16 1024 + 16 (code + 8): with q / 16 that is q (code + 72), and the sum starts from -72 sum(q).
//   * V operand (channels as rows, tokens as k): lane (g, i) takes the channels 4 g .. 4 g + 3 of every
//     group for four tokens; byte permutes pair two tokens' channels, and the codes become exact f16.
//   * probabilities go from the scores' fragment to the V product's by movmatrix.
//   * the maximum moves only when a score exceeds it by 2^8 (a warp vote), so the rescaling is rare. Steps of V
//     are scaled by a power of two that follows them the same way, which keeps p step within f16 at any
//     magnitude of V.
// Eight warps take 16 tokens each of a 128-token tile, with their own rings of cp.async stages (no block
// barrier while keys stream), and merge their (maximum, sum, output) at the end of a segment.
//
// Work: all (sequence, row block, key head) of the call, in 128-token tiles, form one line that is cut
// into equal shares, one per resident block, from the lengths on the device: no host knowledge of them, no idle
// blocks, any mixture of lengths. A segment cut between blocks leaves partial results in a workspace; the
// last of its blocks to arrive adds them up in order, so results do not depend on timing.
#include "kvcache.cuh"

namespace fopt {
namespace kv {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTileTokens = 16 * kWarps;
constexpr int kStages = 4;
constexpr float kLazy = 8.0f;  // log2 by which a score may exceed the running maximum before it moves

struct AttnArgs {
  uint16_t* o;
  const uint16_t* q;
  Cache cache;
  const int32_t* table;
  const int32_t* q_start;
  const int32_t* kv_len;
  int32_t* err;
  float* ws;          // partial results: two slots a block (see slot())
  uint32_t* counter;  // arrivals at the segment that begins in a block; zero between launches
  int batch, tokens, width, hq, group;
  float scale;
  int causal;
};

// ---- the division of work ----
struct Seq {
  int q0, rows;   // first query token; query rows per key head (tokens x group)
  int queries, keys;
  int tiles;      // 128-token tiles, one at least: a sequence without keys still writes its rows
};

// Sequence b's query range and key count, cut to what the arguments allow.
__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b) {
  const int s0 = a.q_start[b], s1 = a.q_start[b + 1], n = a.kv_len[b];
  Seq s;
  s.q0 = min(max(s0, 0), a.tokens);
  const int q1 = min(max(s1, s.q0), a.tokens);
  s.queries = q1 - s.q0;
  s.rows = s.queries * a.group;
  s.keys = (int)min((int64_t)max(n, 0), (int64_t)a.width * a.cache.page_size);
  s.tiles = max(1, (s.keys + kTileTokens - 1) / kTileTokens);
  if (s.q0 != s0 || q1 != s1) atomicExch(a.err, kBadStart);
  if (s.keys != n) atomicExch(a.err, kBadLength);
  return s;
}
template <int R>
__device__ __forceinline__ long long units(const AttnArgs& a, const Seq& s) {
  return (long long)((s.rows + R - 1) / R) * a.cache.heads * s.tiles;
}
// Of `total` units on `n` <= total blocks, block c has [first(c), first(c + 1)).
__device__ __forceinline__ long long first_unit(long long total, int n, int c) { return total * c / n; }
__device__ __forceinline__ int owner(long long total, int n, long long unit) {
  return (int)(((unit + 1) * n - 1) / total);
}

// ---- small pieces ----
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, uint32_t bytes) {  // bytes 0: zeros
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void mma(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float exp2_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float step_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float offset_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// Two codes (nibbles at bits 4-7 and 20-23) as f16 pairs 1024 + 16 (code + 8).
__device__ __forceinline__ uint32_t codes_high(uint32_t x) { return (x & 0x00f000f0u) ^ 0x64806480u; }
// ... as exact f16 codes, from bits 4-7 / 20-23 and from bits 0-3 / 16-19.
__device__ __forceinline__ uint32_t exact_high(uint32_t x) {
  uint32_t r;
  asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(codes_high(x)), "r"(0x2c002c00u), "r"(0xd480d480u));  // / 16 - 72
  return r;
}
__device__ __forceinline__ uint32_t exact_low(uint32_t x) {
  uint32_t r;
  asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"((x & 0x000f000fu) ^ 0x64086408u), "r"(0xe408e408u));  // - 1032
  return r;
}
template <int N>
__device__ __forceinline__ void load_words(uint32_t* w, const uint8_t* p) {
  if constexpr (N == 1) w[0] = *(const uint32_t*)p;
  if constexpr (N == 2) *(uint2*)w = *(const uint2*)p;
  if constexpr (N >= 4) {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) *(uint4*)(w + 4 * i) = ((const uint4*)p)[i];
  }
}
// max over the eight g of a warp's lanes (same i)
__device__ __forceinline__ float max_over_g(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float sum_over_g(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// Shared memory of a block: the warps' rings, then (the rings drained) their partial outputs.
template <int NG, int NB>
struct Shared {
  static constexpr int D = NG * kGroup, R = 8 * NB;
  static constexpr int kCodes = 16 * D / 2, kScales = 16 * NG * 4;      // one tile's K or V
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kRing = kStages * kStage;
  static constexpr int kRow = D + 4;                                    // floats; the pad spreads rows over banks
  static constexpr int kBytes = kWarps * (kRing > R * kRow * 4 ? kRing : R * kRow * 4);
};

// Where a 16-byte chunk of a token's V codes sits in its row: rows two apart, which one load reads
// together, start at the same bank.
template <int NG>
__device__ __forceinline__ int v_chunk(int token, int chunk) {
  if constexpr (NG == 4) return chunk ^ ((token >> 1) & 3);
  if constexpr (NG == 8) return chunk ^ (((token >> 1) & 3) << 1);
  return chunk;
}

// A warp's state over a segment's keys.
template <int NG, int NB>
struct State {
  float o[NB][NG][2][4];   // [channel 32 j + 4 g + 2 mm (+ 1 for c2, c3)] x [row 2 i, 2 i + 1], in 2^ev
  float e[NB][NG][2];      // sum of p offset, this lane's tokens
  float m[NB][2], l[NB][2];
  float vscale;            // 2^-ev
  uint32_t vlimit;         // bf16 bits of the largest step that p step 2^-ev still holds
};

template <int NG, int NB>
struct Query {
  uint32_t f[NB][2 * NG][2];  // fragments of q 2^(8 - e) / 16
  float sum[NB][NG][2];       // sums of q 2^(8 - e) over a group, of the lane's rows 2 i and 2 i + 1
  float scale[NB][2];         // 2^(e - 8) scale log2(e)
  int limit[NB][2];           // keys that the row sees
};

template <int NG, int NB>
__device__ __forceinline__ void load_query(const AttnArgs& a, const Seq& s, int head, int row0, Query<NG, NB>& q) {
  const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
  constexpr int D = NG * kGroup;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const int r = row0 + nb * 8 + g;
    const bool live = r < s.rows;
    const int token = live ? r / a.group : 0;
    const uint16_t* p = a.q + ((int64_t)(s.q0 + token) * a.hq + head * a.group + (live ? r - token * a.group : 0)) * D;
    uint4 w[NG];
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      w[j] = live ? *(const uint4*)(p + j * kGroup + i * 8) : make_uint4(0, 0, 0, 0);
      const uint32_t* x = (const uint32_t*)&w[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, fmaxf(fabsf(step_of(x[e])), fabsf(offset_of(x[e]))));
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    int ex = top > 0.0f ? min(ilogbf(top), 127) : 0;
    // 2^(8 - ex) may pass the f32 range: two factors
    const float up0 = scalbnf(1.0f, (8 - ex) / 2), up1 = scalbnf(1.0f, 8 - ex - (8 - ex) / 2);
    const float down = scalbnf(a.scale * 1.44269504088896340736f, ex - 8);
    float sum[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const uint32_t* x = (const uint32_t*)&w[j];
      float v[8];
      sum[j] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = (e & 1 ? offset_of(x[e >> 1]) : step_of(x[e >> 1])) * up0 * up1 * 0.0625f;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t h = f16x2(v[e], v[e + 4]);  // the pairs that codes_high() makes of a word
        q.f[nb][2 * j + (e >> 1)][e & 1] = h;
        // the sum of what the products take
        float lo, hi;
        asm("{.reg .f16 a, b; mov.b32 {a, b}, %2; cvt.f32.f16 %0, a; cvt.f32.f16 %1, b;}" : "=f"(lo), "=f"(hi) : "r"(h));
        sum[j] += lo + hi;
      }
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
    }
    // the lane's rows as columns of the scores: 2 i and 2 i + 1, held by the lanes of g = 2 i, 2 i + 1
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int from = 4 * (2 * i + c);
#pragma unroll
      for (int j = 0; j < NG; ++j) q.sum[nb][j][c] = 16.0f * __shfl_sync(0xffffffffu, sum[j], from);
      q.scale[nb][c] = __shfl_sync(0xffffffffu, down, from);
      const int rc = row0 + nb * 8 + 2 * i + c;
      // columns past the rows hold q = 0 and no one reads them: they need no mask of their own
      q.limit[nb][c] = rc >= s.rows ? s.keys : a.causal ? min(s.keys, s.keys - s.queries + rc / a.group + 1) : s.keys;
    }
  }
}

// One tile of 16 tokens, from its stage; token0 is its first.
template <int NG, int NB>
__device__ __forceinline__ void tile(const uint8_t* stage, int token0, int keys, int sure, const Query<NG, NB>& q,
                                     State<NG, NB>& s) {
  using S = Shared<NG, NB>;
  const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
  uint32_t kw[2][NG], km[2][NG];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    load_words<NG>(kw[h], stage + (g + 8 * h) * (S::D / 2) + i * NG * 4);
    load_words<NG>(km[h], stage + 2 * S::kCodes + (g + 8 * h) * NG * 4);
  }
  float x[NB][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) x[nb][0] = x[nb][1] = x[nb][2] = x[nb][3] = 0.0f;
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    uint32_t h0[4], h1[4];
    h0[0] = codes_high(kw[0][j] << 4), h0[1] = codes_high(kw[0][j]), h0[2] = codes_high(kw[0][j] >> 4), h0[3] = codes_high(kw[0][j] >> 8);
    h1[0] = codes_high(kw[1][j] << 4), h1[1] = codes_high(kw[1][j]), h1[2] = codes_high(kw[1][j] >> 4), h1[3] = codes_high(kw[1][j] >> 8);
    const float s0 = step_of(km[0][j]), s1 = step_of(km[1][j]), z0 = offset_of(km[0][j]), z1 = offset_of(km[1][j]);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const float a0 = -72.0f * q.sum[nb][j][0], a1 = -72.0f * q.sum[nb][j][1];
      float acc[4] = {a0, a1, a0, a1};
      mma(acc, h0[0], h1[0], h0[1], h1[1], q.f[nb][2 * j][0], q.f[nb][2 * j][1]);
      mma(acc, h0[2], h1[2], h0[3], h1[3], q.f[nb][2 * j + 1][0], q.f[nb][2 * j + 1][1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        x[nb][c] = fmaf(s0, acc[c], fmaf(z0, q.sum[nb][j][c], x[nb][c]));
        x[nb][c + 2] = fmaf(s1, acc[c + 2], fmaf(z1, q.sum[nb][j][c], x[nb][c + 2]));
      }
    }
  }
  uint32_t vm[2][NG];
#pragma unroll
  for (int h = 0; h < 2; ++h) load_words<NG>(vm[h], stage + 2 * S::kCodes + S::kScales + (g + 8 * h) * NG * 4);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 4; ++c) x[nb][c] *= q.scale[nb][c & 1];
  if (token0 + 16 > sure) {  // some row does not see all of it
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = token0 + g + 8 * h;
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (t >= q.limit[nb][c]) x[nb][2 * h + c] = -INFINITY;
      if (t >= keys) {  // slots past the end hold anything: their scales must not meet a zero probability
#pragma unroll
        for (int j = 0; j < NG; ++j) vm[h][j] = 0;
      }
    }
  }
  // does the maximum, or the power of two of the steps, have to move?
  uint32_t steps = 0;
#pragma unroll
  for (int j = 0; j < NG; ++j) steps = __vmaxu2(steps, __vmaxu2(vm[0][j], vm[1][j]));
  bool move = (steps & 0xffffu) > s.vlimit;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 4; ++c) move |= x[nb][c] > s.m[nb][c & 1] + kLazy;
  if (__any_sync(0xffffffffu, move)) {
    uint32_t top = steps & 0x7fffu;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    float by = 1.0f;
    if (top > s.vlimit) {  // the largest step to [2^4, 2^5), and room up to 2^7: p <= 2^8 keeps 2^15
      const int ev = (int)(top >> 7) - 127 - 4;
      const float vscale = scalbnf(1.0f, min(-ev, 126));
      by = s.vscale > 0.0f ? vscale / s.vscale : 0.0f;
      s.vscale = vscale;
      s.vlimit = min(top + (2u << 7), 0x7f7fu);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float was = s.m[nb][c], now = fmaxf(was, max_over_g(fmaxf(x[nb][c], x[nb][c + 2])));
        const float f = now == -INFINITY ? 1.0f : exp2_(was - now);
        s.m[nb][c] = now;
        s.l[nb][c] *= f;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          s.e[nb][j][c] *= f;
#pragma unroll
          for (int mm = 0; mm < 2; ++mm) {
            s.o[nb][j][mm][c] *= f * by;
            s.o[nb][j][mm][c + 2] *= f * by;
          }
        }
      }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const float m = s.m[nb][c & 1];
      x[nb][c] = exp2_(x[nb][c] - (m == -INFINITY ? 0.0f : m));
      s.l[nb][c & 1] += x[nb][c];
    }
  // V: words of tokens 2 i, 2 i + 1, 2 i + 8, 2 i + 9
  uint32_t vw[4][NG / 2];
#pragma unroll
  for (int t = 0; t < 4; ++t) {
    const int token = 2 * i + (t & 1) + 8 * (t >> 1), at = g * NG * 2;  // byte of the row
    load_words<NG / 2>(vw[t], stage + S::kCodes + token * (S::D / 2) + v_chunk<NG>(token, at >> 4) * 16 + (at & 15));
  }
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
    const uint32_t x01 = __byte_perm(vw[0][j >> 1], vw[1][j >> 1], sel), x23 = __byte_perm(vw[2][j >> 1], vw[3][j >> 1], sel);
    const uint32_t y01 = x01 >> 8, y23 = x23 >> 8;
    const uint32_t c0 = exact_low(x01), c1 = exact_high(x01), c2 = exact_low(x23), c3 = exact_high(x23);
    const uint32_t d0 = exact_low(y01), d1 = exact_high(y01), d2 = exact_low(y23), d3 = exact_high(y23);
    const float s0 = step_of(vm[0][j]) * s.vscale, s1 = step_of(vm[1][j]) * s.vscale;
    const float z0 = offset_of(vm[0][j]), z1 = offset_of(vm[1][j]);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const uint32_t b0 = transposed(f16x2(x[nb][0] * s0, x[nb][1] * s0));
      const uint32_t b1 = transposed(f16x2(x[nb][2] * s1, x[nb][3] * s1));
      mma(s.o[nb][j][0], c0, c1, c2, c3, b0, b1);
      mma(s.o[nb][j][1], d0, d1, d2, d3, b0, b1);
#pragma unroll
      for (int c = 0; c < 2; ++c) s.e[nb][j][c] = fmaf(x[nb][c], z0, fmaf(x[nb][c + 2], z1, s.e[nb][j][c]));
    }
  }
}

// A block's partial results of the segment that it shares: [slot][row][D] outputs, then maxima and sums.
// Slot 0 is for a segment that another block began, slot 1 for one that this block begins.
template <int NG, int NB>
struct Partial {
  static constexpr int D = NG * kGroup, R = 8 * NB;
  static constexpr int kFloats = R * (D + 2);
  static __device__ __forceinline__ float* slot(float* ws, int block, bool begins) {
    return ws + ((int64_t)block * 2 + begins) * kFloats;
  }
};

template <int NG, int NB>
__global__ void __launch_bounds__(kThreads, NG <= 4 && NB == 1 ? 2 : 1) tokens_kernel(AttnArgs a) {
  using S = Shared<NG, NB>;
  using P = Partial<NG, NB>;
  constexpr int D = S::D, R = S::R;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ long long sums[kWarps];
  __shared__ long long found_at;
  __shared__ int found;
  __shared__ float ml[2][kWarps][R];
  __shared__ int last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, i = lane & 3;

  // this block's share of the line: the total, then the sequence in which the share begins
  long long mine = 0;
  for (int b = tid; b < a.batch; b += kThreads) mine += units<R>(a, sequence(a, b));
  long long total = mine;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) sums[warp] = total;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += sums[w];
  if (total == 0) return;
  const int blocks = (int)min((long long)gridDim.x, total);
  if (blockIdx.x >= blocks) return;
  long long unit = first_unit(total, blocks, blockIdx.x);
  const long long end = first_unit(total, blocks, blockIdx.x + 1);
  long long before = 0;  // units of the sequences before the chunk
  for (int b0 = 0;; b0 += kThreads) {
    const int b = b0 + tid;
    const long long u = b < a.batch ? units<R>(a, sequence(a, b)) : 0;
    long long upto = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    __syncthreads();
    if (lane == 31) sums[warp] = upto;
    if (tid == 0) found = -1;
    __syncthreads();
    long long here = before;
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) here += sums[w];
      before += sums[w];
    }
    if (unit >= here + upto - u && unit < here + upto) {
      found = b;
      found_at = here + upto - u;
    }
    __syncthreads();
    if (found >= 0) break;
  }
  int b = found;
  long long seq_at = found_at;
  Seq s = sequence(a, b);

  uint8_t* ring = smem + warp * S::kRing;
  const uint32_t ring_u32 = smem_u32(ring);
  while (unit < end) {
    while (unit >= seq_at + units<R>(a, s)) {
      seq_at += units<R>(a, s);
      s = sequence(a, ++b);
    }
    const int seg = (int)((unit - seq_at) / s.tiles);
    const int t0 = (int)(unit - seq_at - (long long)seg * s.tiles);
    const int t1 = (int)min((long long)s.tiles, t0 + (end - unit));
    const int head = seg % a.cache.heads, row0 = seg / a.cache.heads * R;
    const long long seg_at = unit - t0;
    unit += t1 - t0;

    Query<NG, NB> q;
    load_query<NG, NB>(a, s, head, row0, q);
    // keys that any row of the block sees, and that every row sees
    const int rows = min(R, s.rows - row0);
    const int most = a.causal ? min(s.keys, s.keys - s.queries + (row0 + rows - 1) / a.group + 1) : s.keys;
    const int sure = a.causal ? min(s.keys, s.keys - s.queries + row0 / a.group + 1) : s.keys;
    State<NG, NB> st;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      st.m[nb][0] = st.m[nb][1] = -INFINITY;
      st.l[nb][0] = st.l[nb][1] = 0.0f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        st.e[nb][j][0] = st.e[nb][j][1] = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) st.o[nb][j][0][c] = st.o[nb][j][1][c] = 0.0f;
      }
    }
    st.vscale = 0.0f;
    st.vlimit = 0;

    const int32_t* table = a.table + (int64_t)b * a.width;
    auto page_of = [&](int t) -> int {
      const int token = t * kTileTokens + warp * 16;
      return t < t1 && token < most ? table[fdiv(a.cache.by_page, (uint32_t)token)] : 0;
    };
    auto fetch = [&](int t, int page, int stage) {
      const int token = t * kTileTokens + warp * 16;
      if (t < t1 && token < most) {
        const bool there = page >= 0 && page < a.cache.pages;
        if (!there && lane == 0) atomicExch(a.err, kBadPage);
        const uint32_t bytes = there ? 16 : 0;
        const int in_page = token - (int)fdiv(a.cache.by_page, (uint32_t)token) * a.cache.page_size;
        const int64_t row = there ? ((int64_t)page * a.cache.heads + head) * a.cache.page_size + in_page : 0;
        const uint8_t* k = a.cache.k + row * (D / 2);
        const uint8_t* v = a.cache.v + row * (D / 2);
        const uint32_t to = ring_u32 + stage * S::kStage;
#pragma unroll
        for (int c = lane; c < S::kCodes / 16; c += 32) {
          copy16(to + c * 16, k + c * 16, bytes);
          const int tok = c / NG, chunk = c % NG;
          copy16(to + S::kCodes + (tok * NG + v_chunk<NG>(tok, chunk)) * 16, v + c * 16, bytes);
        }
        const uint8_t* ks = (const uint8_t*)(a.cache.k_scale + row * NG);
        const uint8_t* vs = (const uint8_t*)(a.cache.v_scale + row * NG);
#pragma unroll
        for (int c = lane; c < 2 * (S::kScales / 16); c += 32)
          copy16(to + 2 * S::kCodes + c * 16, c < S::kScales / 16 ? ks + c * 16 : vs + (c - S::kScales / 16) * 16, bytes);
      }
      copies_commit();
    };
    int page = page_of(t0);
#pragma unroll
    for (int n = 0; n < kStages - 1; ++n) {
      const int next = page_of(t0 + n + 1);
      fetch(t0 + n, page, n);
      page = next;
    }
    int stage = 0;
    for (int t = t0; t < t1; ++t) {
      const int next = page_of(t + kStages);
      fetch(t + kStages - 1, page, stage ? stage - 1 : kStages - 1);
      page = next;
      copies_wait<kStages - 1>();
      __syncwarp();
      const int token = t * kTileTokens + warp * 16;
      if (token < most) tile<NG, NB>(ring + stage * S::kStage, token, s.keys, sure, q, st);
      __syncwarp();  // all lanes have read the stage before the next copies into it
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
    copies_wait<0>();
    __syncthreads();  // every warp's ring is drained: the outputs go over them

    float* out = (float*)smem + warp * R * S::kRow;
    const float back = st.vscale > 0.0f ? 1.0f / st.vscale : 0.0f;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int r = nb * 8 + 2 * i + c;
        const float l = sum_over_g(st.l[nb][c]);
        if (g == 0) {
          ml[0][warp][r] = st.m[nb][c];
          ml[1][warp][r] = l;
        }
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          const float e = sum_over_g(st.e[nb][j][c]);
          *(float4*)(out + r * S::kRow + j * kGroup + 4 * g) =
              make_float4(fmaf(st.o[nb][j][0][c], back, e), fmaf(st.o[nb][j][0][c + 2], back, e),
                          fmaf(st.o[nb][j][1][c], back, e), fmaf(st.o[nb][j][1][c + 2], back, e));
        }
      }
    __syncthreads();

    auto write_row = [&](int r, int d, float4 v, float l) {  // channels d .. d + 3 of row r
      const int row = row0 + r;
      const float n = l != 0.0f ? 1.0f / l : 0.0f;  // a row that sees no key is 0
      const int token = row / a.group;
      *(uint2*)(a.o + ((int64_t)(s.q0 + token) * a.hq + head * a.group + row - token * a.group) * D + d) =
          make_uint2(bf16x2_rule(v.x * n, v.y * n), bf16x2_rule(v.z * n, v.w * n));
    };
    const bool whole = t0 == 0 && t1 == s.tiles;
    float* part = P::slot(a.ws, blockIdx.x, t0 == 0);
    for (int k = tid; k < rows * (D / 4); k += kThreads) {
      const int r = k / (D / 4), d = k % (D / 4) * 4;
      float m = -INFINITY, l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[0][w][r]);
      float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_(ml[0][w][r] - (m == -INFINITY ? 0.0f : m));
        const float4 v = *(const float4*)((const float*)smem + (w * R + r) * S::kRow + d);
        l = fmaf(f, ml[1][w][r], l);
        sum.x = fmaf(f, v.x, sum.x), sum.y = fmaf(f, v.y, sum.y), sum.z = fmaf(f, v.z, sum.z), sum.w = fmaf(f, v.w, sum.w);
      }
      if (whole) {
        write_row(r, d, sum, l);
      } else {
        *(float4*)(part + r * D + d) = sum;
        if (d == 0) {
          part[R * D + r] = m;
          part[R * D + R + r] = l;
        }
      }
    }
    if (!whole) {
      const int c0 = owner(total, blocks, seg_at), c1 = owner(total, blocks, seg_at + s.tiles - 1);
      __threadfence();
      __syncthreads();
      if (tid == 0) {
        last = atomicAdd(a.counter + c0, 1u) == (uint32_t)(c1 - c0);
        if (last) a.counter[c0] = 0;
        __threadfence();
      }
      __syncthreads();
      if (last) {
        for (int k = tid; k < rows * (D / 4); k += kThreads) {
          const int r = k / (D / 4), d = k % (D / 4) * 4;
          float m = -INFINITY, l = 0.0f;
          for (int c = c0; c <= c1; ++c) m = fmaxf(m, __ldcg(P::slot(a.ws, c, c == c0) + R * D + r));
          float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 4
          for (int c = c0; c <= c1; ++c) {
            const float* p = P::slot(a.ws, c, c == c0);
            const float f = exp2_(__ldcg(p + R * D + r) - (m == -INFINITY ? 0.0f : m));
            const float4 v = __ldcg((const float4*)(p + r * D + d));
            l = fmaf(f, __ldcg(p + R * D + R + r), l);
            sum.x = fmaf(f, v.x, sum.x), sum.y = fmaf(f, v.y, sum.y), sum.z = fmaf(f, v.z, sum.z), sum.w = fmaf(f, v.w, sum.w);
          }
          write_row(r, d, sum, l);
        }
      }
    }
    __syncthreads();  // the outputs are read before the next segment's copies
  }
}

template <int NG, int NB>
void launch_tokens(fopt_ctx* ctx, AttnArgs a, int sms) {
  using S = Shared<NG, NB>;
  const int grid = sms * (NG <= 4 && NB == 1 ? 2 : 1);
  cuda_check(cudaFuncSetAttribute(tokens_kernel<NG, NB>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes),
             "cache attention shared memory");
  const size_t partials = (size_t)grid * 2 * Partial<NG, NB>::kFloats * sizeof(float);
  // the counters first: other variants' partial results must not reach them
  uint8_t* ws = (uint8_t*)cache_workspace(ctx, 4096 + partials);
  a.counter = (uint32_t*)ws;
  a.ws = (float*)(ws + 4096);
  require(grid <= 1024, "fopt_cache_attention: more resident blocks than counters");
  tokens_kernel<NG, NB><<<grid, kThreads, S::kBytes, ctx->stream>>>(a);
  launched(ctx, "cache attention");
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
    int sms = 0;
    cuda_check(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, ctx->device), "SM count");
    // 16 rows a block where a sequence has that many on average: the codes are expanded once for both halves
    const bool two = (int64_t)tokens * a.group > 8 * (int64_t)batch;
    switch (cache->head_dim) {
      case 64: two ? kv::launch_tokens<2, 2>(ctx, a, sms) : kv::launch_tokens<2, 1>(ctx, a, sms); break;
      case 128: two ? kv::launch_tokens<4, 2>(ctx, a, sms) : kv::launch_tokens<4, 1>(ctx, a, sms); break;
      default: kv::launch_tokens<8, 1>(ctx, a, sms); break;
    }
  });
}
