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
// here a lane turns the words that it loaded into fragments in registers. What bounds it are chains of dependent
// instructions at 12 warps an SM (168 registers a thread): 57 % of the issue slots and 0.53 of a copy's rate are used,
// and the first stall is an instruction's own latency. 90 us for one token of each of 64 sequences of 64 to 8192 keys, 8 key
// heads of 128 and 4 query heads to each (3.5 TB/s of codes and scales); 77 us for two tokens at 131072 and 100003
// keys. 16 warps at 128 registers spill (95 us for the first, where 12 took 86).
//   * K operand: lane (g, i) = (lane / 4, lane % 4) takes the 16-byte (D = 128) run of token g that the
//     layout [D % 32 / 8, D / 32, D % 8] puts at i: word j is 8 channels of group j, which make its operand
//     registers of two k16 steps; q's fragments are permuted to match. (x & 0x000f000f) ^ 0x00080008 is a
//     pair of f16 subnormals (code + 8) 2^-24, and (x & 0x00f000f0) ^ 0x00800080 of (code + 8) 2^-20: one
//     instruction a pair and nothing to subtract, with the powers of two in q's fragments and the 8 in the
//     group's offset (offset - 8 step).
//   * V operand (channels as rows, tokens as k): lane (g, i) takes the channels 4 g .. 4 g + 3 of every
//     group for four tokens; byte permutes pair two tokens' channels.
//   * probabilities go from the scores' fragment to the V product's by movmatrix, as p step in f16: half a
//     step of it is 2^-11, an eighth of the output's own rounding. p offset is summed in f32.
//   * the maximum moves only when a score exceeds it by 2^6 (a warp vote), so the rescaling is rare. Steps of V
//     are scaled by a power of two that follows the largest the same way, which keeps p step within f16's upper end.
//     Its lower end is looked at behind the last key: a product p step is off by 2^-11 of itself or by 2^-25 at most,
//     so a run of n keys is right to 2^-10 of the sum of its products if that sum is 2^-14 n at least. Where one is
//     not (a group whose steps are far below another's, or whose tokens of weight have steps far below those of
//     tokens without), the warp takes its run once more, with products in f32 (a call takes five times as long where every
//     run is).
// Four warps take a run of 16-token tiles each, with their own rings of cp.async stages (no block barrier
// while keys stream), and merge their (maximum, sum, output) at the end of a segment.
//
// Segments, of 8 or 16 query rows, are divided between blocks as cache_attention.cuh says.
#include "cache_attention.cuh"

namespace fopt {
namespace kv {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTileTokens = 16 * kWarps;
constexpr int kBlocks = 3;       // resident blocks an SM, where the registers allow (168 a thread)
template <int NG, int NB>
constexpr int tokens_blocks() { return NG <= 4 && NB == 1 ? kBlocks : 2; }
constexpr int kSegmentCost = 4;  // beginning and ending a segment takes about as long as this many tiles
constexpr int kLeast = 2;        // tiles of a share
// A part more to add up takes about a sixth of a tile. Shares of 2 tiles were best at 777 tokens of 8 heads
// (12.4 us; 14.0 with 4), of 8 at 15179 of two heads (20.6; 29.3 with 2), of 8 to 16 at 131072 of one (2 us less than with 5).
constexpr float kByRoot = 0.4f;
constexpr int kStages = 4;
constexpr float kLazy = 6.0f;    // log2 by which a score may exceed the running maximum before it moves
constexpr int kStepTop = 6;      // the largest step is brought to [2^6, 2^7) ...
constexpr float kStepRoom = 512.0f;  // ... and may grow to 2^9: p step <= 2^15
constexpr int kFewRows = 32;     // query rows per key head up to which a sequence is tokens_kernel's
// The sequence's tiles (one at least: a sequence without keys still writes its rows), and how long its segments
// and all of them together are in the division of work.
__device__ __forceinline__ int tiles_of(const Seq& s) { return max(1, (s.keys + kTileTokens - 1) / kTileTokens); }
template <int R>
__device__ __forceinline__ long long units(const AttnArgs& a, const Seq& s) {
  return s.rows >= a.long_rows ? 0 : (long long)((s.rows + R - 1) / R) * a.cache.heads * (tiles_of(s) + kSegmentCost);
}

// ---- small pieces ----
// Counts an arrival: what came before it is seen by whom counts a later one.
__device__ __forceinline__ uint32_t arrive(uint32_t* counter) {
  uint32_t before;
  asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(before) : "l"(counter) : "memory");
  return before;
}
__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
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
// The same from zero sums (no registers to clear).
__device__ __forceinline__ void mma0(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
template <bool FROM_ZERO>
__device__ __forceinline__ void mma_bf16(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (FROM_ZERO)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// Two codes as f16 subnormals: (code + 8) 2^-24 from bits 0-3 and 16-19, (code + 8) 2^-20 from bits 4-7 and 20-23.
__device__ __forceinline__ uint32_t codes_low(const Masks& m, uint32_t x) { return masked(x, m.low, 0x00080008u); }
__device__ __forceinline__ uint32_t codes_high(const Masks& m, uint32_t x) { return masked(x, m.high, 0x00800080u); }
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

// Shared memory of a block: the warps' rings, each then (drained) its warp's partial output.
template <int NG, int NB>
struct Shared {
  static constexpr int D = NG * kGroup, R = 8 * NB;
  static constexpr int kCodes = 16 * D / 2, kScales = 16 * NG * 4;      // one tile's K or V
  static constexpr int kScaleLanes = 2 * kScales / 16;                 // lanes that copy both's scales, 16 bytes each
  static constexpr int kStage = 2 * (kCodes + kScales);
  static constexpr int kRing = kStages * kStage;
  static constexpr int kRow = D + 4;                                    // floats; the pad spreads rows over banks
  static_assert(R * kRow * 4 <= kRing);
  static constexpr int kBytes = kWarps * kRing;
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
  // [channel 32 j + 4 g + 2 mm (+ 1 for c2, c3)] x [row 2 i, 2 i + 1]: sum of p step (code + 8). From the MMAs, in
  // 2^ev and 2^24 for the even channels (c0, c1), 2^20 for the odd ones
  float o[NB][NG][2][4];
  float e[NB][NG][2];      // sum of p (offset - 8 step), this lane's tokens
  float m[NB][2], l[NB][2];  // p = 2^(score - m), m the score's maximum (lagging by up to kLazy); sum of p
  int ev;                  // p step goes into the MMAs as 2^-ev of it, to fit f16's upper end at any magnitude of V
  float vlimit;            // the largest step that p step still holds; infinite: products in f32
  uint32_t stepped;        // groups of which a token of the lane's had a step, a bit each
  __device__ __forceinline__ void clear(bool wide) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      m[nb][0] = m[nb][1] = 0.0f;
      l[nb][0] = l[nb][1] = 0.0f;
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        e[nb][j][0] = e[nb][j][1] = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nb][j][0][c] = o[nb][j][1][c] = 0.0f;
      }
    }
    stepped = 0;
    ev = 0;
    vlimit = wide ? INFINITY : 0.0f;
  }
};

template <int NG, int NB>
struct Query {
  uint32_t f[NB][2 * NG][2];  // fragments of q 2^(8 - e), times 16 where codes_low() meets them
  // Fragments that turn a token's scale words, as they are, into sum_groups (offset - 8 step) (sum of q): k runs
  // over (group, step / offset) of groups 0 .. 3, then (NG = 8) of groups 4 .. 7. The sums are 2^(8 - e - 20) that
  // of the q in f, split into three bf16 parts, 24 bits together.
  static constexpr int kLimbs = NG == 8 ? 6 : 3;
  uint32_t z[NB][kLimbs];
  float scale[NB][2];         // 2^(e + 12) scale log2(e)
  int limit[NB][2];           // keys that the row sees
};

// The lane's part of the rows as it is in memory: 8 channels of each group of row g (of each eight rows).
template <int NG, int NB>
struct RawQuery {
  uint4 w[NB][NG];
  __device__ __forceinline__ void load(const AttnArgs& a, const Seq& s, int head, int row0) {
    const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      const int r = row0 + nb * 8 + g;
      const bool live = r < s.rows;
      const int token = live ? token_of(a, r) : 0;
      const uint16_t* p =
          a.q + ((int64_t)(s.q0 + token) * a.hq + head * a.group + (live ? r - token * a.group : 0)) * (NG * kGroup);
#pragma unroll
      for (int j = 0; j < NG; ++j) w[nb][j] = live ? *(const uint4*)(p + j * kGroup + i * 8) : make_uint4(0, 0, 0, 0);
    }
  }
};

template <int NG, int NB>
__device__ __forceinline__ void load_query(const AttnArgs& a, const Seq& s, int row0, const RawQuery<NG, NB>& raw,
                                           Query<NG, NB>& q) {
  const int lane = threadIdx.x & 31, i = lane & 3;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) {
    const uint4* w = raw.w[nb];
    uint32_t top = 0;  // of the magnitudes, as bf16 bits
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const uint32_t* x = (const uint32_t*)&w[j];
#pragma unroll
      for (int e = 0; e < 4; ++e) top = __vmaxu2(top, x[e] & 0x7fff7fffu);
    }
    top = max(top & 0xffffu, top >> 16);
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int ex = row_exponent(top);
    const float up = power(8 - ex);
    const float down = scalbnf(a.scale * 1.44269504088896340736f, ex + 12);
    float sum[NG];
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const uint32_t* x = (const uint32_t*)&w[j];
      float v[8];
      sum[j] = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = (e & 1 ? offset_of(x[e >> 1]) : step_of(x[e >> 1])) * up;
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        // the pairs that codes_low() and codes_high() make of a word
        const float by = e & 1 ? 1.0f : 16.0f;
        const uint32_t h = f16x2(v[e] * by, v[e + 4] * by);
        q.f[nb][2 * j + (e >> 1)][e & 1] = h;
        // the sum of what the products take
        sum[j] += sum_of(h) / by;
      }
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 1);
      sum[j] += __shfl_xor_sync(0xffffffffu, sum[j], 2);
    }
#pragma unroll
    for (int h = 0; h < (NG == 8 ? 2 : 1); ++h) {
      float rest = 0.0f;  // the sum of group 4 h + i
#pragma unroll
      for (int j = 0; j < NG; ++j)
        if (j == 4 * h + i) rest = sum[j] * 0x1p-20f;
#pragma unroll
      for (int n = 0; n < 3; ++n) {
        const float part = __uint_as_float(f32_to_bf16w(__float_as_uint(rest)));
        rest -= part;
        q.z[nb][h * 3 + n] = __float_as_uint(-8.0f * part) >> 16 | __float_as_uint(part);
      }
    }
    // the lane's rows as columns of the scores: 2 i and 2 i + 1, held by the lanes of g = 2 i, 2 i + 1
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int from = 4 * (2 * i + c);
      q.scale[nb][c] = __shfl_sync(0xffffffffu, down, from);
      const int rc = row0 + nb * 8 + 2 * i + c;
      // columns past the rows hold q = 0 and no one reads them: they need no mask of their own
      q.limit[nb][c] = rc >= s.rows ? s.keys : seen(a, s, rc);
    }
  }
}

// Where in a stage a lane reads: bytes from the start of its K codes, scales (either's) and V codes.
struct Places {
  int k, k_word, scale, v;
  Masks masks;
};
template <int NG>
__device__ __forceinline__ Places places() {
  constexpr int D = NG * kGroup;
  const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3, at = g * NG * 2;
  return {kept(g * (D / 2) + i * NG * 4), kept(g * NG * 4 + i * 4), kept(g * NG * 4),
          kept(2 * i * (D / 2) + v_chunk<NG>(2 * i, at >> 4) * 16 + (at & 15)),
          masks()};
}

// The raw scores q . k of one tile of 16 tokens, from its stage.
template <int NG, int NB>
__device__ __forceinline__ void scores(const uint8_t* stage, const Places& at, const Query<NG, NB>& q, float (*x)[4]) {
  using S = Shared<NG, NB>;
  const int i = threadIdx.x & 3;
  uint32_t kw[2][NG], km[2][NG];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    load_words<NG>(kw[h], stage + at.k + 8 * h * (S::D / 2));
    load_words<NG>(km[h], stage + 2 * S::kCodes + at.scale + 8 * h * NG * 4);
  }
  {
    uint32_t w[2][2] = {};  // scale words of tokens g and g + 8, groups i and i + 4
    const uint8_t* sc = stage + 2 * S::kCodes + at.k_word;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < (NG == 8 ? 2 : 1); ++n)
        if (NG >= 4 || i < NG) w[h][n] = *(const uint32_t*)(sc + 8 * h * NG * 4 + n * 16);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      if constexpr (NG == 8) {
        mma_bf16<true>(x[nb], w[0][0], w[1][0], w[0][1], w[1][1], q.z[nb][0], q.z[nb][3]);
        mma_bf16<false>(x[nb], w[0][0], w[1][0], w[0][1], w[1][1], q.z[nb][1], q.z[nb][4]);
        mma_bf16<false>(x[nb], w[0][0], w[1][0], w[0][1], w[1][1], q.z[nb][2], q.z[nb][5]);
      } else {
        mma_bf16<true>(x[nb], w[0][0], w[1][0], w[0][0], w[1][0], q.z[nb][0], q.z[nb][1]);
        mma_bf16<false>(x[nb], w[0][0], w[1][0], 0u, 0u, q.z[nb][2], 0u);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    const uint32_t x0 = kw[0][j], x1 = kw[1][j], y0 = x0 >> 8, y1 = x1 >> 8;
    const float s0 = step_of(km[0][j]), s1 = step_of(km[1][j]);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      float acc[4];
      mma0(acc, codes_low(at.masks, x0), codes_low(at.masks, x1), codes_high(at.masks, x0), codes_high(at.masks, x1), q.f[nb][2 * j][0], q.f[nb][2 * j][1]);
      mma(acc, codes_low(at.masks, y0), codes_low(at.masks, y1), codes_high(at.masks, y0), codes_high(at.masks, y1), q.f[nb][2 * j + 1][0], q.f[nb][2 * j + 1][1]);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        x[nb][c] = fmaf(s0, acc[c], x[nb][c]);
        x[nb][c + 2] = fmaf(s1, acc[c + 2], x[nb][c + 2]);
      }
    }
  }
}

// The tile's softmax and its share of the output; token0 is its first. wide: the products in f32.
template <int NG, int NB>
__device__ __forceinline__ void values(const uint8_t* stage, const Places& at, int token0, int keys, int sure, bool first, bool wide,
                                       const Query<NG, NB>& q, State<NG, NB>& s, const float (*raw)[4]) {
  using S = Shared<NG, NB>;
  const int lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
  uint32_t vm[2][NG];
#pragma unroll
  for (int h = 0; h < 2; ++h) load_words<NG>(vm[h], stage + 2 * S::kCodes + S::kScales + at.scale + 8 * h * NG * 4);
  float x[NB][4];
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 4; ++c) x[nb][c] = fmaf(raw[nb][c], q.scale[nb][c & 1], -s.m[nb][c & 1]);
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
  float step[2][NG], steps = 0.0f, tops = x[0][0];
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    step[0][j] = step_of(vm[0][j]);
    step[1][j] = step_of(vm[1][j]);
    steps = max3(steps, step[0][j], step[1][j]);
  }
  if (s.stepped + 1 != 1u << NG) {  // seldom after the first tile
#pragma unroll
    for (int j = 0; j < NG; ++j) s.stepped |= (step[0][j] + step[1][j] > 0.0f) << j;
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb) tops = max3(max3(tops, x[nb][0], x[nb][1]), x[nb][2], x[nb][3]);
  if (__any_sync(0xffffffffu, first || tops > kLazy || steps > s.vlimit)) {
    float fall = 1.0f;  // of o, when the steps' power of two moves
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) steps = fmaxf(steps, __shfl_xor_sync(0xffffffffu, steps, o));
    if (steps > s.vlimit) {
      const int ev = max(ilogbf(steps) - kStepTop, -120);
      if (s.vlimit > 0.0f) fall = s.ev - ev < -126 ? 0.0f : power(s.ev - ev);  // before the first step there is no o
      s.ev = ev;
      s.vlimit = fminf(power(ev) * kStepRoom, 0x1.fep127f);
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        // The base moves to the largest score, if that lies far above it; the first tile's scores set it. From the scores
        // themselves, rounded alike: relative to a base far away they have lost bits.
        const float scale = q.scale[nb][c];
        const float x0 = x[nb][c] == -INFINITY ? -INFINITY : __fmul_rn(raw[nb][c], scale);
        const float x1 = x[nb][c + 2] == -INFINITY ? -INFINITY : __fmul_rn(raw[nb][c + 2], scale);
        const float top = max_over_g(fmaxf(x0, x1)), was = s.m[nb][c];
        const float m = first ? (top == -INFINITY ? 0.0f : top) : top - was > kLazy ? top : was;
        const float f = first ? 0.0f : exp2_(was - m), fo = f * fall;
        s.m[nb][c] = m;
        x[nb][c] = x0 - m;
        x[nb][c + 2] = x1 - m;
        s.l[nb][c] *= f;
#pragma unroll
        for (int j = 0; j < NG; ++j) {
          s.e[nb][j][c] *= f;
#pragma unroll
          for (int mm = 0; mm < 2; ++mm) {
            s.o[nb][j][mm][c] *= fo;
            s.o[nb][j][mm][c + 2] *= fo;
          }
        }
      }
  }
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      x[nb][c] = exp2_(x[nb][c]);
      s.l[nb][c & 1] += x[nb][c];
    }
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    const float z0 = fmaf(-8.0f, step[0][j], offset_of(vm[0][j])), z1 = fmaf(-8.0f, step[1][j], offset_of(vm[1][j]));
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) s.e[nb][j][c] = fmaf(x[nb][c], z0, fmaf(x[nb][c + 2], z1, s.e[nb][j][c]));
  }
  if (wide) {
    // token by token: its probabilities from the lane that has them, its codes of this lane's channels
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int left = min(8, keys - token0 - 8 * h);
#pragma unroll 1
      for (int tg = 0; tg < left; ++tg) {
        const int t = 8 * h + tg, chunk = g * NG * 2;
        uint32_t w[NG / 2];
        load_words<NG / 2>(w, stage + S::kCodes + t * (S::D / 2) + v_chunk<NG>(t, chunk >> 4) * 16 + (chunk & 15));
        const uint32_t* scale = (const uint32_t*)(stage + 2 * S::kCodes + S::kScales) + t * NG;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
          const float p0 = __shfl_sync(0xffffffffu, x[nb][2 * h], 4 * tg + i), p1 = __shfl_sync(0xffffffffu, x[nb][2 * h + 1], 4 * tg + i);
#pragma unroll
          for (int j = 0; j < NG; ++j) {
            const float v = step_of(scale[j]);
            const float v0 = p0 * v, v1 = p1 * v;
            const uint32_t codes = (w[j >> 1] >> (16 * (j & 1))) ^ 0x8888u;  // code + 8 of the four channels
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float c = (float)(codes >> (4 * e) & 15u);
              float* o = &s.o[nb][j][e >> 1][2 * (e & 1)];
              o[0] = fmaf(v0, c, o[0]);
              o[1] = fmaf(v1, c, o[1]);
            }
          }
        }
      }
    }
  } else {
    // V: words of tokens 2 i, 2 i + 1, 2 i + 8, 2 i + 9
    uint32_t vw[4][NG / 2];
#pragma unroll
    for (int t = 0; t < 4; ++t)  // (2 i + 1) / 2 and (2 i + 8) / 2 mod 4 are i: the chunk is the same
      load_words<NG / 2>(vw[t], stage + S::kCodes + at.v + ((t & 1) + 8 * (t >> 1)) * (S::D / 2));
    const float down = power(-s.ev);
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 4; ++c) x[nb][c] *= down;
#pragma unroll
    for (int j = 0; j < NG; ++j) {
      const uint32_t sel = j & 1 ? 0x7632u : 0x5410u;
      const uint32_t x01 = __byte_perm(vw[0][j >> 1], vw[1][j >> 1], sel), x23 = __byte_perm(vw[2][j >> 1], vw[3][j >> 1], sel);
      const uint32_t y01 = x01 >> 8, y23 = x23 >> 8;
      const float s0 = step[0][j], s1 = step[1][j];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        const uint32_t b0 = transposed(f16x2(x[nb][0] * s0, x[nb][1] * s0));
        const uint32_t b1 = transposed(f16x2(x[nb][2] * s1, x[nb][3] * s1));
        mma(s.o[nb][j][0], codes_low(at.masks, x01), codes_high(at.masks, x01), codes_low(at.masks, x23), codes_high(at.masks, x23), b0, b1);
        mma(s.o[nb][j][1], codes_low(at.masks, y01), codes_high(at.masks, y01), codes_low(at.masks, y23), codes_high(at.masks, y23), b0, b1);
      }
    }
  }
}

// Whether the products of a run of n keys may have lost too much to f16's lower end, for the whole warp: some row's
// sum over some group is below 2^-14 n a channel, of codes + 8 that are 8 on average (the sum over its 32 channels is
// compared, first a lane's four by themselves: where each of them suffices nothing is exchanged).
template <int NG, int NB>
__device__ __forceinline__ bool too_small(const State<NG, NB>& s, int n) {
  auto lane_sum = [&](int nb, int j, int c) {
    return fmaf(s.o[nb][j][0][c] + s.o[nb][j][1][c], 0x1p24f, (s.o[nb][j][0][c + 2] + s.o[nb][j][1][c + 2]) * 0x1p20f);
  };
  const float least = (float)n * (0x1p-14f * 8.0f * 32.0f);
  bool low = false;
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
      for (int c = 0; c < 2; ++c) low |= lane_sum(nb, j, c) < least * 0.125f;
  if (!__any_sync(0xffffffffu, low)) return false;
  low = false;
  const uint32_t stepped = __reduce_or_sync(0xffffffffu, s.stepped);
#pragma unroll
  for (int j = 0; j < NG; ++j) {
    if (!(stepped >> j & 1)) continue;  // no step: products of zeros
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float sum = sum_over_g(lane_sum(nb, j, c)), l = sum_over_g(s.l[nb][c]);  // by all lanes
        low |= sum < least && l > 0.0f;
      }
  }
  return __any_sync(0xffffffffu, low);
}

// The warp's part of the output, its rows' maxima and sums.
template <int NG, int NB, typename Rows>
__device__ __forceinline__ void leave(const State<NG, NB>& st, bool wide, float* out, Rows& ml) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, i = lane & 3;
  const float even = wide ? 1.0f : 0x1p24f, odd = wide ? 1.0f : 0x1p20f, back = power(st.ev);
#pragma unroll
  for (int nb = 0; nb < NB; ++nb)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int r = nb * 8 + 2 * i + c;
      const float l = sum_over_g(st.l[nb][c]);
      if (g == 0) {
        ml[0][warp][r] = l > 0.0f ? st.m[nb][c] : kNone;
        ml[1][warp][r] = l;
      }
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        const float e = sum_over_g(st.e[nb][j][c]);
        *(float4*)(out + r * Shared<NG, NB>::kRow + j * kGroup + 4 * g) =
            make_float4(fmaf(st.o[nb][j][0][c] * even, back, e), fmaf(st.o[nb][j][0][c + 2] * odd, back, e),
                        fmaf(st.o[nb][j][1][c] * even, back, e), fmaf(st.o[nb][j][1][c + 2] * odd, back, e));
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
__global__ void __launch_bounds__(kThreads, tokens_blocks<NG, NB>()) tokens_kernel(const __grid_constant__ AttnArgs a) {
  using S = Shared<NG, NB>;
  using P = Partial<NG, NB>;
  constexpr int D = S::D, R = S::R;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float ml[2][kWarps][R];
  __shared__ float4 shares_of[kThreads];
  __shared__ int last;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // rows_kernel, if it is launched behind, may begin: it works on other sequences, in memory of its own
  asm volatile("griddepcontrol.launch_dependents;");
  const Start start = share_start<kThreads>(
      a.batch, kLeast, kByRoot, [&](int b) { return units<R>(a, sequence(a, b)); },
      [&](int b) {
        const Seq s = sequence(a, b);
        return s.rows >= a.long_rows ? 0 : tiles_of(s);
      });
  if ((int)blockIdx.x >= start.blocks) return;
  const Shares shares(start.total, start.blocks);
  long long unit = shares.first(blockIdx.x);
  const long long end = shares.first(blockIdx.x + 1);
  int b = start.b;
  long long seq_at = start.seq_at;
  Seq s = sequence(a, b);

  const Places at = places<NG>();
  uint8_t* ring = smem + warp * S::kRing;
  const uint32_t ring_u32 = smem_u32(ring) + lane * 16;
  // what a lane copies of a tile, from where and to where: chunks lane, lane + 32, ... of K and of V, and with
  // one half of the lanes K's scales, with the other V's
  constexpr int kHalf = S::kScaleLanes < 32 ? S::kScaleLanes / 2 : 16;
  const uint8_t* k_lane = a.cache.k + lane * 16;
  const int64_t v_from_k = a.cache.v - a.cache.k;
  const uint8_t* scale_lane =
      lane < kHalf ? (const uint8_t*)a.cache.k_scale + lane * 16 : (const uint8_t*)a.cache.v_scale + (lane - kHalf) * 16;
  // relative to lane * 16, where the lane's K codes go; a second V chunk is 8 (D = 128: 32 chunks on, the same
  // place in its row) or 4 (D = 256) tokens on
  const int scale_to = kept(2 * S::kCodes + (lane < kHalf ? 0 : S::kScales - kHalf * 16));
  const int v_to0 = kept(S::kCodes + (v_chunk<NG>(lane / NG, lane % NG) - lane % NG) * 16);
  const int v_to1 = NG == 8 ? kept(S::kCodes + (v_chunk<NG>(lane / NG + 4, lane % NG) - lane % NG) * 16) : v_to0;
  while (unit < end) {
    while (unit >= seq_at + units<R>(a, s)) {
      seq_at += units<R>(a, s);
      s = sequence(a, ++b);
    }
    const int tiles = tiles_of(s), length = tiles + kSegmentCost;
    const int seg = (int)quotient(unit - seq_at, length);
    const long long seg_at = seq_at + (long long)seg * length;
    // its cost stands before its first tile; a share that ends within it has no tile here
    const int u1 = (int)min((long long)length, end - seg_at);
    const int t0 = max(0, (int)(unit - seg_at) - kSegmentCost), t1 = u1 - kSegmentCost;
    const int head = seg % a.cache.heads, row0 = seg / a.cache.heads * R;
    unit = seg_at + u1;
    if (t1 <= t0) continue;

    // keys that any row of the block sees, and that every row sees
    const int rows = min(R, s.rows - row0);
    const int most = seen(a, s, row0 + rows - 1);
    const int sure = seen(a, s, row0);
    State<NG, NB> st;
    bool first;
    // This warp's run of the segment's tiles, with products in f16 and, if they lost too much, once more in f32.
    for (bool wide = false;; wide = true) {
      st.clear(wide);
      // the run's 16-token tiles, and where in which page it begins
      const int tiles16 = max(0, (min(t1 * kTileTokens, most) - t0 * kTileTokens + 15) / 16);
      int n = t0 * kWarps + tiles16 * warp / kWarps;
      const int n1 = t0 * kWarps + tiles16 * (warp + 1) / kWarps;
      const int32_t* table = a.table + (int64_t)b * a.width;
      int page_at = (int)fdiv(a.cache.by_page, (uint32_t)n * 16);  // entry of the table that `page` is
      const int page_end = (n1 * 16 + a.cache.page_size - 1) / a.cache.page_size;
      const int begin = n * 16 - page_at * a.cache.page_size;  // within the first page
      int left = (a.cache.page_size - begin) / 16;             // tiles of the page not yet fetched
      int page = n < n1 ? table[page_at] : 0;
      int fetched = n;
      // a page of all heads is less than 2^32 bytes: its number times that is one instruction
      const uint32_t page_codes = (uint32_t)a.cache.heads * a.cache.page_size * (D / 2);
      const uint32_t page_scales = (uint32_t)a.cache.heads * a.cache.page_size * (NG * 4);
      const uint8_t* k_head = k_lane + (int64_t)head * a.cache.page_size * (D / 2);
      const uint8_t* sc_head = scale_lane + (int64_t)head * a.cache.page_size * (NG * 4);
      const uint8_t *k, *sc;
      bool there;
      auto enter = [&] {  // the page's first rows
        there = (uint32_t)page < (uint32_t)a.cache.pages;
        if (!there && lane == 0) atomicExch(a.bad, kBadPage);
        k = k_head + (uint64_t)(uint32_t)page * page_codes;
        sc = sc_head + (uint64_t)(uint32_t)page * page_scales;
        page = ++page_at < page_end ? table[page_at] : 0;  // for the next time
      };
      RawQuery<NG, NB> raw;  // on its way with the page number
      raw.load(a, s, head, row0);
      if (n < n1) {
        enter();
        k += begin * (D / 2);
        sc += begin * (NG * 4);
      }
      uint32_t into = 0, from = 0;  // stages, in bytes
      auto fetch = [&] {
        if (fetched < n1) {
          if (left == 0) {
            left = a.cache.page_size / 16;
            enter();
          }
          const uint32_t to = ring_u32 + into;
          if (there) {
#pragma unroll
            for (int c = 0; c * 32 < S::kCodes / 16; ++c) copy16(to + c * 512, k + c * 512);
#pragma unroll
            for (int c = 0; c * 32 < S::kCodes / 16; ++c) copy16(to + (c & 1 ? v_to1 : v_to0) + c * 512, k + v_from_k + c * 512);
#pragma unroll
            for (int c = 0; c * 32 < S::kScaleLanes; ++c)
              if (lane < S::kScaleLanes) copy16(to + scale_to + c * 256, sc + c * 256);
          } else {
            for (int c = lane; c < S::kStage / 16; c += 32) *(uint4*)(ring + into + c * 16) = make_uint4(0, 0, 0, 0);
          }
          k += S::kCodes;
          sc += S::kScales;
          --left;
          ++fetched;
        }
        copies_commit();
        into = into + S::kStage == S::kRing ? 0 : into + S::kStage;
      };
#pragma unroll 1
      for (int c = 0; c < kStages - 1; ++c) fetch();
      Query<NG, NB> q;
      load_query<NG, NB>(a, s, row0, raw, q);  // while the first keys are on their way
      // A tile's scores are computed while the tile before is finished: two independent chains of instructions.
      auto next_stage = [](uint32_t at) { return at + S::kStage == S::kRing ? 0 : at + S::kStage; };
      float x[NB][4];
      if (n < n1) {
        copies_wait<kStages - 2>();
        __syncwarp();
        scores<NG, NB>(ring, at, q, x);
      }
      first = true;
#pragma unroll 1
      for (; n < n1; ++n) {
        fetch();
        copies_wait<kStages - 2>();
        __syncwarp();
        const uint32_t then = next_stage(from);
        float ahead[NB][4];
        scores<NG, NB>(ring + then, at, q, ahead);  // behind the last tile: of what the stage holds, and not used
        values<NG, NB>(ring + from, at, n * 16, s.keys, sure, first, wide, q, st, x);
        first = false;
        __syncwarp();  // all lanes have read the stage before the next copies into it
        from = then;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int c = 0; c < 4; ++c) x[nb][c] = ahead[nb][c];
      }
      copies_wait<0>();
      __syncwarp();  // the ring is drained: the warp's output goes over it
      if (!wide && !first && too_small<NG, NB>(st, (tiles16 / kWarps + 1) * 16)) continue;
      leave<NG, NB>(st, wide, (float*)ring, ml);
      break;
    }
    __syncthreads();

    auto write_row = [&](int r, int d, float4 v, float l) {  // channels d .. d + 3 of row r
      const int row = row0 + r;
      const float n = l != 0.0f ? 1.0f / l : 0.0f;  // a row that sees no key is 0
      const int token = token_of(a, row);
      *(uint2*)(a.o + ((int64_t)(s.q0 + token) * a.hq + head * a.group + row - token * a.group) * D + d) =
          make_uint2(bf16x2_rule(v.x * n, v.y * n), bf16x2_rule(v.z * n, v.w * n));
    };
    const bool whole = t0 == 0 && t1 == tiles;
    float* part = P::slot(a.ws, blockIdx.x, t0 == 0);
    for (int k = tid; k < rows * (D / 4); k += kThreads) {
      const int r = k / (D / 4), d = k % (D / 4) * 4;
      float m = kNone, l = 0.0f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ml[0][w][r]);
      float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float f = exp2_(ml[0][w][r] - m);
        const float4 v = *(const float4*)((const float*)(smem + w * S::kRing) + r * S::kRow + d);
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
      const int c0 = shares.owner(seg_at + kSegmentCost), c1 = shares.owner(seg_at + length - 1);
      __syncthreads();  // what the barrier has ordered before it, one thread's release below covers
      if (tid == 0) {
        last = arrive(a.counter + c0) == (uint32_t)(c1 - c0);
        if (last) a.counter[c0] = 0;
      }
      __syncthreads();
      if (last) {
        // Each part's weight of each row first, by all threads at once; then the sums over the parts, with the parts
        // of a column divided between threads where there are more threads than columns. (One token at 131072 keys
        // of one head: 29 us; 68 with every thread looking at all maxima by itself.)
        const int parts = c1 - c0 + 1, mr = lane % R;
        constexpr int kEach = 32 / R, kStep = kWarps * kEach;
        const int from = c0 + warp * kEach + lane / R;
        float* weight = (float*)smem;  // [part][row]
        auto across = [&](float v, auto f) {
#pragma unroll
          for (int o = R; o < 32; o <<= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
          return v;
        };
        float top = kNone;
        if (mr < rows) {
#pragma unroll 4
          for (int c = from; c <= c1; c += kStep) top = fmaxf(top, __ldcg(P::slot(a.ws, c, c == c0) + R * D + mr));
        }
        top = across(top, [](float x, float y) { return fmaxf(x, y); });
        if (lane < R) ml[0][warp][mr] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, ml[0][w][mr]);
        float l = 0.0f;
        if (mr < rows) {
#pragma unroll 4
          for (int c = from; c <= c1; c += kStep) {
            const float* p = P::slot(a.ws, c, c == c0) + R * D + mr;
            const float f = exp2_(__ldcg(p) - top);
            weight[(c - c0) * R + mr] = f;
            l = fmaf(f, __ldcg(p + R), l);
          }
        }
        l = across(l, [](float x, float y) { return x + y; });
        if (lane < R) ml[1][warp][mr] = l;
        __syncthreads();
        auto row_sum = [&](int r) {
          float t = 0.0f;
#pragma unroll
          for (int w = 0; w < kWarps; ++w) t += ml[1][w][r];
          return t;
        };
        const int columns = rows * (D / 4), split = max(1, kThreads / columns);
        for (int k = tid; k < columns * split; k += kThreads) {
          const int of = split > 1 ? k / columns : 0, column = k - of * columns;
          const int r = column / (D / 4), d = column % (D / 4) * 4;
          float4 sum = make_float4(0, 0, 0, 0);
#pragma unroll 8
          for (int c = of; c < parts; c += split) {
            const float f = weight[c * R + r];
            const float4 v = __ldcg((const float4*)(P::slot(a.ws, c0 + c, c == 0) + r * D + d));
            sum.x = fmaf(f, v.x, sum.x), sum.y = fmaf(f, v.y, sum.y), sum.z = fmaf(f, v.z, sum.z), sum.w = fmaf(f, v.w, sum.w);
          }
          if (split == 1) write_row(r, d, sum, row_sum(r));
          else shares_of[k] = sum;
        }
        if (split > 1) {
          __syncthreads();
          if (tid < columns) {
            float4 sum = shares_of[tid];
            for (int of = 1; of < split; ++of) {
              const float4 v = shares_of[of * columns + tid];
              sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
            }
            write_row(tid / (D / 4), tid % (D / 4) * 4, sum, row_sum(tid / (D / 4)));
          }
        }
      }
    }
    __syncthreads();  // the outputs are read before the next segment's copies
  }
}

constexpr int kCounters = 1024;  // of each kernel, one for each block

template <int NG, int NB>
size_t tokens_workspace(int sms) { return (size_t)sms * tokens_blocks<NG, NB>() * 2 * Partial<NG, NB>::kFloats * sizeof(float); }

template <int NG, int NB>
void launch_tokens(fopt_ctx* ctx, const AttnArgs& a, int sms) {
  using S = Shared<NG, NB>;
  static std::atomic<uint64_t> done;
  require(sms * tokens_blocks<NG, NB>() * S::R * 4 <= S::kBytes, "fopt_cache_attention: more resident blocks than a block adds up");
  allow_shared(ctx, done, (const void*)tokens_kernel<NG, NB>, S::kBytes);
  tokens_kernel<NG, NB><<<sms * tokens_blocks<NG, NB>(), kThreads, S::kBytes, ctx->stream>>>(a);
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
    require((int64_t)tokens * hq <= INT32_MAX, "fopt_cache_attention: too many query rows");
    if (ctx && (batch == 0 || tokens == 0)) return;
    require(o && q && table && q_start && kv_len, "fopt_cache_attention: null argument");
    require((uintptr_t)o % 32 == 0 && (uintptr_t)q % 16 == 0,
            "fopt_cache_attention: q must be 16-byte and o 32-byte aligned");
    require(ctx != nullptr, "null context");
    DeviceGuard guard(ctx);
    a.o = (uint16_t*)o;
    a.q = (const uint16_t*)q;
    a.table = table;
    a.q_start = q_start;
    a.kv_len = kv_len;
    a.err = ctx->dev_err;
    a.bad = ctx->bad_index();
    a.batch = batch;
    a.tokens = tokens;
    a.width = table_width;
    a.hq = hq;
    a.group = hq / cache->heads;
    a.by_group = make_fastdiv((uint32_t)a.group);
    a.scale = scale;
    a.causal = causal != 0;
    const int sms = sm_count(ctx);
    require(sms * kv::kBlocks <= kv::kCounters, "fopt_cache_attention: more resident blocks than counters");
    const int dim = cache->head_dim;
    // 16 rows a block where a sequence has that many on average: the codes are expanded once for both halves
    const bool two = dim != 256 && (int64_t)tokens * a.group > 8 * (int64_t)batch;
    // Sequences of more than kv::kFewRows query rows go to rows_kernel, whose tiles of 256 rows take about as long
    // as that many rows of tokens_kernel. The lengths are the device's, so both are launched, unless no sequence can
    // be that long or the call has no more tokens than sequences: then it is single tokens, for which rows_kernel
    // would only begin and end (4 us).
    // A call that leaves most of the device to tokens_kernel's blocks is its own as well, for rows_kernel's few blocks
    // take longer to begin, to end and over each segment. What each block would have at most, in tiles of 64 keys, decides,
    // from the table's width; the more keys, the more rows_kernel's parts cost. At 8 key heads of 128 and 4 query heads
    // to each (us, rows_kernel / tokens_kernel): 40 queries at 512 keys 27.4 / 18.6 (4 tiles a block), 106 at 2048
    // 43.3 / 43.7 (26), 200 at 512 29.7 / 32.0 (16), 400 at 512 30.9 / 46.7 (32); of one head 400 at 2048 44.0 / 28.8
    // (12), 512 at 8192 65.8 / 76.7 (57), 256 64.5 / 49.3 (29), 16 of 8 query heads at 131072 177 / 85 (55).
    const int64_t width = (int64_t)table_width * cache->page_size;
    const int64_t segments = ((int64_t)tokens * a.group / (two ? 16 : 8) + batch) * cache->heads;
    const double tiles = (double)segments * (double)(width / kv::kTileTokens + 1 + kv::kSegmentCost) / (sms * (two ? 2 : kv::kBlocks));
    const bool light = tiles <= (double)(16 + std::min<int64_t>(width / 256, 64));
    const bool rows = tokens > batch && (int64_t)tokens * a.group > kv::kFewRows && !light;
    a.long_rows = rows ? kv::kFewRows + 1 : INT32_MAX;
    const size_t few = dim == 64 ? (two ? kv::tokens_workspace<2, 2>(sms) : kv::tokens_workspace<2, 1>(sms))
                     : dim == 128 ? (two ? kv::tokens_workspace<4, 2>(sms) : kv::tokens_workspace<4, 1>(sms))
                                  : kv::tokens_workspace<8, 1>(sms);
    // the counters first, so that no variant's partial results reach another's
    const size_t counters = 2 * kv::kCounters * sizeof(uint32_t);
    const size_t bytes = counters + few + (rows ? kv::rows_workspace(dim, sms) : 0);
    // In a capture that is not the context's own the graph takes the memory for its launches from the device's pool:
    // a workspace of the stream would be shared with all that the stream, or another graph of it, runs meanwhile.
    cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
    if (!ctx->capture && ctx->stream) cuda_check(cudaStreamIsCapturing(ctx->stream, &capture), "capture status");
    const bool borrowed = capture != cudaStreamCaptureStatusNone;
    uint8_t* ws = nullptr;
    if (borrowed) {
      cuda_check(cudaMallocAsync((void**)&ws, bytes, ctx->stream), "cache workspace alloc");
      cuda_check(cudaMemsetAsync(ws, 0, counters, ctx->stream), "cache workspace clear");
    } else {
      ws = (uint8_t*)cache_workspace(ctx, bytes);
    }
    a.counter = (uint32_t*)ws;
    a.ws = (float*)(ws + counters);
    switch (dim) {
      case 64: two ? kv::launch_tokens<2, 2>(ctx, a, sms) : kv::launch_tokens<2, 1>(ctx, a, sms); break;
      case 128: two ? kv::launch_tokens<4, 2>(ctx, a, sms) : kv::launch_tokens<4, 1>(ctx, a, sms); break;
      default: kv::launch_tokens<8, 1>(ctx, a, sms); break;
    }
    if (rows) {
      a.counter += kv::kCounters;
      a.ws = (float*)(ws + counters + few);
      kv::launch_rows(ctx, a, dim, sms);
    }
    if (borrowed) cuda_check(cudaFreeAsync(ws, ctx->stream), "cache workspace free");
  });
}
