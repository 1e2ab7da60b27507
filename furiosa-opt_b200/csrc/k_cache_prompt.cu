// Attention over the paged 4-bit cache for sequences with many query rows (prompts and pieces of them), on the
// fifth-generation tensor cores.
//
// The query rows of one key head are (token, query head of its group) pairs; a segment is 256 of them, as two
// 128-row tiles, against all keys that they see, in tiles of 128 tokens. 512 threads, one block an SM:
//   warp 0      owns tensor memory and issues, per key tile, S_t = Q_t K^T and O_t += P_t V for t = 0, 1;
//   warps 1-7   expand codes, in turn K or V of 32 tokens: a lane takes one token, reads its row straight from the
//               cache's pages (64 contiguous bytes at D = 128) ahead of its turn, and writes it as f16 into the
//               128-byte-swizzled tile (three warps took longer than a tile's products);
//   warps 8-15  softmax: a thread per query row reads its scores from tensor memory, keeps the running maximum and
//               sum, and writes P as f16 over the first half of its scores.
// The roles' loops are short on purpose. They run side by side, and unrolled over a tile (500 to 600 instructions each)
// they missed the instruction cache so often that an instruction took 10 cycles a warp, the more the more warps.
// While one tile's softmax runs the tensor cores work on the other. Every wait is bounded (2 s) and reports
// through the context's error word.
//
// K's offsets go in apart: a code times its step has 3 + 8 bits and is exact in f16, where code * step + offset
// would be rounded (to 2^-12 of K, which sharp scores of a hundred and more turn into percents of P). The offsets'
// share of a score, sum_groups offset (sum of q), is one more step of the same product, over k = (part, group) with
// the sums of q in two f16 parts.
//
// f16 holds 11 bits of a value where bf16 would hold 8, but not every size of it: every 32 tokens' K is scaled by a
// power of two and V by another, so that the largest is in [2^4, 2^9); where tokens are more than 2^6 apart, each by
// its own, so that a large one, hidden or of no weight, takes nothing from its neighbours. K's comes back with the
// scores. V's, 2^ev, goes into the exponent: with x = score + ev, P = 2^(x - m) and O = sum P V 2^-ev, where the base m
// follows the largest x, which P brings to 2^10 at least: f16 holds 24 bits below that, so tokens of little weight
// count, a hundred thousand of them too. What one scale has to hold are the groups of 32 channels of one token: 2^-18
// of the largest and less loses bits.
//
// The sum of probabilities has a base of its own, a score n near the largest: l = sum P 2^(m - ev - n), so that V's
// size takes nothing from its range; outputs are O / l 2^(m - n).
//
// A 16-byte chunk holds 8 codes in the order that pairs come out of a word (0, 4, 1, 5, 2, 6, 3, 7): for K the
// queries are stored in the same order, for V the output's columns are put right when they leave.
//
// What bounds it: the tensor cores take 34 steps of M 128, N 128, K 16 per key tile (about 3300 cycles, 1.75 us); the
// exponentials take 2048, the expansion about 450 issue slots of each scheduler. A period is 3.2 us, since each of the
// two tiles takes about 2 us of softmax and then waits for 0.9 us of products: 150 us for 4 pieces of 512 tokens at 512
// to 4096 keys, 8 key heads of 128 and 4 query heads to each (0.52 PFLOP/s), 81 us for 8 prompts of 512, where 5.5 us
// around the 1 to 4 periods of a segment go into its queries, first scores and output. Tiles whose tokens have
// exponents of their own take three times as long (431 us for the pieces if all had).
#include "cache_attention.cuh"
#include "tcgen05.cuh"

namespace fopt {
namespace kv {
namespace {

using namespace attn;

constexpr int kRowThreads = 512;         // 128 registers each
constexpr int kHalf = 16384;             // 128 rows of 64 f16 (128 bytes), the unit of the swizzled tiles
constexpr int kOffsets = 128 * 32;        // 128 rows of 16 f16: the sums of a tile's q (or the offsets of 128 keys)
constexpr int kCost = 2;                 // key tiles that beginning and ending a segment takes as long as
constexpr int kLeast = 4;                // units of a share
// A part more to add up (66 KB for each of two tiles, by one SM) takes about as long as a unit. Of 16 tokens at 131072
// keys of one head of 8 query heads: 177 us; 347 without this rule, in shares of 7 units (159 with it then).
constexpr float kByRoot = 1.0f;
constexpr int kUncut = 8;                // segments of fewer tiles are not shared between blocks
// log2 of the largest P as the base is set, and up to which it may grow before the base moves. (On the cases above
// 10 to 15 take no longer than 0 to 14.)
constexpr float kNominal = 10.0f, kMostP = 15.0f;
constexpr int kEven = 6;                  // log2 by which 32 tokens' sizes may differ under one scale
constexpr float kLazySum = 20.0f;         // ... and a score that of l, where it is looked at
constexpr float kFarScore = 0x1p22f;      // up to which bases and V's exponents add up exactly
constexpr float kFarBack = 80.0f;         // log2 up to which P gives its share of l: probabilities below 2^-46 may vanish
constexpr float kLog2e = 1.44269504088896340736f;

// At D = 256 one 128-row tile of queries and 64 keys at a time are what tensor memory (64 columns of scores, 256 of
// outputs) and shared memory hold; products and softmax take turns. 512 queries at 2382 keys and 370 at 370, 3 key
// heads and 5 query heads to each: 84 us (210 by tokens_kernel).
template <int NG>
struct Tiles {
  static constexpr int D = NG * kGroup, kHalves = D / 64;
  static constexpr int kQueries = NG == 8 ? 1 : 2, kRows = 128 * kQueries;  // row tiles and rows of a segment
  static constexpr int kKeys = NG == 8 ? 64 : 128, kQuarters = kKeys / 32;  // of a key tile, and a warp's turns with its K
  // Warps that expand codes. More than a tile and a half of turns would let a warp come to a stage two uses ahead, which
  // the parity that it waits for could not tell: as it is, its turn before has waited for a product that comes, in the
  // order of issue, behind the stage's last use but one.
  static constexpr int kExpand = NG == 8 ? 6 : 7;
  static constexpr int kQ = kHalves * kHalf;         // bytes of Q_t
  static constexpr int kKeyHalf = kKeys * 128, kTile = kHalves * kKeyHalf;  // of 64 channels of a key tile, of K or V
  static constexpr int kKeyOffsets = kKeys * 32;     // of its offset step
  // Q, 2 stages of K and of V, the offset steps of Q and K, alignment, barriers and scales; more than half an
  // SM's, since a second block would only wait for tensor memory
  static constexpr int kRaw = 32 * NG * 16;  // what a warp holds of 32 tokens' K or V
  static constexpr int kExponents = 4 * kKeys;  // of K, and of V: a byte for each token of four key tiles
  static constexpr int kAll = kQueries * (kQ + kOffsets) + 4 * kTile + 2 * kKeyOffsets + kExpand * kRaw + 1024 + 512 + 2 * kExponents;
  static constexpr int kBytes = kAll > 120000 ? kAll : 120000;
  static constexpr int kSlot = kRows * (D + 3);      // floats of a partial result

  static __device__ __forceinline__ int blocks_of(const Seq& s) { return (s.rows + kRows - 1) / kRows; }
  // Key tiles of a row block: up to the last key that its last row sees, one at least.
  static __device__ __forceinline__ int tiles_of(const AttnArgs& a, const Seq& s, int rb) {
    return max(1, (max(0, seen(a, s, min(s.rows, (rb + 1) * kRows) - 1)) + kKeys - 1) / kKeys);
  }
  static __device__ __forceinline__ long long units(const AttnArgs& a, const Seq& s) {
    if (s.rows < a.long_rows) return 0;
    long long n = 0;
    for (int rb = 0; rb < blocks_of(s); ++rb) n += tiles_of(a, s, rb) + kCost;
    return n * a.cache.heads;
  }
};

struct Item {
  Seq s;
  int b, head, row0;
  int t0, t1, tiles;  // this block's key tiles of the segment, and all of them
  long long at;       // the segment's first unit
};

// A block's segments in order. Every role of the block walks them by itself.
template <typename T>
struct Walk {
  const AttnArgs& a;
  long long pos, end, rb_at;
  int b, rb;
  Seq s;

  __device__ __forceinline__ Walk(const AttnArgs& args, const Start& st, const Shares& sh)
      : a(args), pos(sh.first(blockIdx.x)), end(sh.first(blockIdx.x + 1)), rb_at(st.seq_at), b(st.b), rb(0),
        s(sequence(args, st.b)) {}

  __device__ bool next(Item& it) {
    while (pos < end) {
      int length;
      for (;;) {  // the row block that holds pos
        if (s.rows < a.long_rows || rb == T::blocks_of(s)) {
          s = sequence(a, ++b);
          rb = 0;
          continue;
        }
        length = T::tiles_of(a, s, rb) + kCost;
        if (pos < rb_at + (long long)length * a.cache.heads) break;
        rb_at += (long long)length * a.cache.heads;
        ++rb;
      }
      const int head = (int)quotient(pos - rb_at, length);
      const long long at = rb_at + (long long)head * length;
      int from = (int)(pos - at), to = (int)min((long long)length, end - at);
      if (length < kUncut + kCost) {  // whole, to the block on whose side of the cut its middle is
        if (from > 0) {
          if (2 * from >= length) {
            pos = at + length;
            continue;
          }
          from = 0;
        }
        if (to < length) {
          if (2 * to < length) {
            pos = end;
            break;
          }
          to = length;
        }
      }
      pos = at + to;
      it.t0 = max(0, from - kCost);
      it.t1 = to - kCost;
      if (it.t1 <= it.t0) continue;  // within its cost, which stands before its first tile
      it.s = s;
      it.b = b;
      it.head = head;
      it.row0 = rb * T::kRows;
      it.tiles = length - kCost;
      it.at = at;
      return true;
    }
    return false;
  }
};

// Eight codes of a word as four f16 pairs code * step + offset. The codes are exact first: 1024 + (code + 8) - 1032
// and (1024 + 16 (code + 8)) / 16 - 72.
__device__ __forceinline__ uint4 expand(const Masks& m, uint32_t x, uint32_t step, uint32_t offset) {
  auto value = [&](uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(c), "r"(step), "r"(offset));
    return r;
  };
  auto low = [&](uint32_t w) {
    uint32_t r;
    asm("add.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(masked(w, m.low, 0x64086408u)), "r"(0xe408e408u));
    return value(r);
  };
  auto high = [&](uint32_t w) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(masked(w, m.high, 0x64806480u)), "r"(0x2c002c00u), "r"(0xd480d480u));
    return value(r);
  };
  const uint32_t y = x >> 8;
  return make_uint4(low(x), high(x), low(y), high(y));
}

// Scores of keys from `left` on become -inf.
__device__ __forceinline__ void hide(uint32_t* s, int left) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (i >= left) s[i] = 0xff800000u;
}

// Two outputs times `by` as bf16 under the library's rule (half to even, subnormals to signed zero, one NaN).
__device__ __forceinline__ uint32_t rounded(float lo, float hi, float by) {
  float x, y;
  asm("mul.ftz.f32 %0, %1, %2;" : "=f"(x) : "f"(lo), "f"(by));
  asm("mul.ftz.f32 %0, %1, %2;" : "=f"(y) : "f"(hi), "f"(by));
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
  // an output is NaN where its row's sum is, the whole row
  return by == by ? r : 0x7fc07fc0u;
}

__device__ __forceinline__ void store32(void* p, const uint32_t* y) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]),
               "r"(y[4]), "r"(y[5]), "r"(y[6]), "r"(y[7])
               : "memory");
}

// Where chunk c (16 bytes) of row t of a tile is.
__device__ __forceinline__ uint32_t place(int t, int c) { return (c >> 3) * kHalf + t * 128 + (((c & 7) ^ (t & 7)) << 4); }
// ... and chunk c (0, 1) of row t of an offset step: unswizzled 8-row by 16-byte blocks, the two of a row group
// next to each other.
__device__ __forceinline__ uint32_t offsets_place(int t, int c) { return (t >> 3) * 256 + c * 128 + (t & 7) * 16; }
__device__ __forceinline__ uint64_t offsets_desc(uint32_t addr) {
  uint64_t d = (uint64_t)((addr & 0x3FFFF) >> 4);
  d |= (uint64_t)(128 >> 4) << 16;  // between the blocks of a row group (along k)
  d |= (uint64_t)(256 >> 4) << 32;  // between row groups
  d |= (uint64_t)1 << 46;
  return d;
}
__device__ __forceinline__ void async_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

template <int N>
__device__ __forceinline__ void load_row(uint32_t* w, const void* p, bool there) {
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = 0;
  if (!there) return;
  if constexpr (N == 2) *(uint2*)w = __ldg((const uint2*)p);
#pragma unroll
  for (int i = 0; i < N / 4; ++i) *(uint4*)(w + 4 * i) = __ldg((const uint4*)p + i);
}

// A token's place: its page (looked up ahead of its row) and the row's number in the images. Past the keys, or of no
// page: none, and zeros are what is read, whatever the slot holds.
struct Spot {
  int page, in_page;
  bool inside;
};
__device__ __forceinline__ Spot spot_of(const AttnArgs& a, const Item& it, int token) {
  Spot p{-1, 0, token < it.s.keys};
  if (p.inside) {
    const int entry = (int)fdiv(a.cache.by_page, (uint32_t)token);
    p.page = a.table[(int64_t)it.b * a.width + entry];
    p.in_page = token - entry * a.cache.page_size;
  }
  return p;
}
__device__ __forceinline__ bool row_at(const AttnArgs& a, const Item& it, const Spot& p, int64_t& row) {
  const bool there = p.page >= 0 && p.page < a.cache.pages;
  if (p.inside && !there) atomicExch(a.bad, kBadPage);
  row = there ? ((int64_t)p.page * a.cache.heads + it.head) * a.cache.page_size + p.in_page : 0;
  return there;
}

constexpr int kLowest = -120;  // of the exponents

// The exponents that bring the largest values of a warp's tokens to [2^4, 2^9), from the sizes of their groups: the
// largest of them for all, or, where they lie further apart than kEven, each its own. Zeros do not count: `none` if
// there is nothing else.
struct Exponents {
  int all, own;
  bool apart;
};
template <int NG>
__device__ __forceinline__ Exponents exponents(const uint32_t* scales, int none) {
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < NG; ++j) top = fmaxf(top, fmaf(8.0f, step_of(scales[j]), fabsf(offset_of(scales[j]))));
  const int size = (int)((__float_as_uint(top) & 0x7fffffffu) >> 23);
  const int most = __reduce_max_sync(0xffffffffu, size), least = __reduce_min_sync(0xffffffffu, size ? size : 255);
  auto exponent = [](int bits) { return min(max(bits - 127 - 4, kLowest), 120); };
  Exponents e{most ? exponent(most) : none, 0, most - least > kEven};
  e.own = e.apart ? exponent(size ? size : least) : e.all;
  return e;
}

// A tile's scores are the products times the row's factor and the keys' power of two: together not 0, for a hidden key's
// -inf is multiplied as well.
__device__ __forceinline__ float score_factor(float row, float keys) { return fmaxf(row * keys, 0x1p-126f); }

// A finite score's: an infinite one's row is NaN anyway.
__device__ __forceinline__ bool far_score(float base) { return fabsf(base) > kFarScore && fabsf(base) < INFINITY; }

// A row's bases: of l, and of O relative to it, so that a score far from zero takes nothing from V's exponents.
struct Bases {
  float l, o;
};
// The softmax of one tile by itself, 32 keys at a time, for tiles whose tokens have exponents of their own (k_own, v_own),
// and where one exponential does not serve both P and l or scores are too far from zero for the sums of bases that
// rows_kernel makes. Apart from it, so that the roles' code beside it stays as it is (within rows_kernel this cost
// 15 us of 142, called for or not). P goes over the scores; returns l, and moves the bases.
__device__ __noinline__ float own_tile(uint32_t scores, int keys, uint32_t outputs, int channels, int left, float qs, const int8_t* k_own,
                                       const int8_t* v_own, bool first, float l, Bases& base) {
  auto load = [&](int c, float* s) {
    tld32(scores + 32 * c, (uint32_t*)s);
    tld_wait_regs((uint32_t*)s);
    hide((uint32_t*)s, left - 32 * c);
#pragma unroll
    for (int i = 0; i < 32; ++i) s[i] = __fmul_rn(s[i], score_factor(qs, power(k_own[32 * c + i])));  // rounded as the base is
  };
  float most = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < keys / 32; ++c) {
    float s[32];
    load(c, s);
#pragma unroll
    for (int i = 0; i < 32; ++i) most = fmaxf(most, s[i]);
  }
  if (first) base = {most == -INFINITY ? 0.0f : rintf(most), 0.0f};
  else if (most > base.l + kLazySum) {
    const float up = rintf(most) - base.l;
    l *= exp2_(-up);
    base = {rintf(most), base.o - up};
  }
  float top = -INFINITY;
#pragma unroll 1
  for (int c = 0; c < keys / 32; ++c) {
    float s[32];
    load(c, s);
#pragma unroll
    for (int i = 0; i < 32; ++i) top = fmaxf(top, s[i] - base.l + (float)v_own[32 * c + i]);
  }
  const float was = base.o;
  if (first ? top != -INFINITY : top > was + kMostP) base.o = rintf(top) - kNominal;
  if (__any_sync(0xffffffffu, !first && base.o != was)) {
    const float f = exp2_(was - base.o);
#pragma unroll 1
    for (int c = 0; c < channels / 32; ++c) {
      float o[32];
      tld32(outputs + 32 * c, (uint32_t*)o);
      tld_wait_regs((uint32_t*)o);
#pragma unroll
      for (int i = 0; i < 32; ++i) o[i] *= f;
      tst32(outputs + 32 * c, (const uint32_t*)o);
    }
  }
#pragma unroll 1
  for (int c = 0; c < keys / 32; ++c) {
    float s[32];
    uint32_t p[16];
    load(c, s);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float x0 = s[i] - base.l, x1 = s[i + 1] - base.l;
      l += exp2_(x0) + exp2_(x1);
      p[i >> 1] = f16x2(exp2_(x0 + ((float)v_own[32 * c + i] - base.o)), exp2_(x1 + ((float)v_own[32 * c + i + 1] - base.o)));
    }
    tst16(scores + 16 * c, p);
  }
  return l;
}

template <int NG>
__global__ void __launch_bounds__(kRowThreads, 1) rows_kernel(AttnArgs a) {
  using T = Tiles<NG>;
  constexpr int D = T::D;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
  uint8_t* sQ = smem;  // tile t at sQ + t * kQ
  uint8_t* sK = smem + T::kQueries * T::kQ;  // stage n at sK + n * kTile
  uint8_t* sV = sK + 2 * T::kTile;
  uint8_t* sQz = sV + 2 * T::kTile;  // the offset steps: of tile t at sQz + t * kOffsets, of stage n at sKz + n * kKeyOffsets
  uint8_t* sKz = sQz + T::kQueries * kOffsets;
  uint8_t* raw = sKz + 2 * T::kKeyOffsets;  // rows as they are in the cache, of the expanding warps
  uint64_t* bars = (uint64_t*)(raw + T::kExpand * T::kRaw);
  uint64_t* k_full = bars;         // [2]
  uint64_t* k_empty = bars + 2;    // [2]
  uint64_t* v_full = bars + 4;     // [2]
  uint64_t* v_empty = bars + 6;    // [2]
  uint64_t* x_full = bars + 8;     // [4] the exponents of key tile n are in place n % 4
  uint64_t* q_full = bars + 12;    // [2] of tile t
  uint64_t* s_full = bars + 14;    // [2]
  uint64_t* p_ready = bars + 16;   // [2]
  uint64_t* o_done = bars + 18;    // [2] the segment's last product
  uint64_t* met = bars + 20;       // [2] the 128 softmax threads of a tile among themselves
  float* k_back = (float*)(bars + 22);  // [4][4] 2^ek of each 32 tokens of a key tile
  float* v_up = k_back + 16;            // [4][4] ev
  uint32_t* tmem_slot = (uint32_t*)(v_up + 16);
  volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
  int* last = (int*)(tmem_slot + 2);    // [2]
  uint64_t* apart = (uint64_t*)(last + 2);  // [4] a byte for K and V of each 32 tokens: do they have exponents of their own?
  int8_t* k_own = (int8_t*)bars + 512;      // [4][kKeys] the tokens' exponents
  int8_t* v_own = k_own + T::kExponents;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Start start = share_start<kRowThreads>(
      a.batch, kLeast, kByRoot, [&](int b) { return T::units(a, sequence(a, b)); },
      [&](int b) {
        const Seq s = sequence(a, b);
        return s.rows < a.long_rows ? 0 : T::tiles_of(a, s, T::blocks_of(s) - 1);
      });
  // The launch does not wait for tokens_kernel's end (they share nothing); this kernel's end does, for what follows.
  if ((int)blockIdx.x >= start.blocks) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    return;
  }
  const Shares shares(start.total, start.blocks);

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&k_full[i]), T::kQuarters);
      mbar_init(smem_u32(&k_empty[i]), 1);
      mbar_init(smem_u32(&v_full[i]), T::kQuarters);
      mbar_init(smem_u32(&v_empty[i]), 1);
      mbar_init(smem_u32(&q_full[i]), 128);
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&p_ready[i]), 128);
      mbar_init(smem_u32(&o_done[i]), 1);
      mbar_init(smem_u32(&met[i]), 128);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&x_full[i]), 2 * T::kQuarters);
      apart[i] = 0;
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  Walk<T> walk(a, start, shares);
  Item it;
  bool more = walk.next(it);  // the first segment, while tensor memory is allocated
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = *tmem_slot;  // S0, S1 (128 columns each), O0, O1 (at 256 and 384); or S0 and O0 of 256 columns

  if (warp == 0) {
    if (lane == 0) {
      // f16 x f16 -> f32, M = 128
      const uint32_t base = (1u << 4) | ((uint32_t)(128 >> 4) << 24);
      const uint32_t qk = base | ((uint32_t)(T::kKeys >> 3) << 17), pv = base | ((uint32_t)(D >> 3) << 17) | kIdescBMajorMN;
      auto scores = [&](int t, int n) {  // S_t of key tile n
        const uint64_t qd = sdesc(smem_u32(sQ + t * T::kQ)), kd = sdesc(smem_u32(sK + (n & 1) * T::kTile));
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          mma_bf16(tmem + t * 128, qd + ((uint32_t)((k >> 2) * kHalf + (k & 3) * 32) >> 4),
                   kd + ((uint32_t)((k >> 2) * T::kKeyHalf + (k & 3) * 32) >> 4), qk, k != 0);
        }
        mma_bf16(tmem + t * 128, offsets_desc(smem_u32(sQz + t * kOffsets)),
                 offsets_desc(smem_u32(sKz + (n & 1) * T::kKeyOffsets)), qk, 1);
        commit(smem_u32(&s_full[t]));
      };
      int n = 0, seg = 0;  // key tiles and segments so far
      bool ok = true;
      for (; ok && more; ++seg) {
        const int n1 = n + it.t1 - it.t0;
        ok = mbar_wait(smem_u32(&k_full[n & 1]), (n >> 1) & 1, abort_flag, a.err, 401);
        for (int t = 0; ok && t < T::kQueries; ++t) {
          ok = mbar_wait(smem_u32(&q_full[t]), seg & 1, abort_flag, a.err, 402);
          if (!ok) break;
          fence_after();
          scores(t, n);
        }
        if (ok) commit(smem_u32(&k_empty[n & 1]));
        more = walk.next(it);  // the next segment, while this one's scores are on their way
        for (int first = n; ok && n < n1; ++n) {
          for (int t = 0; ok && t < T::kQueries; ++t) {
            ok = (t || mbar_wait(smem_u32(&v_full[n & 1]), (n >> 1) & 1, abort_flag, a.err, 403)) &&
                 mbar_wait(smem_u32(&p_ready[t]), n & 1, abort_flag, a.err, 404);
            if (!ok) break;
            fence_after();
            const uint64_t vd = vdesc(smem_u32(sV + (n & 1) * T::kTile), T::kKeyHalf);
#pragma unroll
            for (int k = 0; k < T::kKeys / 16; ++k)
              mma_bf16_ta(tmem + 256 + t * 128, tmem + t * 128 + 8 * k, vd + (uint64_t)(128 * k), pv, (n - first) | k);
            const bool last_tile = t == T::kQueries - 1;
            if (last_tile) commit(smem_u32(&v_empty[n & 1]));
            if (n + 1 == n1) {
              commit(smem_u32(&o_done[t]));
            } else {
              // behind the product that reads P_t out of the same columns: one thread's MMAs run in order
              ok = t || mbar_wait(smem_u32(&k_full[(n + 1) & 1]), ((n + 1) >> 1) & 1, abort_flag, a.err, 405);
              if (!ok) break;
              fence_after();
              scores(t, n + 1);
              if (last_tile) commit(smem_u32(&k_empty[(n + 1) & 1]));
            }
          }
        }
      }
    }
    __syncwarp();
  } else if (warp <= T::kExpand) {
    const Masks m = masks();
    // The next row is on its way in registers while the current one is expanded from shared memory, where a loop can
    // index it: [piece of 16 bytes][lane]. A lane reads back what it wrote itself.
    uint4* mine = (uint4*)(raw + (warp - 1) * T::kRaw) + lane;
    uint4 codes[NG];
    uint32_t scales[NG];
    bool ok = true;
    int t = more ? it.t0 : 0;
    constexpr int kQuarters = T::kQuarters;
    int u = warp - 1, n = 0;  // which of a tile's turns (K of its quarters, then V), and the tile's number
    auto in_tile = [&] {  // ... when u has been counted on
      while (more && u >= 2 * kQuarters) {
        u -= 2 * kQuarters;
        ++n;
        if (++t == it.t1) {
          more = walk.next(it);
          t = it.t0;
        }
      }
    };
    in_tile();
    auto load = [&](const Spot& at) {
      int64_t row;
      const bool there = row_at(a, it, at, row);
      load_row<4 * NG>((uint32_t*)codes, (u < kQuarters ? a.cache.k : a.cache.v) + row * (NG * 16), there);
      load_row<NG>(scales, (u < kQuarters ? a.cache.k_scale : a.cache.v_scale) + row * NG, there);
    };
    if (more) load(spot_of(a, it, t * T::kKeys + u % kQuarters * 32 + lane));
    while (more) {
      const bool is_v = u >= kQuarters;
      const int quarter = u % kQuarters, row = quarter * 32 + lane, stage = n & 1, at4 = (n & 3) * 4 + quarter;
      const uint32_t full = smem_u32(is_v ? &v_full[stage] : &k_full[stage]);
      const uint32_t empty = smem_u32(is_v ? &v_empty[stage] : &k_empty[stage]), parity = ((n >> 1) & 1) ^ 1;
      const uint32_t known = smem_u32(&x_full[n & 3]);
      // zeros of V do not lift the base of P; what is past the keys has no part in it
      const Exponents e = exponents<NG>(scales, is_v && t * T::kKeys + quarter * 32 < it.s.keys ? kLowest : 0);
      const float f = power(-e.own);
      // by code word of a piece (of two, where K's group of words is two pieces): steps and offsets of what its pairs of
      // codes are (see the loop)
      constexpr int kWords = NG == 8 ? 8 : 4;
      uint32_t step[kWords], offset[kWords], z[8] = {};
#pragma unroll
      for (int w = 0; w < kWords; ++w) {
        const int g = NG == 2 ? w & 1 : w, h = NG == 2 ? 0 : NG == 4 ? w & 1 : w & 3;
        const float s = step_of(scales[g]) * f;
        step[w] = is_v ? f16x2(step_of(scales[2 * h]) * f, step_of(scales[2 * h + 1]) * f) : f16x2(s, s);
        offset[w] = is_v ? f16x2(offset_of(scales[2 * h]) * f, offset_of(scales[2 * h + 1]) * f) : 0;
      }
      // K's offsets: k = part * NG + group for the two parts of the sums of q, then zeros
#pragma unroll
      for (int j = 0; j < NG / 2; ++j)
        z[j] = z[j + NG / 2] = f16x2(offset_of(scales[2 * j]) * f, offset_of(scales[2 * j + 1]) * f);
#pragma unroll
      for (int i = 0; i < NG; ++i) mine[i * 32] = codes[i];
      // the next turn: its page is looked up while this one's row is expanded
      u += T::kExpand;
      in_tile();
      Spot next{-1, 0, false};
      if (more) next = spot_of(a, it, t * T::kKeys + u % kQuarters * 32 + lane);

      ok = mbar_wait(empty, parity, abort_flag, a.err, 411);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      // place n % 4: the softmax of tile n - 4 is over, or the product of n - 2 could not be
      (is_v ? v_own : k_own)[(at4 & ~3) * (T::kKeys / 4) + row] = (int8_t)e.own;
      __syncwarp();
      if (lane == 0) {
        if (is_v) v_up[at4] = (float)e.all;
        else k_back[at4] = power(e.all);
        ((uint8_t*)(apart + (at4 >> 2)))[(is_v ? 4 : 0) + quarter] = e.apart;
        mbar_arrive(known);
      }
      if (!is_v) {
        uint8_t* tz = sKz + stage * T::kKeyOffsets;
        *(uint4*)(tz + offsets_place(row, 0)) = make_uint4(z[0], z[1], z[2], z[3]);
        *(uint4*)(tz + offsets_place(row, 1)) = make_uint4(z[4], z[5], z[6], z[7]);
      }
      uint8_t* to = (is_v ? sV : sK) + stage * T::kTile + row * 128;
      // Word w of piece i is chunk: of K (words in the order of [D % 32 / 8, D / 32]) 4 group + run, of V its number.
      auto chunk_at = [&](int c) { return (uint4*)(to + (c >> 3) * T::kKeyHalf + (((c & 7) ^ (row & 7)) << 4)); };
      const int c1 = is_v ? 1 : 4, c2 = is_v ? 2 : NG == 2 ? 1 : 8, c3 = is_v ? 3 : NG == 2 ? 5 : 12;
      auto piece = [&](int i, int c, int from) {
        const uint4 w = mine[i * 32];
        *chunk_at(c) = expand(m, w.x, step[from], offset[from]);
        *chunk_at(c + c1) = expand(m, w.y, step[from + 1], offset[from + 1]);
        *chunk_at(c + c2) = expand(m, w.z, step[from + 2], offset[from + 2]);
        *chunk_at(c + c3) = expand(m, w.w, step[from + 3], offset[from + 3]);
      };
      if constexpr (NG == 8) {
#pragma unroll 1
        for (int i = 0; i < NG; i += 2) {
          piece(i, is_v ? 4 * i : i >> 1, 0);
          piece(i + 1, is_v ? 4 * i + 4 : 16 + (i >> 1), 4);
        }
      } else {
        const int by_piece = is_v ? 4 : NG == 4 ? 1 : 2;
#pragma unroll 1
        for (int i = 0; i < NG; ++i) piece(i, i * by_piece, 0);
      }
      load(next);
      async_fence();
      __syncwarp();
      if (lane == 0) mbar_arrive(full);
    }
  } else if (warp >= 8 && warp < 8 + 4 * T::kQueries) {
    const int t = (warp - 8) >> 2, quarter = warp & 3;  // tile, and the tensor-memory lanes that the warp may read
    const int r = quarter * 32 + lane;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t tS = tmem + t * 128 + lanes, tO = tmem + 256 + t * 128 + lanes;
    uint8_t* tq = sQ + t * T::kQ;

    // Rows of q and o (16 bytes a lane) start at their number * D.
    auto number = [&](const Item& x, int row) -> int {
      const int token = token_of(a, row);
      return (x.s.q0 + token) * a.hq + x.head * a.group + row - token * a.group;
    };
    constexpr int kPer = NG * 4, kAtOnce = 32 / kPer;  // lanes a row, rows at a time
    // Copies the warp's 32 queries as they are to their places in Q_t, kPer lanes to a row ...
    auto fetch_query = [&](const Item& x) {
      const int row = x.row0 + t * 128 + r, mine = row < x.s.rows ? number(x, row) : -1;
      const int chunk = lane % kPer;
#pragma unroll 4
      for (int k = 0; k < kPer; ++k) {
        const int in_warp = k * kAtOnce + lane / kPer, from = __shfl_sync(0xffffffffu, mine, in_warp);
        uint8_t* to = tq + place(quarter * 32 + in_warp, chunk);
        if (from >= 0)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to)), "l"(a.q + (int64_t)from * D + chunk * 8) : "memory");
        else
          *(uint4*)to = make_uint4(0, 0, 0, 0);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    // ... where each thread turns its row into f16, chunk by chunk, and sums its groups. Returns the factor of the row's
    // scores (K's powers of two aside).
    auto put_query = [&]() -> float {
      asm volatile("cp.async.wait_group 0;" ::: "memory");
      __syncwarp();
      uint32_t top = 0;  // of the magnitudes, as bf16 bits
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 w = *(const uint4*)(tq + place(r, c));
        top = __vmaxu2(top, __vmaxu2(__vmaxu2(w.x & 0x7fff7fffu, w.y & 0x7fff7fffu), __vmaxu2(w.z & 0x7fff7fffu, w.w & 0x7fff7fffu)));
      }
      top = max(top & 0xffffu, top >> 16);
      const int e = row_exponent(top);
      // the scale's sign goes into q, so that the largest score is the largest product
      const float up = a.scale < 0.0f ? -power(8 - e) : a.scale > 0.0f ? power(8 - e) : 0.0f;
      uint32_t z[8] = {};  // k = part * NG + group: the groups' sums in two f16 parts
#pragma unroll
      for (int j = 0; j < NG; ++j) {
        float sum = 0.0f;
#pragma unroll 2
        for (int i = 0; i < 4; ++i) {
          uint4* at = (uint4*)(tq + place(r, 4 * j + i));
          const uint4 w = *at;
          const uint32_t y[4] = {w.x, w.y, w.z, w.w};
          float v[8];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            v[2 * c] = step_of(y[c]) * up;
            v[2 * c + 1] = offset_of(y[c]) * up;
          }
          // 8 bits fit f16's 11 but for values below 2^-22 of the row's largest: the sum is that of what is stored
          sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
          *at = make_uint4(f16x2(v[0], v[4]), f16x2(v[1], v[5]), f16x2(v[2], v[6]), f16x2(v[3], v[7]));
        }
        const uint32_t one = f16x2(sum, 0.0f), two = f16x2(sum - low_half(one), 0.0f);
        z[j >> 1] |= j & 1 ? one << 16 : one & 0xffffu;
        z[(j + NG) >> 1] |= j & 1 ? two << 16 : two & 0xffffu;
      }
      uint8_t* tz = sQz + t * kOffsets;
      *(uint4*)(tz + offsets_place(r, 0)) = make_uint4(z[0], z[1], z[2], z[3]);
      *(uint4*)(tz + offsets_place(r, 1)) = make_uint4(z[4], z[5], z[6], z[7]);
      async_fence();
      mbar_arrive(smem_u32(&q_full[t]));
      return scalbnf(fabsf(a.scale) * kLog2e, e - 8);
    };

    uint32_t meetings = 0;
    auto meet = [&]() -> bool {  // a barrier of the tile's softmax threads whose wait is bounded
      mbar_arrive(smem_u32(&met[t]));
      const bool here = mbar_wait(smem_u32(&met[t]), meetings++ & 1, abort_flag, a.err, 424);
      return __all_sync(0xffffffffu, here);
    };
    auto scale_outputs = [&](float f) {  // the row's O_t, complete and not being added to
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        tld32(tO + 32 * c, o);
        tld_wait_regs(o);
#pragma unroll
        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tst32(tO + 32 * c, o);
      }
      tst_wait();
    };
    bool ok = true;
    Item done;  // the segment whose output is still in O_t
    float qs = 0.0f, l = 0.0f;
    Bases bases{0.0f, 0.0f};
    int n = 0;
    // Each part stands here once, in one place: the roles' code together has to stay in the instruction cache.
    for (int seg = 0; more || seg; ++seg) {
      // the scores of the segment before are complete, so Q_t is free: this one's query goes in before that one's
      // output leaves
      if (more) {
        fetch_query(it);
        qs = put_query();
      }
      if (seg) {
        ok = mbar_wait(smem_u32(&o_done[t]), (seg - 1) & 1, abort_flag, a.err, 423);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        const bool whole = done.t0 == 0 && done.t1 == done.tiles, rows = done.row0 + t * 128 < done.s.rows;
        // partial results: [D / 4][128] float4, so that a warp's rows are contiguous, then the bases and sums
        auto slot = [&](int block, bool begins) { return a.ws + ((int64_t)block * 2 + begins) * T::kSlot + t * 128 * (D + 3); };
        int c0 = 0, c1 = 0;
        bool output = rows;
        if (!whole && rows) {
          float* part = slot(blockIdx.x, done.t0 == 0);
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            tld32(tO + 32 * c, (uint32_t*)o);
            tld_wait_regs((uint32_t*)o);
#pragma unroll
            for (int i = 0; i < 8; ++i) ((float4*)part)[(8 * c + i) * 128 + r] = *(float4*)(o + 4 * i);
          }
          part[D * 128 + r] = l == 0.0f ? kNone : bases.l;  // a NaN sum stays one
          part[D * 128 + 128 + r] = bases.o;
          part[D * 128 + 256 + r] = l;
          c0 = shares.owner(done.at + kCost);
          c1 = shares.owner(done.at + done.tiles + kCost - 1);
          if (!(ok = meet())) break;
          if (r == 0) {
            __threadfence();  // covers what the meeting has ordered before it
            uint32_t* counter = a.counter + 2 * c0 + t;
            last[t] = atomicAdd(counter, 1u) == (uint32_t)(c1 - c0);
            if (last[t]) *counter = 0;
            __threadfence();
          }
          if (!(ok = meet())) break;
          output = last[t];
          if (!(ok = meet())) break;  // last[t] has been read
          if (output) {  // the parts' sum goes into O_t
            bases = {kNone, 2.0f * kNone};
            l = 0.0f;
#pragma unroll 4
            for (int c = c0; c <= c1; ++c) bases.l = fmaxf(bases.l, __ldcg(slot(c, c == c0) + D * 128 + r));
#pragma unroll 4
            for (int c = c0; c <= c1; ++c) {
              const float* q = slot(c, c == c0) + D * 128 + r;
              const float up = __ldcg(q) - bases.l;
              l = fmaf(exp2_(up), __ldcg(q + 256), l);
              bases.o = fmaxf(bases.o, up + __ldcg(q + 128));
            }
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              float o[32];
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0.0f;
#pragma unroll 2
              for (int b = c0; b <= c1; ++b) {
                const float* q = slot(b, b == c0);
                const float f = exp2_(__ldcg(q + D * 128 + r) - bases.l + __ldcg(q + D * 128 + 128 + r) - bases.o);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                  const float4 v = __ldcg((const float4*)q + (8 * c + i) * 128 + r);
                  o[4 * i] = fmaf(f, v.x, o[4 * i]), o[4 * i + 1] = fmaf(f, v.y, o[4 * i + 1]);
                  o[4 * i + 2] = fmaf(f, v.z, o[4 * i + 2]), o[4 * i + 3] = fmaf(f, v.w, o[4 * i + 3]);
                }
              }
              tst32(tO + 32 * c, (const uint32_t*)o);
            }
            tst_wait();
          }
        }
        if (output) {
          // 2^lift / l, which may lie outside f32 where the outputs do not: then a part of it goes in ahead
          float lift = bases.o;
          if (__any_sync(0xffffffffu, lift < -90.0f)) {
            scale_outputs(lift < -90.0f ? 0x1p-64f : 1.0f);
            if (lift < -90.0f) lift += 64.0f;
          }
          const float half = exp2_(0.5f * lift), scale = l != 0.0f ? 1.0f / l * half * half : 0.0f;
          const int row = done.row0 + t * 128 + r, mine = row < done.s.rows ? number(done, row) : -1;
          uint16_t* out = a.o + (int64_t)max(mine, 0) * D;
#pragma unroll 1
          for (int c = 0; c < D / 64; ++c) {
            float o[64];
            tld32(tO + 64 * c, (uint32_t*)o);
            tld32(tO + 64 * c + 32, (uint32_t*)o + 32);
            tld_wait_regs((uint32_t*)o);
            tld_wait_regs((uint32_t*)o + 32);
            if (mine < 0) continue;
            // 64 columns in the order of the codes -> 64 / NG neighbouring channels of each group, whole sectors
#pragma unroll
            for (int j = 0; j < NG; ++j) {
              uint32_t y[32 / NG];
#pragma unroll
              for (int i = 0; i < 32 / NG; ++i) {  // channels 2 i, 2 i + 1 of the run: code word `word`, its codes e, e + 1
                const int g = i / 2, word = g * (NG / 2) + j / 2, e = 2 * (i & 1);
                y[i] = rounded(o[8 * word + 2 * e + (j & 1)], o[8 * word + 2 * e + 2 + (j & 1)], scale);
              }
#pragma unroll
              for (int i = 0; i < 32 / NG / 8; ++i)
                store32(out + j * kGroup + c * (64 / NG) + 16 * i, y + 8 * i);
              if constexpr (NG == 8) *(uint4*)(out + j * kGroup + c * 8) = *(const uint4*)y;
            }
          }
        }
        // O_t may be overwritten: the arrival at p_ready of the next segment's first tile comes after these reads
        fence_before();
      }
      if (!more) break;
      done = it;
      more = walk.next(it);  // while the first scores are on their way
      const int row = done.row0 + t * 128 + r;
      const int limit = row < done.s.rows ? seen(a, done.s, row) : done.s.keys;  // rows past the last are not stored
      l = 0.0f;
      bases = {0.0f, 0.0f};
      for (int kt = done.t0; kt < done.t1; ++kt, ++n) {
        ok = mbar_wait(smem_u32(&x_full[n & 3]), (n >> 2) & 1, abort_flag, a.err, 421) &&
             mbar_wait(smem_u32(&s_full[t]), n & 1, abort_flag, a.err, 422);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        const int left = limit - kt * T::kKeys;  // keys of the tile that the row sees
        const bool cut = __any_sync(0xffffffffu, left < T::kKeys), first = kt == done.t0;
        const float* kb = k_back + (n & 3) * 4;
        const float* vu = v_up + (n & 3) * 4;
        // the largest x, then the base
        float top = -INFINITY, least = INFINITY;  // least: the smallest ev
        const int8_t *ko = k_own + (n & 3) * T::kKeys, *vo = v_own + (n & 3) * T::kKeys;
        const bool uneven = apart[n & 3] != 0;
#pragma unroll 1
        for (int h = 0; !uneven && h < T::kKeys / 64; ++h) {  // two loads at a time on their way
          uint32_t s[64];
          tld32(tS + 64 * h, s);
          tld32(tS + 64 * h + 32, s + 32);
          tld_wait_regs(s);
          tld_wait_regs(s + 32);
          if (cut) {
            hide(s, left - 64 * h);
            hide(s + 32, left - 64 * h - 32);
          }
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t* y = s + 32 * c;
            float high[2] = {__uint_as_float(y[0]), __uint_as_float(y[1])};
#pragma unroll
            for (int i = 2; i < 30; i += 4) {
              high[0] = max3(high[0], __uint_as_float(y[i]), __uint_as_float(y[i + 1]));
              high[1] = max3(high[1], __uint_as_float(y[i + 2]), __uint_as_float(y[i + 3]));
            }
            high[0] = max3(high[0], __uint_as_float(y[30]), __uint_as_float(y[31]));
            top = fmaxf(top, fmaf(fmaxf(high[0], high[1]), score_factor(qs, kb[2 * h + c]), vu[2 * h + c]));
            least = fminf(least, vu[2 * h + c]);
          }
        }
        // The bases are whole numbers, which makes the sums of them and V's exponents exact, up to kFarScore.
        const float was = bases.l + bases.o;
        const float m = first ? (top == -INFINITY ? 0.0f : rintf(top) - kNominal) : top > was + kMostP ? rintf(top) - kNominal : was;
        float ml = bases.l;
        if (first) {  // not above the largest score
          float largest = vu[0];
#pragma unroll
          for (int i = 1; i < T::kQuarters; ++i) largest = fmaxf(largest, vu[i]);
          ml = m - largest;
        }
        // Where V is far smaller than what set the base, or scores have risen far above l's, P has lost bits that l needs
        // (or l would pass f32's range).
        bool far = uneven || m - least - ml > kFarBack || far_score(m) || far_score(ml);
        if (__any_sync(0xffffffffu, far || (!first && m != was))) {
          far = __any_sync(0xffffffffu, far);
          // S_t was issued behind the last O_t += P_t V: it is complete
          if (!far && !first) scale_outputs(exp2_(was - m));
        }
        if (far) {
          Bases moved = bases;
          l = own_tile(tS, T::kKeys, tO, D, left, qs, ko, vo, first, l, moved);
          bases = moved;
        } else {
          bases = {ml, m - ml};
#pragma unroll 1
          for (int h = 0; h < T::kKeys / 64; ++h) {  // P goes over columns whose scores have been read: 16 c .. 16 c + 15
            uint32_t s[64];
            tld32(tS + 64 * h, s);
            tld32(tS + 64 * h + 32, s + 32);
            tld_wait_regs(s);
            tld_wait_regs(s + 32);
            if (cut) {
              hide(s, left - 64 * h);
              hide(s + 32, left - 64 * h - 32);
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float v_e = vu[2 * h + c], f = score_factor(qs, kb[2 * h + c]), up = v_e - m;
              const uint64_t f2 = pack_f32x2(f, f), up2 = pack_f32x2(up, up);
              uint64_t part[2] = {0, 0};
              uint32_t p[16];
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                float x0, x1;
                unpack_f32x2(fma_f32x2(pack_f32x2(__uint_as_float(s[32 * c + i]), __uint_as_float(s[32 * c + i + 1])), f2, up2), x0, x1);
                const float p0 = exp2_(x0), p1 = exp2_(x1);
                part[(i >> 1) & 1] = add_f32x2(part[(i >> 1) & 1], pack_f32x2(p0, p1));
                p[i >> 1] = f16x2(p0, p1);
              }
              tst16(tS + 32 * h + 16 * c, p);
              float s0, s1, s2, s3;
              unpack_f32x2(part[0], s0, s1);
              unpack_f32x2(part[1], s2, s3);
              l = fmaf((s0 + s1) + (s2 + s3), exp2_(m - v_e - ml), l);
            }
          }
        }
        tst_wait();
        fence_before();
        mbar_arrive(smem_u32(&p_ready[t]));
      }
      if (!ok) break;
    }
  }
  fence_before();
  __syncthreads();
  fence_after();
  if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

}  // namespace

size_t rows_workspace(int head_dim, int sms) {
  return (size_t)sms * 2 * (head_dim == 64 ? Tiles<2>::kSlot : head_dim == 128 ? Tiles<4>::kSlot : Tiles<8>::kSlot) * sizeof(float);
}

void launch_rows(fopt_ctx* ctx, const AttnArgs& a, int head_dim, int sms) {
  static std::atomic<uint64_t> done[3];
  auto go = [&](auto kernel, int smem) {
    allow_shared(ctx, done[head_dim / 128], (const void*)kernel, smem);
    // Beside tokens_kernel and not behind it: a batch of both kinds (6 sequences, 1999 keys the longest, 7 query heads
    // to a key head of 64) takes 34 us instead of 44, and where there are prompts alone tokens_kernel's empty launch
    // is hidden.
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = sms;
    cfg.blockDim = kRowThreads;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    cuda_check(cudaLaunchKernelEx(&cfg, kernel, a), "cache attention launch");
    launched(ctx, "cache attention");
  };
  if (head_dim == 64) go(rows_kernel<2>, Tiles<2>::kBytes);
  else if (head_dim == 128) go(rows_kernel<4>, Tiles<4>::kBytes);
  else go(rows_kernel<8>, Tiles<8>::kBytes);
}

}  // namespace kv
}  // namespace fopt
