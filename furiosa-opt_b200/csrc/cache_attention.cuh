// Shared by the two kernels of attention over the paged 4-bit cache: the arguments, the division of a call's
// work between blocks, and the expansion of codes.
//
// The division: all (sequence, block of query rows, key head) segments of a call, each as long as its tiles of
// keys plus what beginning and ending a segment costs, form one line that is cut into equal shares, one per
// resident block, from the lengths on the device. So a call needs no lengths on the host, no block idles
// and any mixture of lengths balances. A segment cut between blocks leaves partial results (maximum, sum,
// output) in a workspace; the last of its blocks to arrive adds them up in the order of the keys, so results do
// not depend on timing. No block waits for another.
#pragma once

#include "kvcache.cuh"

namespace fopt {
namespace kv {

struct AttnArgs {
  uint16_t* o;
  const uint16_t* q;
  Cache cache;
  const int32_t* table;
  const int32_t* q_start;
  const int32_t* kv_len;
  int32_t* err;  // expired waits
  int32_t* bad;  // indices that were skipped
  float* ws;          // partial results: two slots a block
  uint32_t* counter;  // arrivals at the segment that begins in a block; zero between launches
  int batch, tokens, width, hq, group;
  FastDiv by_group;  // query row -> query token
  int long_rows;      // sequences with this many query rows per key head are rows_kernel's, others tokens_kernel's
  float scale;
  int causal;
};

constexpr int kMostKeys = INT32_MAX - 131071;  // so that tiles and pages past the last key stay within 32 bits
constexpr float kNone = -0x1p120f;  // the maximum of a part that has no score; its sum is 0

struct Seq {
  int q0, rows;  // first query token; query rows per key head (tokens x group)
  int queries, keys;
};

// Sequence b's query range and key count, cut to what the arguments allow.
__device__ __forceinline__ Seq sequence(const AttnArgs& a, int b) {
  const int s0 = a.q_start[b], s1 = a.q_start[b + 1], n = a.kv_len[b];
  Seq s;
  s.q0 = min(max(s0, 0), a.tokens);
  const int q1 = min(max(s1, s.q0), a.tokens);
  s.queries = q1 - s.q0;
  s.rows = s.queries * a.group;
  s.keys = (int)min((int64_t)min(max(n, 0), kMostKeys), (int64_t)a.width * a.cache.page_size);
  if (s.q0 != s0 || q1 != s1) atomicExch(a.bad, kBadStart);
  if (s.keys != n) atomicExch(a.bad, kBadLength);
  return s;
}
// Keys that the sequence's query row sees (at most 0: none).
__device__ __forceinline__ int token_of(const AttnArgs& a, int row) { return (int)fdiv(a.by_group, (uint32_t)row); }
__device__ __forceinline__ int seen(const AttnArgs& a, const Seq& s, int row) {
  return a.causal ? min(s.keys, s.keys - s.queries + token_of(a, row) + 1) : s.keys;
}

__device__ __forceinline__ long long quotient(long long a, long long b) {  // both >= 0; a 64-bit division takes long
  return ((a | b) >> 32) ? a / b : (long long)((uint32_t)a / (uint32_t)b);
}
// Of `total` units on n <= total blocks, the first total % n blocks have one more than the others.
struct Shares {
  long long each;
  int more;
  __device__ __forceinline__ Shares(long long total, int n) : each(quotient(total, n)), more((int)(total - each * n)) {}
  __device__ __forceinline__ long long first(int c) const { return each * c + min(c, more); }
  __device__ __forceinline__ int owner(long long unit) const {
    const long long wide = (each + 1) * more;
    return unit < wide ? (int)quotient(unit, each + 1) : more + (int)quotient(unit - wide, each);
  }
};

// Where a block's share begins: the line's length, the blocks that have a share, and the sequence in which this
// one's begins with the position of that sequence's first unit. For all threads of the block, with `units(b)`
// the length of sequence b, and `segment(b)` that of its longest segment. Shares have at least `least` units, and
// `by_root` sqrt(the longest segment): one block adds up a segment's parts one after the other, so n units in shares
// of u take u + (n / u) times what a part costs, least at u ~ sqrt(n). Blocks without a share get
// blocks <= blockIdx.x.
struct Start {
  long long total, seq_at;
  int blocks, b;
};
template <int THREADS, typename Units, typename Segment>
__device__ __forceinline__ Start share_start(int batch, int least, float by_root, Units units, Segment segment) {
  constexpr int kW = THREADS / 32;
  __shared__ long long sums[kW];
  __shared__ int tops[kW];
  __shared__ long long found_at;
  __shared__ int found;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long first = tid < batch ? units(tid) : 0;
  long long total = first;
  int top = tid < batch ? segment(tid) : 0;
  for (int b = tid + THREADS; b < batch; b += THREADS) {
    total += units(b);
    top = max(top, segment(b));
  }
  top = __reduce_max_sync(0xffffffffu, top);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) {
    sums[warp] = total;
    tops[warp] = top;
  }
  __syncthreads();
  total = 0;
#pragma unroll
  for (int w = 0; w < kW; ++w) {
    total += sums[w];
    top = max(top, tops[w]);
  }
  least = max(least, (int)(by_root * sqrtf((float)top)));
  Start st{total, 0, (int)min((long long)gridDim.x, (total + least - 1) / least), 0};
  if ((int)blockIdx.x >= st.blocks) return st;
  const long long unit = Shares(total, st.blocks).first(blockIdx.x);
  long long before = 0;  // units of the sequences before the chunk
  for (int b0 = 0;; b0 += THREADS) {
    const int b = b0 + tid;
    const long long u = b0 == 0 ? first : b < batch ? units(b) : 0;
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
#pragma unroll
    for (int w = 0; w < kW; ++w) {
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
  st.b = found;
  st.seq_at = found_at;
  return st;
}

__device__ __forceinline__ float exp2_(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ uint32_t f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low_half(uint32_t f16s) {
  float r;
  asm("{.reg .f16 a, b; mov.b32 {a, b}, %1; cvt.f32.f16 %0, a;}" : "=f"(r) : "r"(f16s));
  return r;
}
__device__ __forceinline__ float high_half(uint32_t f16s) {
  float r;
  asm("{.reg .f16 a, b; mov.b32 {a, b}, %1; cvt.f32.f16 %0, b;}" : "=f"(r) : "r"(f16s));
  return r;
}
__device__ __forceinline__ float sum_of(uint32_t f16s) { return low_half(f16s) + high_half(f16s); }
// A scale word's step and offset.
__device__ __forceinline__ float step_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float offset_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }
// A value that the compiler keeps in its register instead of computing it again from the lane number.
__device__ __forceinline__ int kept(int x) {
  asm volatile("" : "+r"(x));
  return x;
}
// Codes come out of a word of eight two at a time, as (x & mask) ^ flip: one lop3 with the mask in a register (with
// both constants immediate it takes two instructions).
struct Masks {
  uint32_t low, high;  // bits 0-3 and 16-19; bits 4-7 and 20-23
};
__device__ __forceinline__ Masks masks() { return {(uint32_t)kept(0x000f000f), (uint32_t)kept(0x00f000f0)}; }
__device__ __forceinline__ uint32_t masked(uint32_t x, uint32_t mask, uint32_t flip) {
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(r) : "r"(x), "r"(mask), "r"(flip));
  return r;
}

__device__ __forceinline__ float power(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }  // e in -126 .. 127
// A row of queries whose largest magnitude, as bf16 bits, is `top` in [2^e, 2^(e + 1)) times 2^(8 - e) is f16 with full
// precision. Below 2^-118 rows stay smaller.
__device__ __forceinline__ int row_exponent(uint32_t top) { return max((int)(top >> 7) - 127, -118); }

// Launches rows_kernel for the sequences of at least a.long_rows rows (head_dim 64 or 128). `ws` holds
// rows_workspace() bytes; `counter` two counters per SM.
size_t rows_workspace(int head_dim, int sms);
void launch_rows(fopt_ctx* ctx, const AttnArgs& a, int head_dim, int sms);

}  // namespace kv
}  // namespace fopt
