// Shared by the kernels around the paged 4-bit key / value cache: the rotation's parameters, the cache's
// images and the argument checks of the entry points.
#pragma once

#include <algorithm>
#include <cmath>

#include "ctx.hpp"

namespace fopt {
namespace kv {

constexpr int kGroup = 32;      // channels that share a (step, offset)
constexpr int kMaxPairs = 128;  // rotated pairs of a head
constexpr int kSlots = 16;      // page sizes are multiples of this: attention's tile height

struct Rope {
  // Angle per position of each pair as a fraction of a turn, in 2^-64 turns: position * turn wraps modulo
  // one turn, so the product is the reduced angle with no rounding that grows with the position.
  unsigned long long turn[kMaxPairs];
  double magnitude;
  int pairs;  // 0: no rotation
  int interleaved;
};

struct Cache {
  uint8_t* k;
  uint8_t* v;
  uint32_t* k_scale;  // (step, offset) of a group as one word, the step in the low half
  uint32_t* v_scale;
  int pages, page_size, heads;
  FastDiv by_page;  // slot / page_size
};

// The checks that every call on a cache makes, and its images as kernels take them.
inline Cache checked(const fopt_paged_cache* c, const char* who) {
  const std::string w = std::string(who) + ": ";
  require(c && c->k && c->v && c->k_scale && c->v_scale, w + "null argument");
  require(((uintptr_t)c->k | (uintptr_t)c->v | (uintptr_t)c->k_scale | (uintptr_t)c->v_scale) % 16 == 0,
          w + "the cache's images must be 16-byte aligned");
  require(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, w + "head_dim must be 64, 128 or 256");
  require(c->heads > 0 && c->pages > 0, w + "empty cache");
  require(c->page_size > 0 && c->page_size % kSlots == 0 && c->page_size <= 65536,
          w + "page_size must be a multiple of 16, at most 65536");
  require((int64_t)c->pages * c->page_size <= INT32_MAX, w + "slots past 2^31");
  require((int64_t)c->heads * c->page_size * c->head_dim <= UINT32_MAX, w + "a page past 2^32 elements");
  Cache k{(uint8_t*)c->k, (uint8_t*)c->v, (uint32_t*)c->k_scale, (uint32_t*)c->v_scale, c->pages, c->page_size,
          c->heads, make_fastdiv((uint32_t)c->page_size)};
  return k;
}

// guarded(), with the message kept for fopt_last_error(NULL) too where there is no context: the checks of
// arguments come before the context is used, so a binding can be tested without a GPU.
template <typename Fn>
fopt_status checked_call(fopt_ctx* ctx, Fn&& fn) {
  return guarded(ctx, [&] {
    try {
      fn();
    } catch (const Fail& f) {
      if (!ctx) g_noctx_err = f.msg;
      throw;
    }
  });
}

// Row (page, head, slot of the page) as a row number of the images; slots count 64-bit.
__device__ __forceinline__ int64_t row_of(const Cache& c, int slot, int head) {
  const int page = (int)fdiv(c.by_page, (uint32_t)slot);
  return ((int64_t)page * c.heads + head) * c.page_size + (slot - page * c.page_size);
}

}  // namespace kv
}  // namespace fopt

struct fopt_rope {
  fopt::kv::Rope r;
};
