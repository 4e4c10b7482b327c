// kv4.cuh — the paged 4-bit KV cache as its kernels see it: pages of 16-token tiles, each tile K codes, V codes and the
// fp16 scale and bias of every 64 dims of each token's K and V (the byte order is in include/agxc.h).
#pragma once

#include "common.cuh"
#include "internal.h"

namespace agxc {

// a / b for 0 <= a, 0 < b, in 32 bits where that does
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((a | b) >> 32) ? a / b : static_cast<long long>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b));
}

struct Kv4 {
  uint8_t* data = nullptr;
  int pages = 0, kvh = 0, page = 0;  // page = tokens a page
};

template <int HD>
struct Kv4Tile {
  static constexpr int G = HD / 64;                  // groups of 64 dims
  static constexpr int kCodes = 16 * HD / 2;         // bytes of K (or V) codes
  static constexpr int kSb = 2 * kCodes;             // where the scale/bias entries start
  static constexpr int kEntry = 8 * G;               // bytes of a token's entry: [K, V][group]{scale, bias}
  static constexpr int kBytes = 2 * kCodes + 16 * kEntry;
  // byte of token t (0..15), group g, byte i (dims 2i, 2i + 1 of the group)
  __device__ static int k_at(int t, int g, int i) { return t * 32 * G + (i >> 3) * 8 * G + 8 * g + (i & 7); }
  __device__ static int v_at(int t, int g, int i) {
    return kCodes + (t >> 3) * 256 * G + (4 * (i >> 2) + ((t & 7) >> 1)) * 8 * G + (t & 1) * 4 * G + 4 * g + (i & 3);
  }
  __device__ static uint8_t* ptr(const Kv4& c, int page, int head, int tile) {
    return c.data + ((static_cast<size_t>(page) * c.kvh + head) * (c.page >> 4) + tile) * kBytes;
  }
};

inline int kv4_check(const agxc_kv4_cache* c, const char* who) {
  const std::string w(who);
  if (!c || !c->data_dev) return fail(AGXC_EINVAL, w + ": null cache");
  if (reinterpret_cast<uintptr_t>(c->data_dev) % 16) return fail(AGXC_EINVAL, w + ": the cache must be 16-byte aligned");
  if (c->head_dim != 64 && c->head_dim != 128) return fail(AGXC_EINVAL, w + ": head_dim 64 or 128");
  if (c->pages < 1 || c->kv_heads < 1) return fail(AGXC_EINVAL, w + ": at least one page and one KV head");
  if (c->page_size < 16 || c->page_size % 16) return fail(AGXC_EINVAL, w + ": page_size a positive multiple of 16");
  return 0;
}

inline Kv4 kv4_of(const agxc_kv4_cache& c) {
  Kv4 k;
  k.data = static_cast<uint8_t*>(c.data_dev);
  k.pages = c.pages;
  k.kvh = c.kv_heads;
  k.page = c.page_size;
  return k;
}

}  // namespace agxc
