// What the sources of the paged key/value cache share (kv_cache.hip, kv_pages.hip).
#pragma once

#include "common.h"

namespace mlcv {

// Slots of a cache, positions of a row, tokens of a write, query rows of a kv head: the last tile's or page's positions
// still are ints
constexpr int64_t KV_MOST = INT32_MAX - 255;
constexpr int KV_MAX_REQ = 4096;  // requests of a call that holds them all in LDS

__device__ __forceinline__ int clamp_i(int v, int lo, int hi) { return v < lo ? lo : v > hi ? hi : v; }

// Inclusive prefix sums of one value per thread over the workgroup (NT threads); `part` holds a sum per wave.
template <int NT>
__device__ __forceinline__ long long block_scan(long long v, long long* part) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const long long u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  if (lane == 63) part[w] = v;
  __syncthreads();
  long long before = 0;
#pragma unroll
  for (int i = 0; i < NT / 64 - 1; ++i) before += i < w ? part[i] : 0;
  __syncthreads();
  return v + before;
}

// Whether one of the first `outs` arrays of ints shares memory with any other
struct Ints {
  const void* p;
  int64_t n;
};
inline bool overlap(const Ints* a, int outs, int all) {
  for (int i = 0; i < outs; ++i)
    for (int j = i + 1; j < all; ++j) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(a[i].p), y = reinterpret_cast<uintptr_t>(a[j].p);
      if (a[i].n > 0 && a[j].n > 0 && x < y + 4 * a[j].n && y < x + 4 * a[i].n) return true;
    }
  return false;
}

inline bool kv_page_ok(int page) { return page == 16 || page == 32 || page == 64 || page == 128; }
inline bool kv_hd_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int log2_of(int page) { return page == 16 ? 4 : page == 32 ? 5 : page == 64 ? 6 : 7; }

}  // namespace mlcv
