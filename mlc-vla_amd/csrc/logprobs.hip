// Log probabilities from logits (mlcv_token_logprobs): of given tokens, of the best alternatives, and the entropy, in one
// pass over the row.  With m = max x, c = scale * log2(e) and y = c (x - m):
//   s = sum 2^y, u = sum -y 2^y      log p(t) = scale (x_t - m) - ln s      H = ln s + ln 2 * u / s
// m is the wave's running maximum, so that y is 0 for it and negative otherwise whatever its size: s is at least 1, both sums
// have terms of one sign and the entropy is never negative; the sums are rebased where the maximum grows.  float32 throughout.
// As one fused operation, c x - (c m), y would be an instruction less, but for the maximum the rounding of c m, which passes 128
// where c |m| passes 2^32: a wave that meets only logits masked with -1e10 would have an infinite sum.
//
// Alternatives are ranked by a 64-bit key, the logit's bits in an order of integers over the complement of its index:
// no two are equal, and equal logits rank by their index.  A wave holds its best 64 sorted, one per lane.  A logit that passes
// the threshold is inserted; where many do, as at the row's beginning, they are sorted and merged by the bitonic network.  The
// threshold is the wave's k-th best, or the least that the waves of the row know to be below k.
//
// Bound by the read of the logits where there are many rows (1001 of 257152 in bf16: 95.3 us, 5.4 TB/s), with 9.5 vector
// instructions per logit and lane beside it; for few rows by the latency of selecting (16 rows: 8.6 us in 512 workgroups and
// 3.8 in the join; without alternatives 7.9 in all).
#include "kernels.h"
#include "mlcvla.h"
#include "rows.h"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace mlcv {

namespace {

typedef unsigned long long u64;

constexpr int LP_W = 4;         // waves per workgroup
constexpr int LP_U = 4;         // chunks of 8 logits in flight per lane
constexpr int LP_GROUP = 64 * LP_W * LP_U;
constexpr int LP_JW = 8;        // waves per workgroup of the join
constexpr int LP_TOP = 64;      // most alternatives: one per lane
constexpr float LN2 = 0.6931471805599453f;

struct LpArgs {
  const void* x;
  int64_t stride;  // elements between rows
  const int32_t* tokens;
  float *lp, *entropy, *top_lp;
  int32_t* top_ids;
  float* stats;  // of the splits: (m, s, u, -) [rows][S]
  u64* keys;     // and their best [rows][S][k]
  int32_t rows, vocab, given, k, S, per;  // per: chunks of 8 logits per split
  float scale, c;                         // c = scale * log2(e)
};

template <int TYPE>
struct LpType;
template <>
struct LpType<MLCV_DTYPE_F16> {
  typedef _Float16 T;
};
template <>
struct LpType<MLCV_DTYPE_BF16> {
  typedef __bf16 T;
};
template <>
struct LpType<MLCV_DTYPE_F32> {
  typedef float T;
};

__device__ __forceinline__ u64 key_of(float x, uint32_t i) {
  const uint32_t b = __float_as_uint(x + 0.0f);  // -0 ranks as 0
  return (u64)(b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u)) << 32 | ~i;
}
__device__ __forceinline__ float value_of(u64 key) {
  const uint32_t o = (uint32_t)(key >> 32);
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ u64 lane_of(u64 v, int lane) {
  return (u64)(uint32_t)__builtin_amdgcn_readlane((int)(v >> 32), lane) << 32 |
         (uint32_t)__builtin_amdgcn_readlane((int)v, lane);
}
// v of lane ^ M, M < 16, within the registers: the crossbar of LDS takes four times as long
template <int M>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  auto dpp = [](uint32_t x, auto ctrl) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, decltype(ctrl)::value, 0xf, 0xf, true);
  };
  if constexpr (M == 1) return dpp(v, std::integral_constant<int, 0xb1>());   // quads [1 0 3 2]
  if constexpr (M == 2) return dpp(v, std::integral_constant<int, 0x4e>());   // quads [2 3 0 1]
  if constexpr (M == 4) return dpp(dpp(v, std::integral_constant<int, 0x1b>()), std::integral_constant<int, 0x141>());  // 3 ^ 7
  if constexpr (M == 8) return dpp(v, std::integral_constant<int, 0x128>());  // rows of 16 turned by 8
}
// f over all lanes, in every lane
template <class F>
__device__ __forceinline__ float wave_all(float v, F f) {
  auto dpp = [](float x, auto ctrl) {
    return __uint_as_float((uint32_t)__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v = f(v, dpp(v, std::integral_constant<int, 0xb1>()));   // lane ^ 1
  v = f(v, dpp(v, std::integral_constant<int, 0x4e>()));   // ^ 2
  v = f(v, dpp(v, std::integral_constant<int, 0x141>()));  // the other four of eight
  v = f(v, dpp(v, std::integral_constant<int, 0x140>()));  // the other eight of sixteen
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = f(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return f(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
__device__ __forceinline__ float all_max(float v) {
  return wave_all(v, [](float x, float y) { return fmaxf(x, y); });
}
__device__ __forceinline__ float all_sum(float v) {
  return wave_all(v, [](float x, float y) { return x + y; });
}

// one step of the bitonic network over lanes S apart
template <int S>
__device__ __forceinline__ u64 exchange(u64 v, bool larger) {
  const uint32_t l = (uint32_t)v, h = (uint32_t)(v >> 32);
  u64 a = v, b;
  if constexpr (S < 16) {
    b = (u64)lane_xor<S>(h) << 32 | lane_xor<S>(l);
  } else {  // both lanes of a pair receive the lower lane's and the upper's
    const auto x = S == 16 ? __builtin_amdgcn_permlane16_swap(l, l, false, false) : __builtin_amdgcn_permlane32_swap(l, l, false, false);
    const auto y = S == 16 ? __builtin_amdgcn_permlane16_swap(h, h, false, false) : __builtin_amdgcn_permlane32_swap(h, h, false, false);
    a = (u64)y[0] << 32 | x[0];
    b = (u64)y[1] << 32 | x[1];
  }
  return (a > b) == larger ? a : b;
}
// The same for values alone: a third of the instructions.  Falling.
template <int S>
__device__ __forceinline__ float exchange(float v, bool larger) {
  const uint32_t b = __float_as_uint(v);
  float x = v, y;
  if constexpr (S < 16) {
    y = __uint_as_float(lane_xor<S>(b));
  } else {
    const auto z = S == 16 ? __builtin_amdgcn_permlane16_swap(b, b, false, false) : __builtin_amdgcn_permlane32_swap(b, b, false, false);
    x = __uint_as_float(z[0]);
    y = __uint_as_float(z[1]);
  }
  return larger ? fmaxf(x, y) : fminf(x, y);
}

// lanes SIZE / 2, SIZE / 4, .. 1 apart: each run of SIZE lanes, first falling then rising (or the reverse), becomes sorted
template <int SIZE, class V>
__device__ __forceinline__ V settle(V v, bool falling, int lane) {
  if constexpr (SIZE >= 64) v = exchange<32>(v, ((lane & 32) == 0) == falling);
  if constexpr (SIZE >= 32) v = exchange<16>(v, ((lane & 16) == 0) == falling);
  if constexpr (SIZE >= 16) v = exchange<8>(v, ((lane & 8) == 0) == falling);
  if constexpr (SIZE >= 8) v = exchange<4>(v, ((lane & 4) == 0) == falling);
  if constexpr (SIZE >= 4) v = exchange<2>(v, ((lane & 2) == 0) == falling);
  return exchange<1>(v, ((lane & 1) == 0) == falling);
}
template <class V>
__device__ __forceinline__ V sort64(V v, bool falling, int lane) {
  v = settle<2>(v, (lane & 2) == 0, lane);
  v = settle<4>(v, (lane & 4) == 0, lane);
  v = settle<8>(v, (lane & 8) == 0, lane);
  v = settle<16>(v, (lane & 16) == 0, lane);
  v = settle<32>(v, ((lane & 32) == 0) == falling, lane);
  return settle<64>(v, falling, lane);
}
// the best 64 of a falling and a rising list, falling
__device__ __forceinline__ u64 merge64(u64 a, u64 b, int lane) { return settle<64>(a > b ? a : b, true, lane); }

// Sums relative to a maximum
struct Sums {
  float m, s, u;
};
// What is taken off a logit: m, but 0 where there is none yet, as -inf less itself is no number
__device__ __forceinline__ float base_of(float m) { return m == -INFINITY ? 0.f : m; }
// From the own maximum to m, which is not below it
__device__ __forceinline__ void rebase(Sums& v, float m, float c) {
  const float y = v.m == -INFINITY ? -INFINITY : (v.m - m) * c, f = __builtin_amdgcn_exp2f(y);
  v.u = f * (v.u - v.s * fmaxf(y, -1000.f));  // f = 0 below
  v.s *= f;
  v.m = m;
}

// the largest float32 below a finite one; -inf stays
__device__ __forceinline__ float below(float x) {
  const uint32_t b = __float_as_uint(x);
  return x == -INFINITY ? x : x == 0.f ? __uint_as_float(0x80000001u) : __uint_as_float(x > 0.f ? b - 1 : b + 1);
}

template <bool TOP, int WPR>
struct Scan {
  Sums v;        // the maximum is the wave's, the sums each lane's
  float base;    // base_of it
  float c, thr;  // what a logit has to pass to matter beyond the sums
  u64 list;
  u64* buf;            // 576 keys of the wave
  volatile float* kw;  // of each wave of the row, its (k / WPR)-th best (rounded up) so far
  int k, w, lane;

  __device__ __forceinline__ void init(float c_, int k_, u64* buf_, volatile float* kw_, int w_, int lane_) {
    c = c_;
    k = k_;
    buf = buf_;
    kw = kw_;
    w = w_;
    lane = lane_;
    v.m = thr = -INFINITY;
    // Values that the compiler does not know: where it knows the -inf, it turns x > -inf into "x differs from -inf", and the
    // ballot of that into an instruction which is true for NaN.
    asm volatile("" : "+v"(v.m), "+v"(thr));
    v.s = v.u = 0.f;
    base = base_of(v.m);
    list = 0;
  }
  __device__ __forceinline__ void raise(float big) {
    if (!__any(big > v.m)) return;
    const float wm = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(all_max(big))));
    base = base_of(wm);
    rebase(v, wm, c);
  }
  // one key of the wave's into the list
  __device__ __forceinline__ void insert(u64 key) {
    const int at = __popcll(__ballot(list > key));
    const uint32_t l = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)list, 0x138, 0xf, 0xf, true);  // of the lane before
    const uint32_t h = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(list >> 32), 0x138, 0xf, 0xf, true);
    list = lane < at ? list : lane == at ? key : (u64)h << 32 | l;
  }
  // the buffer's keys from the last n <= 64 of its first `pend` on into the list
  __device__ __forceinline__ void take(int n, int pend) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    list = merge64(list, sort64(lane < n ? buf[pend - n + lane] : 0, false, lane), lane);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
  // What the wave now knows.  Its own k-th best: later logits have to be larger, as equal ones rank behind.  And where
  // every wave of the row has ceil(k / WPR) of at least some value, k have: equal ones may still rank before those.
  __device__ __forceinline__ void publish() {
    const u64 kth = lane_of(list, k - 1);
    if (kth) thr = fmaxf(thr, value_of(kth));
    if constexpr (WPR > 1) {
      const u64 mine = lane_of(list, (k + WPR - 1) / WPR - 1);
      if (mine && lane == 0) kw[w] = value_of(mine);
    }
  }
  __device__ __forceinline__ void listen() {
    if constexpr (WPR > 1) {
      float low = kw[0];
#pragma unroll
      for (int i = 1; i < WPR; ++i) low = fminf(low, kw[i]);
      thr = fmaxf(thr, below(__uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(low)))));
    }
  }
  // Logits x[n] of indices i0[n] .. + 7, the largest of each big[n], of all `top` (NaN where one is among them); some lane's
  // passes thr or is NaN.
  template <int U>
  __device__ __forceinline__ void look(const float (&x)[U][8], const int (&i0)[U], float (&big)[U], float top) {
    if (__any(top != top)) {  // the largest of the others
      top = -INFINITY;
#pragma unroll
      for (int n = 0; n < U; ++n) {
        big[n] = -INFINITY;
#pragma unroll
        for (int e = 0; e < 8; ++e) big[n] = x[n][e] > big[n] ? x[n][e] : big[n];
        top = fmaxf(top, big[n]);
      }
    }
    raise(top);
    if constexpr (!TOP) {
      thr = v.m;
      return;
    }
    listen();
    const u64 lanes = __ballot(top > thr);
    if (!lanes) return;
    float bar = thr;  // where many lanes have something, the k-th of their largest bounds what can matter
    if (__popcll(lanes) > 16)
      bar = fmaxf(bar, below(__uint_as_float(__builtin_amdgcn_readlane(
                           __float_as_uint(sort64(fmaxf(top, -INFINITY), true, lane)), k - 1))));
#pragma unroll
    for (int n = 0; n < U; ++n) {
      // All of a chunk is compared with one threshold: equal logits of it may have lower indices than those that are
      // taken first.
      const float t0 = fmaxf(bar, thr);
      if (!__any(big[n] > t0)) continue;
      u64 b[8];
      int all = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        b[e] = __ballot(x[n][e] > t0);
        all += __popcll(b[e]);
      }
      if (all <= 12) {  // one by one
#pragma unroll
        for (int e = 0; e < 8; ++e)
          for (; b[e]; b[e] &= b[e] - 1) {
            const int l = __builtin_ctzll(b[e]);
            const float y = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x[n][e]), l));
            insert(key_of(y, (uint32_t)(__builtin_amdgcn_readlane(i0[n], l) + e)));
          }
      } else {  // 64 at a time
        int pend = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          if ((b[e] >> lane) & 1)
            buf[pend + __builtin_amdgcn_mbcnt_hi((uint32_t)(b[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b[e], 0))] =
                key_of(x[n][e], i0[n] + e);
          pend += __popcll(b[e]);
        }
        for (; pend > 0; pend -= 64) take(min(pend, 64), pend);
      }
      publish();
    }
  }
  // Before the first look: the waves of a row tell one another the ceil(k / WPR)-th of their lanes' largest.
  __device__ __forceinline__ void meet(float top) {
    const float v = sort64(fmaxf(top, -INFINITY), true, lane);
    if (lane == (k + WPR - 1) / WPR - 1) kw[w] = v;
    __syncthreads();
  }
  template <int U>
  __device__ __forceinline__ void add(const float (&x)[U][8], const int (&i0)[U], bool begin) {
    // The maximum that keeps a NaN.  fmaxf of a signalling one and a number may be NaN too, so a number next to it would be
    // lost; it is sorted out where there is one, and no logit has to be made quiet first, an instruction each (1001 rows of
    // 257152, the same logits again, 97.6 -> 92.1 us).
    auto max3 = [](float a, float b, float c) { return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c); };
    float big[U], top = -INFINITY;
#pragma unroll
    for (int n = 0; n < U; ++n) {
      const float* y = x[n];
      big[n] = max3(max3(y[0], y[1], y[2]), max3(y[3], y[4], y[5]), __builtin_elementwise_maximum(y[6], y[7]));
      top = __builtin_elementwise_maximum(top, big[n]);
    }
    if constexpr (TOP && WPR > 1)
      if (begin) meet(top);
    if (__any(!(top <= thr))) look<U>(x, i0, big, top);
#pragma unroll
    for (int n = 0; n < U; ++n) {
      float s[8], u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y = (x[n][e] - base) * c;
        s[e] = __builtin_amdgcn_exp2f(y);
        u[e] = fmaxf(y, -1000.f);  // a masked logit's y is -inf, its weight 0
      }
      v.s += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
#pragma unroll
      for (int e = 0; e < 8; ++e) v.u = __builtin_fmaf(-u[e], s[e], v.u);
    }
  }
  __device__ __forceinline__ void end() {
    v.s = all_sum(v.s);
    v.u = all_sum(v.u);
  }
};

// The logit of a row's given token number i, and whether there is one
template <int TYPE>
__device__ __forceinline__ float given_logit(const LpArgs& a, int row, int i, bool& there) {
  typedef typename LpType<TYPE>::T T;
  const int t = i < a.given ? a.tokens[(int64_t)row * a.given + i] : -1;
  there = t >= 0 && t < a.vocab;
  return there ? (float)load_global(static_cast<const T*>(a.x) + (int64_t)row * a.stride + t) : 0.f;
}

// The row's results by one wave, from its sums and its sorted best; z0, there: given_logit of token number `lane`.
template <int TYPE>
__device__ __forceinline__ void finish(const LpArgs& a, int row, Sums v, u64 list, int lane, float z0, bool there) {
  typedef typename LpType<TYPE>::T T;
  const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
  const float ls = logf(v.s);
  // a row whose mask leaves nothing: s = 0.  Halves, as the difference of the largest logits of either sign is past float32.
  auto lp = [&](float z) { return v.s == 0.f ? -INFINITY : (0.5f * z - 0.5f * v.m) * (2.f * a.scale) - ls; };
  if (lane == 0 && a.entropy) a.entropy[row] = v.s == 0.f ? 0.f : ls + LN2 * (v.u / v.s);
  for (int i = lane; i < a.given; i += 64) {
    if (i != lane) z0 = given_logit<TYPE>(a, row, i, there);
    a.lp[(int64_t)row * a.given + i] = there ? lp(z0) : 0.f;
  }
  if (!a.k) return;
  int32_t* ids = a.top_ids + (int64_t)row * a.k;
  float* lps = a.top_lp + (int64_t)row * a.k;
  if (lane < a.k && list) {
    ids[lane] = (int32_t)~(uint32_t)list;
    lps[lane] = lp(value_of(list));
  }
  // fewer unmasked logits than alternatives: the masked ones by their index, then what is no number
  int have = __popcll(__ballot(lane < a.k && list));
  for (int nan = 0; nan < 2 && have < a.k; ++nan)
    for (int64_t i0 = 0; i0 < a.vocab && have < a.k; i0 += 64) {
      const int64_t i = i0 + lane;
      const float z = i < a.vocab ? (float)load_global(x + i) : 0.f;
      const bool ok = nan ? z != z : z == -INFINITY;
      const u64 b = __ballot(ok);
      const int at =
          have + (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0));
      if (ok && at < a.k) {
        ids[at] = (int32_t)i;
        lps[at] = lp(z);
      }
      have += __popcll(b);
    }
}

// WPR waves share a row's split.  The row is cut into chunks of 8 logits from the 16-byte boundary at or before its first
// one; a wave's chunks follow one another in ascending order.
template <int TYPE, bool TOP, int WPR>
__global__ __launch_bounds__(64 * LP_W) void logprobs_kernel(const LpArgs a) {
  typedef typename LpType<TYPE>::T T;
  constexpr int V = sizeof(T) / 2, U = LP_U;  // 16-byte loads of a chunk, chunks in flight
  __shared__ u64 buf[LP_W][TOP ? 63 + 8 * 64 + 1 : 1];
  __shared__ Sums part[LP_W];
  __shared__ float kw[LP_W];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = WPR == 1 ? blockIdx.x * LP_W + w : blockIdx.x / a.S;
  const int split = WPR == 1 ? 0 : blockIdx.x % a.S;
  if (WPR == 1 && row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int chunks = (int)(((int64_t)a.vocab + off + 7) >> 3);
  const int last = (int)min((int64_t)chunks, (int64_t)(split + 1) * a.per);
  const int first = (int)((int64_t)split * a.per) + (WPR == 1 ? 0 : w) * 64;
  Scan<TOP, WPR> scan;
  scan.init(a.c, a.k, buf[w], kw, w, lane);
  const int whole = (int)(((int64_t)a.vocab + off) >> 3);  // chunks from here on end behind the row
  // a wave without chunks takes one round too, as the waves meet in it
  for (int at = first; at == first || at < last; at += 64 * WPR * U) {
    float z[U][8];
    int at0[U];
#pragma unroll
    for (int n = 0; n < U; ++n) at0[n] = (at + 64 * WPR * n + lane) * 8 - off;
    if (at + 64 * WPR * (U - 1) + 63 < min(last, whole) && (at > 0 || !off)) {
      u4 raw[U][V];
#pragma unroll
      for (int n = 0; n < U; ++n)
#pragma unroll
        for (int i = 0; i < V; ++i) raw[n][i] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(x + at0[n]) + i);
#pragma unroll
      for (int n = 0; n < U; ++n)
#pragma unroll
        for (int e = 0; e < 8; ++e) z[n][e] = (float)reinterpret_cast<const T*>(raw[n])[e];
    } else {  // the row's ends
#pragma unroll
      for (int n = 0; n < U; ++n) {
        const int ch = at + 64 * WPR * n + lane;
        u4 raw[V];
        if (ch < last && ch < whole && at0[n] >= 0) {
#pragma unroll
          for (int i = 0; i < V; ++i) raw[i] = load_global(reinterpret_cast<const u4*>(x + at0[n]) + i);
#pragma unroll
          for (int e = 0; e < 8; ++e) z[n][e] = (float)reinterpret_cast<const T*>(raw)[e];
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            z[n][e] = ch < last && at0[n] + e >= 0 && at0[n] + e < a.vocab ? (float)load_global(x + at0[n] + e) : -INFINITY;
        }
      }
    }
    scan.template add<U>(z, at0, at == first);
  }
  scan.end();
  if constexpr (WPR > 1) {
    if constexpr (TOP) buf[w][lane] = scan.list;
    if (lane == 0) part[w] = scan.v;
    __syncthreads();
    if (w > 0) return;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < LP_W; ++i) m = fmaxf(m, part[i].m);
    Sums v{m, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < LP_W; ++i) {
      Sums q = part[i];
      rebase(q, m, a.c);
      v.s += q.s;
      v.u += q.u;
    }
    scan.v = v;
    if constexpr (TOP)
#pragma unroll
      for (int i = 1; i < LP_W; ++i) scan.list = merge64(scan.list, buf[i][63 - lane], lane);
    if (a.S > 1) {
      const int64_t o = (int64_t)row * a.S + split;
      if (lane == 0) *reinterpret_cast<f4*>(a.stats + 4 * o) = (f4){v.m, v.s, v.u, 0.f};
      if (TOP && lane < a.k) a.keys[o * a.k + lane] = scan.list;
      return;
    }
  }
  bool there;
  const float z0 = given_logit<TYPE>(a, row, lane, there);
  finish<TYPE>(a, row, scan.v, scan.list, lane, z0, there);
}

// The splits of a row: a workgroup per row, its waves take splits in turn and meet in pairs.
template <int TYPE>
__global__ __launch_bounds__(64 * LP_JW) void logprobs_join_kernel(const LpArgs a) {
  __shared__ u64 lists[LP_JW][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x;
  const int64_t o = (int64_t)row * a.S;
  u64 list = 0;
  // the sums and the given tokens are on their way while the lists are merged
  f4 p = {-INFINITY, 0.f, 0.f, 0.f};
  float z0 = 0.f;
  bool there = false;
  if (w == 0) {
    if (lane < a.S) p = load_global(reinterpret_cast<const f4*>(a.stats) + o + lane);
    z0 = given_logit<TYPE>(a, row, lane, there);
  }
  if (a.k) {
    constexpr int Q = 4;  // lists on their way at once
    for (int s0 = w; s0 < a.S; s0 += Q * LP_JW) {
      u64 key[Q];
#pragma unroll
      for (int q = 0; q < Q; ++q) {
        const int s = s0 + q * LP_JW;
        // the first as it is, the others from their end
        const int at = s == w ? lane : 63 - lane;
        key[q] = s < a.S && at < a.k ? load_global(a.keys + (o + s) * a.k + at) : 0;
      }
#pragma unroll
      for (int q = 0; q < Q; ++q)
        if (s0 + q * LP_JW < a.S) list = s0 + q * LP_JW == w ? key[q] : merge64(list, key[q], lane);
    }
    lists[w][lane] = list;
#pragma unroll
    for (int h = LP_JW / 2; h > 0; h >>= 1) {
      __syncthreads();
      if (w < h) lists[w][lane] = list = merge64(list, lists[w + h][63 - lane], lane);
    }
  }
  if (w > 0) return;
  Sums v{-INFINITY, 0.f, 0.f};
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    if (s0 > 0) p = s0 + lane < a.S ? load_global(reinterpret_cast<const f4*>(a.stats) + o + s0 + lane) : (f4){-INFINITY, 0.f, 0.f, 0.f};
    const float m = fmaxf(v.m, all_max(p[0]));
    Sums q{p[0], p[1], p[2]};
    rebase(q, m, a.c);
    rebase(v, m, a.c);
    v.s += all_sum(q.s);
    v.u += all_sum(q.u);
  }
  finish<TYPE>(a, row, v, list, lane, z0, there);
}

// How a call is cut: waves of a row (1 or 4), splits of it and their chunks
struct LpPlan {
  int wpr, S, per;
  size_t bytes;
};
LpPlan lp_plan(int rows, int vocab, int k) {
  LpPlan p;
  // A wave for each row where there are enough of them, as it selects once and not four times: 4000 rows of 4096, 8192 and
  // 32000 logits take 19.4, 28.4 and 68.0 us, with four waves 28.1, 29.3 and 72.1; 4000 of 257152 336 and 331 (without
  // alternatives 329 and 313); 2000 of 8192 21.1 and 18.8, 1000 of 4096 11.6 and 11.5, 64 of 4096 10.8 and 7.4.  Up to 2048 logits
  // are one round of one wave.
  p.wpr = vocab <= 2048 || rows >= (vocab <= 4096 ? 1000 : 4000) ? 1 : LP_W;
  const int chunks = (int)(((int64_t)vocab + 7 + 7) >> 3);
  // Splits that make about 1200 workgroups, of a round of loads (8192 logits) at least, and none of less than three rounds,
  // where the join's launch costs more.  257152 logits, 20 alternatives (5 from 300 rows on): 16 rows 13.7 us with 32
  // splits, 15.3 with 16, 58.5 with one; 64 rows 22.8, 21.7 and 60.8; 300 rows 42.4 with 4, 44.3 with 8, 48.4 with 2, 60.3 with
  // one; 1001 rows 96.8 with one, 101.9 with 2 (20 calls on end, without the host).  32000 logits: 64 rows 12.1 with 4, 16.5
  // with one; 16384: 16 rows 13.9 with 2, 10.7 with one.
  const int rounds = (int)(((int64_t)vocab + 8 * LP_GROUP - 1) / (8 * LP_GROUP));
  int S = p.wpr == 1 || rounds < 3 ? 1 : std::max(1, std::min((int)((1200 + (int64_t)rows / 2) / rows), rounds));
  p.per = (chunks + S - 1) / S;
  if (S > 1) p.per = (p.per + LP_GROUP - 1) / LP_GROUP * LP_GROUP;  // only the last split ends within a round of loads
  p.S = (chunks + p.per - 1) / p.per;
  p.bytes = p.S > 1 ? (size_t)rows * p.S * (16 + 8 * (size_t)k) : 0;
  return p;
}

template <int TYPE, bool TOP>
int lp_launch(const LpArgs& a, const LpPlan& p, hipStream_t st) {
  if (p.wpr == 1) {
    logprobs_kernel<TYPE, TOP, 1><<<(unsigned)(((int64_t)a.rows + LP_W - 1) / LP_W), 64 * LP_W, 0, st>>>(a);
  } else {
    logprobs_kernel<TYPE, TOP, LP_W><<<(unsigned)((int64_t)a.rows * p.S), 64 * LP_W, 0, st>>>(a);
  }
  MLCV_HIP(hipGetLastError());
  if (p.S > 1) {
    logprobs_join_kernel<TYPE><<<(unsigned)a.rows, 64 * LP_JW, 0, st>>>(a);
    MLCV_HIP(hipGetLastError());
  }
  return 0;
}

int lp_sizes_ok(int32_t rows, int32_t vocab, int32_t top) {
  MLCV_REQUIRE(rows >= 0 && vocab > 0, "bad size");
  MLCV_REQUIRE(vocab <= INT32_MAX - (1 << 20), "vocab is too large");
  MLCV_REQUIRE(top >= 0 && top <= LP_TOP && top <= vocab, "top must be at most 64 and at most vocab");
  // a launch holds less than 2^32 threads
  MLCV_REQUIRE(rows <= (int)(UINT32_MAX / (64 * LP_JW)), "too many rows");
  return 0;
}

}  // namespace
}  // namespace mlcv

using namespace mlcv;

extern "C" {

int mlcv_token_logprobs_workspace(int32_t rows, int32_t vocab, int32_t top, size_t* bytes) {
  MLCV_REQUIRE(bytes, "null pointer");
  MLCV_TRY(lp_sizes_ok(rows, vocab, top));
  *bytes = rows ? lp_plan(rows, vocab, top).bytes : 0;
  return 0;
}

int mlcv_token_logprobs(const void* logits, int32_t dtype, int64_t stride, int32_t rows, int32_t vocab, float scale,
                        const int32_t* tokens, int32_t given, float* logprobs, float* entropy, int32_t top,
                        int32_t* top_ids, float* top_logprobs, void* workspace, size_t workspace_bytes, void* stream) {
  MLCV_REQUIRE(dtype == MLCV_DTYPE_F16 || dtype == MLCV_DTYPE_BF16 || dtype == MLCV_DTYPE_F32,
               "logits are float16, bfloat16 or float32");
  MLCV_TRY(lp_sizes_ok(rows, vocab, top));
  MLCV_REQUIRE(given >= 0, "bad size");
  MLCV_REQUIRE(scale >= 1e-6f && scale <= 1e6f, "scale must be between 1e-6 and 1e6");
  if (rows == 0) return 0;
  MLCV_REQUIRE(logits && (given == 0 || (tokens && logprobs)) && (top == 0 || (top_ids && top_logprobs)),
               "null pointer");
  MLCV_REQUIRE(reinterpret_cast<uintptr_t>(logits) % (dtype == MLCV_DTYPE_F32 ? 4 : 2) == 0, "logits are not aligned");
  const LpPlan p = lp_plan(rows, vocab, top);
  MLCV_REQUIRE(p.bytes == 0 || (workspace && (reinterpret_cast<uintptr_t>(workspace) & 15) == 0 &&
                                workspace_bytes >= p.bytes),
               "workspace missing, not 16-byte aligned or too small");
  const Rows::Int size = dtype == MLCV_DTYPE_F32 ? 4 : 2;
  const int64_t ints = 4 * (int64_t)rows;
  const Rows arrays[] = {Rows(given ? logprobs : nullptr, ints * given), Rows(entropy, ints), Rows(top ? top_ids : nullptr, ints * top),
                         Rows(top ? top_logprobs : nullptr, ints * top), Rows(workspace, (int64_t)p.bytes),
                         Rows(logits, rows, stride * size, 1, 0, vocab * size), Rows(given ? tokens : nullptr, ints * given)};
  MLCV_REQUIRE(!any_meet(arrays, 5, 7), "outputs or workspace overlap the inputs or one another");
  LpArgs a{};
  a.x = logits;
  a.stride = stride;
  a.tokens = tokens;
  a.lp = logprobs;
  a.entropy = entropy;
  a.top_lp = top_logprobs;
  a.top_ids = top_ids;
  a.stats = static_cast<float*>(workspace);
  a.keys = workspace ? reinterpret_cast<u64*>(a.stats + 4 * (size_t)rows * p.S) : nullptr;
  a.rows = rows;
  a.vocab = vocab;
  a.given = given;
  a.k = top;
  a.S = p.S;
  a.per = p.per;
  a.scale = scale;
  a.c = scale * 1.4426950408889634f;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (dtype == MLCV_DTYPE_F16)
    return top ? lp_launch<MLCV_DTYPE_F16, true>(a, p, st) : lp_launch<MLCV_DTYPE_F16, false>(a, p, st);
  if (dtype == MLCV_DTYPE_BF16)
    return top ? lp_launch<MLCV_DTYPE_BF16, true>(a, p, st) : lp_launch<MLCV_DTYPE_BF16, false>(a, p, st);
  return top ? lp_launch<MLCV_DTYPE_F32, true>(a, p, st) : lp_launch<MLCV_DTYPE_F32, false>(a, p, st);
}

}  // extern "C"
