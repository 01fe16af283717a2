// Log probabilities from logits (mlcv_token_logprobs): of given tokens, of the best alternatives, and the entropy, in one
// pass over the row.  With m = max x, c = scale * log2(e) and y = c (x - m):
//   s = sum 2^y, u = sum -y 2^y      log p(t) = scale (x_t - m) - ln s      H = ln s + ln 2 * u / s
// m is the wave's running maximum, so that no y is positive, both sums have terms of one sign and the entropy of a
// row that is almost certain keeps its digits; the sums are rebased where the maximum grows.  float32 throughout.
//
// Alternatives are ranked by a 64-bit key, the logit's bits in an order of integers over the complement of its index:
// no two are equal, and equal logits rank by their index.  A wave holds its best 64 sorted, one per lane, and
// appends what passes the k-th of them to a buffer of its own; 64 at a time are sorted and merged by the bitonic
// network.  Of n logits in random order about k ln(n / k) pass.
#include "kernels.h"
#include "mlcvla.h"

#include <algorithm>
#include <cmath>

namespace mlcv {

namespace {

typedef unsigned long long u64;

constexpr int LP_W = 4;         // waves per workgroup
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
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
  return v;
}

// one step of the bitonic network: lanes `stride` apart, the larger key to the lower lane where down
__device__ __forceinline__ u64 exchange(u64 v, int stride, bool down, int lane) {
  const u64 o = __shfl_xor(v, stride);
  return (((lane & stride) == 0) == down) == (v > o) ? v : o;
}
__device__ __forceinline__ u64 sort64(u64 v, int lane) {
#pragma unroll
  for (int size = 2; size <= 64; size <<= 1)
#pragma unroll
    for (int s = size >> 1; s > 0; s >>= 1) v = exchange(v, s, (lane & size) == 0, lane);
  return v;
}
// the best 64 of two sorted lists, sorted
__device__ __forceinline__ u64 merge64(u64 a, u64 b, int lane) {
  const u64 o = __shfl(b, 63 - lane);
  a = a > o ? a : o;
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) a = exchange(a, s, true, lane);
  return a;
}

// Sums relative to a maximum.  y = x * ce - mc in one fused operation: ce is c, but 2^-20 where c |m| would leave float32's
// range; logits of that size are equal or 2^70 apart.
struct Sums {
  float m, s, u;
};
struct Base {
  float ce, mc;
};
__device__ __forceinline__ Base base_of(float m, float c) {
#pragma clang fp contract(off)  // mc is the rounded product wherever it is used
  Base b;
  b.ce = fabsf(m) * c < 0x1p120f ? c : 0x1p-20f;
  b.mc = m == -INFINITY ? 0.f : m * b.ce;
  return b;
}
// From the own maximum to m, whose base is b.  The sums are relative to their rounded mc, and the two mc's difference is what
// counts.
__device__ __forceinline__ void rebase(Sums& v, float m, Base b, float c) {
#pragma clang fp contract(off)
  const float y = v.m == -INFINITY ? -INFINITY : base_of(v.m, c).mc - b.mc, f = __builtin_amdgcn_exp2f(y);
  v.u = f * (v.u - v.s * fmaxf(y, -1000.f));  // f = 0 below
  v.s *= f;
  v.m = m;
}

template <bool TOP>
struct Scan {
  Sums v;       // the maximum is the wave's, the sums each lane's
  Base base;
  float c, thr;  // what a logit has to pass to matter beyond the sums
  u64 list;
  u64* buf;
  int k, pend, lane;

  __device__ __forceinline__ void init(float c_, int k_, u64* buf_, int lane_) {
    c = c_;
    k = k_;
    buf = buf_;
    lane = lane_;
    v.m = thr = -INFINITY;
    v.s = v.u = 0.f;
    base = base_of(v.m, c);
    list = 0;
    pend = 0;
  }
  // `n` <= 64 of the buffer's keys into the list
  __device__ __forceinline__ void take(int n) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    list = merge64(list, sort64(lane < n ? buf[lane] : 0, lane), lane);
    const u64 rest = lane < pend - n ? buf[n + lane] : 0;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (lane < pend - n) buf[lane] = rest;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    pend -= n;
  }
  // logits x of indices i0 .. + 7; `big` the largest; some lane's passes thr
  __device__ __forceinline__ void look(const float (&x)[8], int i0, float big) {
    const float wm = __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(wave_max(big))));
    if (wm > v.m) {
      base = base_of(wm, c);
      rebase(v, wm, base, c);
    }
    if constexpr (!TOP) {
      thr = v.m;
      return;
    }
    // All of this block is compared with the threshold from before it: equal logits of it may have lower indices than
    // those that are taken first.
    const float t0 = thr;
    int all = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) all += __popcll(__ballot(x[e] > t0));
    u64 low = 0;
    if (all > 64) {  // the k-th of the lanes' best bounds what can matter
      int at = 0;
#pragma unroll
      for (int e = 7; e >= 0; --e) at = x[e] == big ? e : at;
      low = lane_of(sort64(big > t0 ? key_of(big, i0 + at) : 0, lane), k - 1);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const u64 key = key_of(x[e], i0 + e);
      const bool ok = x[e] > t0 && key >= low;
      const u64 b = __ballot(ok);
      if (!b) continue;
      if (ok) buf[pend + __builtin_amdgcn_mbcnt_hi((uint32_t)(b >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)b, 0))] = key;
      pend += __popcll(b);
      if (pend >= 64) take(64);
    }
    const u64 kth = lane_of(list, k - 1), bound = kth > low ? kth : low;
    if (bound) thr = fmaxf(thr, value_of(bound));
  }
  __device__ __forceinline__ void add(const float (&x)[8], int i0) {
    const float big = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])), fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
    if (__any(big > thr)) look(x, i0, big);
    float s[8], u[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float y = __builtin_fmaf(x[e], base.ce, -base.mc);
      s[e] = __builtin_amdgcn_exp2f(y);
      u[e] = fmaxf(y, -1000.f);  // a masked logit's y is -inf, its weight 0
    }
    v.s += ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
#pragma unroll
    for (int e = 0; e < 8; ++e) v.u = __builtin_fmaf(-u[e], s[e], v.u);
  }
  __device__ __forceinline__ void end() {
    if constexpr (TOP)
      if (pend) take(pend);
    v.s = wave_sum(v.s);
    v.u = wave_sum(v.u);
  }
};

// The row's results by one wave, from its sums and its sorted best.
template <int TYPE>
__device__ __forceinline__ void finish(const LpArgs& a, int row, Sums v, u64 list, int lane) {
  typedef typename LpType<TYPE>::T T;
  const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
  // the sums are relative to the rounded mc; its distance from m c counts where the two meet
  const Base b0 = base_of(v.m, a.c);
  const float le = logf(v.s), ls = le - (fabsf(v.m) < INFINITY ? LN2 * __builtin_fmaf(v.m, b0.ce, -b0.mc) : 0.f);
  // a row whose mask leaves nothing: s = 0
  auto lp = [&](float z) { return v.s == 0.f ? -INFINITY : (z - v.m) * a.scale - ls; };
  if (lane == 0 && a.entropy) a.entropy[row] = v.s == 0.f ? 0.f : le + LN2 * (v.u / v.s);
  for (int i = lane; i < a.given; i += 64) {
    const int64_t at = (int64_t)row * a.given + i;
    const int t = a.tokens[at];
    a.lp[at] = t >= 0 && t < a.vocab ? lp((float)load_global(x + t)) : 0.f;
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
  constexpr int V = sizeof(T) / 2, U = 4;  // 16-byte loads of a chunk, chunks in flight
  __shared__ u64 buf[LP_W][TOP ? 128 : 1];
  __shared__ Sums part[LP_W];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = WPR == 1 ? blockIdx.x * LP_W + w : blockIdx.x / a.S;
  const int split = WPR == 1 ? 0 : blockIdx.x % a.S;
  if (WPR == 1 && row >= a.rows) return;
  const T* x = static_cast<const T*>(a.x) + (int64_t)row * a.stride;
  const int off = (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T));
  const int chunks = (int)(((int64_t)a.vocab + off + 7) >> 3);
  const int last = (int)min((int64_t)chunks, (int64_t)(split + 1) * a.per);
  const int first = (int)((int64_t)split * a.per) + (WPR == 1 ? 0 : w) * 64 + lane;
  Scan<TOP> scan;
  scan.init(a.c, a.k, buf[w], lane);
  // whole chunks, as long as every lane of the wave has U of them
  int at = first;
  const int whole = min(last, (int)(((int64_t)a.vocab + off) >> 3));  // chunks before this one end within the row
  auto any_chunk = [&](int ch) {
    float z[8];
    const int64_t i0 = (int64_t)ch * 8 - off;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      z[e] = ch < last && i0 + e >= 0 && i0 + e < a.vocab ? (float)load_global(x + i0 + e) : -INFINITY;
    scan.add(z, (int)i0);
  };
  if (off && at - lane == 0) {  // the first chunk begins before the row
    any_chunk(at);
    at += 64 * WPR;
  }
  for (; at - lane + 64 * WPR * (U - 1) + 63 < whole; at += 64 * WPR * U) {
    u4 raw[U][V];
#pragma unroll
    for (int n = 0; n < U; ++n)
#pragma unroll
      for (int i = 0; i < V; ++i)
        raw[n][i] = load_global(reinterpret_cast<const u4*>(x + ((int64_t)(at + 64 * WPR * n) * 8 - off)) + i);
#pragma unroll
    for (int n = 0; n < U; ++n) {
      float z[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) z[e] = (float)reinterpret_cast<const T*>(raw[n])[e];
      scan.add(z, (at + 64 * WPR * n) * 8 - off);
    }
  }
  for (; at - lane < last; at += 64 * WPR) any_chunk(at);
  scan.end();
  if constexpr (WPR > 1) {
    if constexpr (TOP) buf[w][lane] = scan.list;
    if (lane == 0) part[w] = scan.v;
    __syncthreads();
    if (w > 0) return;
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < LP_W; ++i) m = fmaxf(m, part[i].m);
    const Base b = base_of(m, a.c);
    Sums v{m, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < LP_W; ++i) {
      Sums q = part[i];
      rebase(q, m, b, a.c);
      v.s += q.s;
      v.u += q.u;
    }
    scan.v = v;
    if constexpr (TOP)
#pragma unroll
      for (int i = 1; i < LP_W; ++i) scan.list = merge64(scan.list, buf[i][lane], lane);
    if (a.S > 1) {
      const int64_t o = (int64_t)row * a.S + split;
      if (lane == 0) *reinterpret_cast<f4*>(a.stats + 4 * o) = (f4){v.m, v.s, v.u, 0.f};
      if (TOP && lane < a.k) a.keys[o * a.k + lane] = scan.list;
      return;
    }
  }
  finish<TYPE>(a, row, scan.v, scan.list, lane);
}

// The splits of a row: a workgroup per row, its waves take splits in turn and meet in pairs.
template <int TYPE>
__global__ __launch_bounds__(64 * LP_JW) void logprobs_join_kernel(const LpArgs a) {
  __shared__ u64 lists[LP_JW][64];
  const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), row = blockIdx.x;
  const int64_t o = (int64_t)row * a.S;
  u64 list = 0;
  if (a.k) {
    for (int s = w; s < a.S; s += LP_JW) {
      const u64 key = lane < a.k ? load_global(a.keys + (o + s) * a.k + lane) : 0;
      list = s == w ? key : merge64(list, key, lane);
    }
    lists[w][lane] = list;
#pragma unroll
    for (int h = LP_JW / 2; h > 0; h >>= 1) {
      __syncthreads();
      if (w < h) lists[w][lane] = list = merge64(list, lists[w + h][lane], lane);
    }
  }
  if (w > 0) return;
  Sums v{-INFINITY, 0.f, 0.f};
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    const int s = s0 + lane;
    const f4 p = s < a.S ? load_global(reinterpret_cast<const f4*>(a.stats) + o + s) : (f4){-INFINITY, 0.f, 0.f, 0.f};
    const float m = fmaxf(v.m, wave_max(p[0]));
    const Base b = base_of(m, a.c);
    Sums q{p[0], p[1], p[2]};
    rebase(q, m, b, a.c);
    rebase(v, m, b, a.c);
    v.s += wave_sum(q.s);
    v.u += wave_sum(q.u);
  }
  finish<TYPE>(a, row, v, list, lane);
}

// How a call is cut: waves of a row (1 or 4), splits of it and their chunks
struct LpPlan {
  int wpr, S, per;
  size_t bytes;
};
LpPlan lp_plan(int rows, int vocab, int k) {
  LpPlan p;
  p.wpr = vocab <= 4096 ? 1 : LP_W;
  const int chunks = (int)(((int64_t)vocab + 7 + 7) >> 3);
  // as many splits as make four workgroups per CU, of 8192 logits at least
  int S = p.wpr == 1 ? 1 : std::max(1, std::min((1024 + rows - 1) / rows, chunks / 1024));
  p.per = (chunks + S - 1) / S;
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
