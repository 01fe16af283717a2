// Queries and keys of packed tokens, before they are attended or cached: each head's RMS norm (optional) and the
// rotation of its first `rd` dims to the token's position, in one pass (mlcv_qk_rope).
//   y = x / sqrt(mean(x^2) + eps) * (w + offset)
//   (y_i, y_{i + rd/2}) turned by the angle pos * theta^(-2 i / rd), i < rd / 2; the dims from rd on stay y
// Everything between the load and the one rounding at the end is float32; the angles are not: at position 131072 a
// float32 angle is off by 2^-8 of a radian.  They are float64 products in turns, of which whole turns are taken off before
// they become float32.
//
// Bound by memory for many tokens (24124 tokens of 40 heads of 128 in bf16: 92.4 us, 5.35 TB/s read and written; a copy reaches
// 5.2), by latency for few (16 tokens of 9 heads of 256: 4 us).
#include "kernels.h"
#include "mlcvla.h"

#include <algorithm>
#include <cmath>

namespace mlcv {

namespace {

constexpr int RP_NT = 256;  // threads per workgroup: four waves, a token each

struct RopeArgs {
  const void *x[2], *w[2];  // queries, keys; their norms' weights
  void* out[2];
  int64_t tok[2], head[2], otok[2], ohead[2];  // element strides
  const int32_t *cu, *kv_lens, *pos;
  int32_t tokens, B, H, rows, rd, w_f32;  // rows: heads of both
  float eps, offset;
  // turns per position of pair i = 8 j + e: one[e] times oct[b] for each bit b of j
  double oct[4], one[8];
};

template <int TYPE>
struct RopeType;
template <>
struct RopeType<MLCV_DTYPE_F16> {
  typedef _Float16 T;
};
template <>
struct RopeType<MLCV_DTYPE_BF16> {
  typedef __bf16 T;
};
template <>
struct RopeType<MLCV_DTYPE_F32> {
  typedef float T;
};

// 8 elements at p, by 16-byte loads and stores past the caches, as each element is read and written once, or one by one
template <class T, bool VEC>
struct Piece {
  T v[8] __attribute__((aligned(16)));
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i)
        reinterpret_cast<u4*>(v)[i] = __builtin_nontemporal_load(reinterpret_cast<const u4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = load_global(p + i);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) __builtin_nontemporal_store(reinterpret_cast<const u4*>(v)[i], reinterpret_cast<u4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i] = v[i];
    }
  }
};

// What is fused is written out below, so that every form of the kernel rounds alike.
//
// sin and cos of 2 pi r, |r| <= 1/2: the nearest quarter turn is taken off, which leaves |x| <= pi / 4, where the Taylor
// polynomials to x^9 and x^10 end within 2e-9
__device__ __forceinline__ void turn(float r, float& s, float& c) {
  const float n = __builtin_rintf(4.0f * r);
  const float x = __builtin_fmaf(-0.25f, n, r) * 6.283185307179586f, z = x * x;
  auto f = [](float a, float b, float c) { return __builtin_fmaf(a, b, c); };
  const float sx = x * f(z, f(z, f(z, f(z, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), 1.0f);
  const float cx = f(z, f(z, f(z, f(z, f(z, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
  const int q = (int)n;
  const float a = q & 1 ? cx : sx, b = q & 1 ? sx : cx;
  s = q & 2 ? -a : a;
  c = (q + 1) & 2 ? -b : b;
}

// the last b with cu[b] <= t, by 64 comparisons at a time; -1 if there is none
__device__ __forceinline__ int find_request(const int32_t* cu, int B, int t, int lane) {
  int lo = 0, hi = B;
  for (;;) {
    const int step = (hi - lo + 63) >> 6;
    const int64_t i = lo + (int64_t)lane * step;
    const unsigned long long le = __ballot(i < hi && load_global(cu + (i < hi ? i : lo)) <= t);
    if (!le) return -1;
    lo += (63 - __builtin_clzll(le)) * step;
    if (step == 1) return lo;
    hi = min(hi, lo + step);
  }
}

// A lane takes the dims 8 j .. + 7 and their partners rd / 2 further on of one head (two neighbouring pieces where they
// are not rotated), so a wave 64 * 16 / HD heads of a token at a time, and a pair never leaves its lane.
template <int TYPE, int HD, bool NORM, bool VEC>
__global__ __launch_bounds__(RP_NT) void qk_rope_kernel(const RopeArgs a) {
  typedef typename RopeType<TYPE>::T T;
  constexpr int LPH = HD / 16, NG = 64 / LPH;  // lanes of a head, heads at once
  const int lane = threadIdx.x & 63, g = lane / LPH, j = lane % LPH;
  const bool rot = j < a.rd / 16;
  const int lo = rot ? 8 * j : a.rd + 16 * (j - a.rd / 16), hi = rot ? lo + a.rd / 2 : lo + 8;

  double f[8];
  {
    double at = rot ? 1.0 : 0.0;
#pragma unroll
    for (int b = 0; b < 4; ++b) at *= (j >> b) & 1 ? a.oct[b] : 1.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = at * a.one[e];
  }
  float w[2][16];
  if constexpr (NORM) {
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int d = e < 8 ? lo + e : hi + e - 8;
        w[z][e] = !a.w[z] ? 1.0f
                          : a.offset + (a.w_f32 ? load_global(static_cast<const float*>(a.w[z]) + d)
                                                : (float)load_global(static_cast<const T*>(a.w[z]) + d));
      }
  }
  const int waves = gridDim.x * (RP_NT / 64);
  for (int t = __builtin_amdgcn_readfirstlane(blockIdx.x * (RP_NT / 64) + (threadIdx.x >> 6)); t < a.tokens;
       t += waves) {
    int64_t pos;
    if (a.pos) {
      pos = a.pos[t];
    } else {
      const int b = find_request(a.cu, a.B, t, lane);
      if (b < 0) continue;
      const int next = a.cu[b + 1];
      if (next <= t) continue;  // behind the last request
      pos = (int64_t)a.kv_lens[b] - ((int64_t)next - t);
    }
    float c[8], s[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const double p = (double)pos * f[e];
      turn((float)__builtin_fma((double)pos, f[e], -__builtin_rint(p)), s[e], c[e]);
    }
    for (int r0 = 0; r0 < a.rows; r0 += NG) {
      const int row = r0 + g;
      if (row >= a.rows) continue;
      const int z = row >= a.H, h = z ? row - a.H : row;
      const T* p = static_cast<const T*>(z ? a.x[1] : a.x[0]) + (int64_t)t * (z ? a.tok[1] : a.tok[0]) +
                   (int64_t)h * (z ? a.head[1] : a.head[0]);
      Piece<T, VEC> u, v;
      u.load(p + lo);
      v.load(p + hi);
      float x[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = (float)u.v[e];
        x[8 + e] = (float)v.v[e];
      }
      if constexpr (NORM) {
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) sq = __builtin_fmaf(x[e], x[e], sq);
#pragma unroll
        for (int o = 1; o < LPH; o <<= 1) sq += __shfl_xor(sq, o);
        const float n = 1.0f / sqrtf(__builtin_fmaf(sq, 1.0f / HD, a.eps));
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = x[e] * n * (z ? w[1][e] : w[0][e]);
      }
      if (a.rd == HD || rot) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float y0 = __builtin_fmaf(x[e], c[e], -(x[8 + e] * s[e])), y1 = __builtin_fmaf(x[8 + e], c[e], x[e] * s[e]);
          // rounded to float32 first everywhere: some forms would get an instruction that rounds to 16 bits at once
          asm("" : "+v"(y0), "+v"(y1));
          u.v[e] = (T)y0;
          v.v[e] = (T)y1;
        }
      } else if constexpr (NORM) {  // not rotated: by an angle of 0 an infinite neighbour would make it NaN
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          u.v[e] = (T)x[e];
          v.v[e] = (T)x[8 + e];
        }
      }
      T* o = static_cast<T*>(z ? a.out[1] : a.out[0]) + (int64_t)t * (z ? a.otok[1] : a.otok[0]) +
             (int64_t)h * (z ? a.ohead[1] : a.ohead[0]);
      u.store(o + lo);
      v.store(o + hi);
    }
  }
}

template <int TYPE, int HD>
int rope_launch(const RopeArgs& a, bool norm, bool vec, hipStream_t st) {
  // What the GPU holds at once, four waves a SIMD, so that a wave's frequencies and weights serve many tokens and all end
  // together: 24124 tokens of 40 heads of 128 in bf16 with norms take 92.4 us with 1024 workgroups, 98.7 with 2048, 108.9 with
  // 512.  (Plain stores and loads 100.0, and 106.5 with 2048.)
  const unsigned grid = (unsigned)std::min(((int64_t)a.tokens + 3) / 4, (int64_t)1024);
  if (norm) {
    if (vec) qk_rope_kernel<TYPE, HD, true, true><<<grid, RP_NT, 0, st>>>(a);
    else qk_rope_kernel<TYPE, HD, true, false><<<grid, RP_NT, 0, st>>>(a);
  } else {
    if (vec) qk_rope_kernel<TYPE, HD, false, true><<<grid, RP_NT, 0, st>>>(a);
    else qk_rope_kernel<TYPE, HD, false, false><<<grid, RP_NT, 0, st>>>(a);
  }
  MLCV_HIP(hipGetLastError());
  return 0;
}
template <int TYPE>
int rope_launch(const RopeArgs& a, int hd, bool norm, bool vec, hipStream_t st) {
  return hd == 64    ? rope_launch<TYPE, 64>(a, norm, vec, st)
         : hd == 128 ? rope_launch<TYPE, 128>(a, norm, vec, st)
                     : rope_launch<TYPE, 256>(a, norm, vec, st);
}

}  // namespace
}  // namespace mlcv

using namespace mlcv;

extern "C" int mlcv_qk_rope(const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok, int64_t k_head,
                            int32_t dtype, int32_t tokens, const int32_t* cu_seqlens, int32_t B,
                            const int32_t* kv_lens, const int32_t* positions, int32_t H, int32_t KV, int32_t hd,
                            int32_t rotary, double theta, int32_t norm, const void* q_weight, const void* k_weight,
                            int32_t w_dtype, float w_offset, float eps, void* q_out, int64_t qo_tok, int64_t qo_head,
                            void* k_out, int64_t ko_tok, int64_t ko_head, void* stream) {
  MLCV_REQUIRE(dtype == MLCV_DTYPE_F16 || dtype == MLCV_DTYPE_BF16 || dtype == MLCV_DTYPE_F32,
               "q and k are float16, bfloat16 or float32");
  MLCV_REQUIRE(tokens >= 0 && B >= 0 && H > 0 && KV > 0, "bad size");
  MLCV_REQUIRE(H <= INT32_MAX / 4 && KV <= INT32_MAX / 4, "too many heads");
  MLCV_REQUIRE(B <= INT32_MAX - 64, "too many requests");
  MLCV_REQUIRE(hd == 64 || hd == 128 || hd == 256, "head_dim must be 64, 128 or 256");
  MLCV_REQUIRE(rotary >= 0 && rotary <= hd && rotary % 16 == 0, "rotary must be a multiple of 16 up to head_dim");
  MLCV_REQUIRE(theta >= 1.0 && theta < 1e30, "theta must be at least 1 and below 1e30");
  MLCV_REQUIRE(norm || (!q_weight && !k_weight), "weights go with norm");
  MLCV_REQUIRE(!norm || (eps >= 0.f && eps < INFINITY), "eps must be finite and not negative");
  MLCV_REQUIRE((!q_weight && !k_weight) || w_dtype == dtype || w_dtype == MLCV_DTYPE_F32,
               "weights are float32 or of the type of q and k");
  MLCV_REQUIRE((!q_weight && !k_weight) || std::isfinite(w_offset), "w_offset must be finite");
  MLCV_REQUIRE(!positions != !(cu_seqlens || kv_lens) || tokens == 0, "positions, or cu_seqlens and kv_lens");
  if (tokens == 0 || (!positions && B == 0)) return 0;
  MLCV_REQUIRE(q && k && q_out && k_out && (positions || (cu_seqlens && kv_lens)), "null pointer");
  // the last round of a wave's tokens still is an int
  MLCV_REQUIRE(tokens <= INT32_MAX - 16384, "more than 2^31 - 16385 tokens");
  auto in_place = [&](int64_t tok, int64_t otok, int64_t heads, int64_t head, int64_t ohead) {
    return (tokens == 1 || tok == otok) && (heads == 1 || head == ohead);
  };
  MLCV_REQUIRE((q != q_out || in_place(q_tok, qo_tok, H, q_head, qo_head)) &&
                   (k != k_out || in_place(k_tok, ko_tok, KV, k_head, ko_head)),
               "an out that is its input must have its strides");
  MLCV_REQUIRE(rows_apart(tokens, qo_tok, H, qo_head, hd) && rows_apart(tokens, ko_tok, KV, ko_head, hd),
               "rows of out overlap");
  RopeArgs a{};
  a.x[0] = q;
  a.x[1] = k;
  a.w[0] = q_weight;
  a.w[1] = k_weight;
  a.out[0] = q_out;
  a.out[1] = k_out;
  const int64_t strides[8] = {q_tok, k_tok, q_head, k_head, qo_tok, ko_tok, qo_head, ko_head};
  for (int z = 0; z < 2; ++z) {
    a.tok[z] = strides[z];
    a.head[z] = strides[2 + z];
    a.otok[z] = strides[4 + z];
    a.ohead[z] = strides[6 + z];
  }
  a.cu = cu_seqlens;
  a.kv_lens = kv_lens;
  a.pos = positions;
  a.tokens = tokens;
  a.B = B;
  a.H = H;
  a.rows = H + KV;
  a.rd = rotary;
  a.w_f32 = w_dtype == MLCV_DTYPE_F32;
  a.eps = eps;
  a.offset = w_offset;
  const double pi2 = 6.283185307179586476925;
  for (int b = 0; b < 4; ++b) a.oct[b] = rotary ? std::pow(theta, -2.0 * (8 << b) / rotary) : 1.0;
  for (int e = 0; e < 8; ++e) a.one[e] = rotary ? std::pow(theta, -2.0 * e / rotary) / pi2 : 0.0;
  const int per = dtype == MLCV_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
  bool vec = true;
  for (const void* p : {q, k, (const void*)q_out, (const void*)k_out})
    vec = vec && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
  for (const int64_t s : strides) vec = vec && s % per == 0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == MLCV_DTYPE_F16    ? rope_launch<MLCV_DTYPE_F16>(a, hd, norm != 0, vec, st)
         : dtype == MLCV_DTYPE_BF16 ? rope_launch<MLCV_DTYPE_BF16>(a, hd, norm != 0, vec, st)
                                    : rope_launch<MLCV_DTYPE_F32>(a, hd, norm != 0, vec, st);
}
