// Queries and keys of packed tokens, before they are attended or cached: each head's RMS norm (optional) and the
// rotation of its first `rd` dims to the token's position, in one pass (mlcv_qk_rope).
//   y = x / sqrt(mean(x^2) + eps) * (w + offset)
//   (y_i, y_{i + rd/2}) turned by the angle pos * theta^(-2 i / rd), i < rd / 2; the dims from rd on stay y
// Everything between the load and the one rounding at the end is float32; the angles are not: at position 131072 a
// float32 angle is off by 2^-8 of a radian.  They are float64 products in turns, of which whole turns are taken off before
// they become float32.
//
// Bound by memory for many tokens (24124 tokens of 40 heads of 128 in bf16: 90 us, 5.5 TB/s read and written; a copy reaches
// 5.1), by latency for few (16 tokens of 9 heads of 256: 4.1 us).  Figures below are of calls on end in a graph, without the host.
#include "kernels.h"
#include "mlcvla.h"
#include "rows.h"

#include <algorithm>
#include <cmath>

namespace mlcv {

namespace {

constexpr int RP_NT = 256;       // threads per workgroup: four waves, a token each
constexpr int RP_GROUPS = 1280;  // workgroups at most
constexpr int RP_PACK = 8;       // tokens of a wave at once at most: 16 heads of 64, two or more of a token
constexpr int RP_ROUND = RP_GROUPS * (RP_NT / 64) * RP_PACK;  // tokens that all of them take at once at most

struct RopeArgs {
  const void *x[2], *w[2];  // queries, keys; their norms' weights
  void* out[2];
  int64_t tok[2], head[2], otok[2], ohead[2];  // element strides
  const int32_t *cu, *kv_lens, *pos;
  int32_t tokens, B, H, rows, rd, w_f32;  // rows: heads of both
  int32_t pack, part;                     // tokens that a wave takes at once; heads of one that it takes
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

// How a row is read and written: element by element; by 16 bytes; stores past the caches; loads too
enum RopeAccess { RP_SINGLE, RP_WIDE, RP_FAR_STORES, RP_FAR };

// 4 elements at p and 4 at p + gap (16-bit types: 8 in a row)
template <class T, int ACCESS>
struct Piece {
  static constexpr bool VEC = ACCESS != RP_SINGLE;
  T v[8] __attribute__((aligned(16)));
  __device__ __forceinline__ void load(const T* p, int gap) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        const u4* q = reinterpret_cast<const u4*>(p + i * gap);
        reinterpret_cast<u4*>(v)[i] = ACCESS == RP_FAR ? __builtin_nontemporal_load(q) : load_global(q);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = load_global(p + (i < 4 ? i : i - 4 + gap));
    }
  }
  __device__ __forceinline__ void store(T* p, int gap) const {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) {
        u4* q = reinterpret_cast<u4*>(p + i * gap);
        if constexpr (ACCESS == RP_WIDE) *q = reinterpret_cast<const u4*>(v)[i];
        else __builtin_nontemporal_store(reinterpret_cast<const u4*>(v)[i], q);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) p[i < 4 ? i : i - 4 + gap] = v[i];
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

// A lane takes 8 dims of one head and their partners rd / 2 further on (16 dims that are not rotated, where there are such),
// so a wave 1024 / HD heads at a time, and a pair never leaves its lane: heads of one token, one round after another, or of
// a.pack tokens at once where they have few.  Sines and cosines are computed once per token and pair, spread over the lanes,
// and handed round through LDS; by each lane for its own pairs they are four to sixteen times as many (100000 tokens of 3
// heads of 64 in bf16, one token at a time: 76 us; now 21.6, and 42.9 with the sines handed round but one token at a time).
template <int TYPE, int HD, bool NORM, int ACCESS>
__global__ __launch_bounds__(RP_NT, 4) void qk_rope_kernel(const RopeArgs a) {
  typedef typename RopeType<TYPE>::T T;
  constexpr int LPH = HD / 16, NG = 64 / LPH;  // lanes of a head, heads at once
  __shared__ double freq[HD / 2];              // turns per position
  __shared__ __attribute__((aligned(16))) float sc[RP_NT / 64][2][NG * HD / 2];  // of each wave's tokens: sines, cosines
  __shared__ __attribute__((aligned(16))) float wt[NORM ? 2 * HD : 1];
  const int lane = threadIdx.x & 63, g = lane / LPH, j = lane % LPH;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int half = a.rd / 2;  // pairs
  const int turned = a.rd / 16;  // lanes of a head that are
  const bool rot = j < turned;
  // Element e < 8 of the lane is dim lo + (e < 4 ? e : e - 4 + gap), element 8 + e the same from hi on.  float32: in fours, so
  // that neighbouring lanes' 16-byte pieces are neighbours (12000 tokens of 40 heads of 128: 113.4 -> 97.8 us).
  constexpr bool FOURS = sizeof(T) == 4;
  const int step8 = FOURS ? 4 : 8, gap = FOURS ? 4 * (rot ? turned : LPH - turned) : 4;
  const int lo = rot ? step8 * j : a.rd + step8 * (j - turned), hi = rot ? lo + half : lo + 8 * (LPH - turned);
  for (int i = threadIdx.x; i < half; i += RP_NT) {
    double f = 1.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) f = (i & 7) == e ? a.one[e] : f;
#pragma unroll
    for (int b = 0; b < 4; ++b) f *= (i >> (3 + b)) & 1 ? a.oct[b] : 1.0;
    freq[i] = f;
  }
  if constexpr (NORM)
    for (int i = threadIdx.x; i < 2 * HD; i += RP_NT) {
      const int z = i / HD, d = i % HD;
      wt[i] = !a.w[z] ? 1.0f
                      : a.offset + (a.w_f32 ? load_global(static_cast<const float*>(a.w[z]) + d)
                                            : (float)load_global(static_cast<const T*>(a.w[z]) + d));
    }
  __syncthreads();

  // this lane's token of a block, its head of the first round, and the heads up to which the wave goes
  const int from = (int)blockIdx.y * a.part, to = min(a.rows, from + a.part);
  const int mine = a.pack > 1 ? g / a.rows : 0, row0 = a.pack > 1 ? g - mine * a.rows : g + from;
  const bool has = mine < a.pack && row0 < to;
  // Up to 64 requests: their offsets and lengths stay in the lanes.  Up to 4096: every `stride`-th offset does, and a token's
  // request is found by one more round of loads.
  const int stride = (a.B + 63) >> 6;
  int cu0 = 0, cu1 = 0, lens = 0;
  if (!a.pos && lane * (int64_t)stride < a.B) {
    cu0 = load_global(a.cu + lane * stride);
    cu1 = load_global(a.cu + lane * stride + 1);
    lens = load_global(a.kv_lens + lane * stride);
  }
  const int step = (int)gridDim.x * (RP_NT / 64) * a.pack;
  for (int t0 = ((int)blockIdx.x * (RP_NT / 64) + w) * a.pack; t0 < a.tokens; t0 += step) {
    const int t = t0 + mine;
    Piece<T, ACCESS> u, v;
    auto in = [&](int row) {
      const int z = row >= a.H, h = z ? row - a.H : row;
      const T* p = static_cast<const T*>(z ? a.x[1] : a.x[0]) + (int64_t)t * (z ? a.tok[1] : a.tok[0]) +
                   (int64_t)h * (z ? a.head[1] : a.head[0]);
      u.load(p + lo, gap);
      v.load(p + hi, gap);
    };
    bool there = has && t < a.tokens;
    if (there) in(row0);  // on their way while the angles are found
    bool behind = false;
    int next = 0, len = 0;  // of the request of the last token looked up
    for (int i = 0; i < a.pack; ++i) {
      const int ti = min(t0 + i, a.tokens - 1);
      int64_t p = 0;
      bool none = false;
      if (a.pos) {
        p = a.pos[ti];
      } else {
        if (i == 0 || ti >= next) {
          const unsigned long long le = __ballot(lane * (int64_t)stride < a.B && cu0 <= ti);
          const int at = le ? 63 - __builtin_clzll(le) : 0;
          if (stride == 1) {
            next = le ? __builtin_amdgcn_readlane(cu1, at) : ti;
            len = __builtin_amdgcn_readlane(lens, at);
          } else if (stride <= 64) {
            const int k = min(at * stride + lane, a.B - 1);
            const int c0 = load_global(a.cu + k), c1 = load_global(a.cu + k + 1), l = load_global(a.kv_lens + k);
            const unsigned long long in = __ballot(lane < stride && c0 <= ti);
            const int b = in ? 63 - __builtin_clzll(in) : 0;
            next = le && in ? __builtin_amdgcn_readlane(c1, b) : ti;
            len = __builtin_amdgcn_readlane(l, b);
          } else {
            const int b = find_request(a.cu, a.B, ti, lane);
            next = b < 0 ? ti : a.cu[b + 1];
            len = b < 0 ? 0 : a.kv_lens[b];
          }
        }
        none = ti >= next;  // before the first request or behind the last
        p = (int64_t)len - ((int64_t)next - ti);
      }
      // the pairs of this token
      for (int k = lane; k < half; k += 64) {
        const double f = freq[k], turns = (double)p * f;
        float s, c;
        turn((float)__builtin_fma((double)p, f, -__builtin_rint(turns)), s, c);
        sc[w][0][i * half + k] = s;
        sc[w][1][i * half + k] = c;
      }
      if (mine == i) behind = none;
    }
    there = there && !behind;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    float s[8], c[8];
    const int at = rot ? mine * half + lo : 0;
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
      const int k = e && rot ? at + gap : at;
      *reinterpret_cast<f4*>(s + e) = *reinterpret_cast<const f4*>(&sc[w][0][k]);
      *reinterpret_cast<f4*>(c + e) = *reinterpret_cast<const f4*>(&sc[w][1][k]);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int row = row0; there && row < to; row += NG) {
      if (row != row0) in(row);
      const int z = row >= a.H, h = z ? row - a.H : row;
      float x[16];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = (float)u.v[e];
        x[8 + e] = (float)v.v[e];
      }
      if constexpr (NORM) {
        auto squares = [&] {
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < 16; ++e) sq = __builtin_fmaf(x[e], x[e], sq);
#pragma unroll
          for (int o = 1; o < LPH; o <<= 1) sq += __shfl_xor(sq, o);
          return sq;
        };
        float sq = squares(), eps = a.eps;
        // a head whose squares leave float32's range (where eps does not hide them) is normed in other units
        const float unit = sq == INFINITY ? 0x1p-70f : sq < 0x1p-100f && eps < 0x1p-100f ? 0x1p100f : 1.0f;
        if (TYPE != MLCV_DTYPE_F16 && unit != 1.0f) {
#pragma unroll
          for (int e = 0; e < 16; ++e) x[e] *= unit;
          sq = squares();
          eps = eps * unit * unit;
        }
        const float n = 1.0f / sqrtf(__builtin_fmaf(sq, 1.0f / HD, eps));
#pragma unroll
        for (int e = 0; e < 16; e += 4) {
          const f4 y = *reinterpret_cast<const f4*>(wt + z * HD + (e < 8 ? lo : hi) + (e & 4 ? gap : 0));
#pragma unroll
          for (int i = 0; i < 4; ++i) x[e + i] = x[e + i] * n * y[i];
        }
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
      u.store(o + lo, gap);
      v.store(o + hi, gap);
    }
  }
}

template <int TYPE, int HD, bool NORM>
int rope_launch(RopeArgs a, bool vec, hipStream_t st) {
  constexpr int NG = 64 / (HD / 16);
  static_assert(NG / 2 <= RP_PACK, "a round of tokens");
  a.pack = std::max(1, NG / a.rows);
  // What the GPU holds at once, five waves a SIMD, each taking tokens in turn: 24000 tokens of 40 heads of 128 with norms take
  // 87.1 us with 1280 workgroups, 87.7 with 1024, 30000 of 9 heads of 256 56.0 and 59.2; with twice as many it is 87.2 and 57.9.
  // Few tokens: several waves for each, as far as there are rounds of heads (16 tokens of 40 heads of 256 3.9 us, with one 8.0).
  const int64_t most = RP_GROUPS, groups = ((int64_t)a.tokens + 4 * a.pack - 1) / (4 * a.pack);
  const int rounds = (a.rows + NG - 1) / NG, parts = (int)std::max<int64_t>(1, std::min<int64_t>(rounds, most / groups));
  a.part = (rounds + parts - 1) / parts * NG;
  const dim3 grid((unsigned)std::min(groups, most), (unsigned)((a.rows + a.part - 1) / a.part));
  // Past the caches, as far as it pays: stores where each covers whole 64 bytes (16 for each lane of a head that is rotated,
  // and of those that are not), loads where each covers whole lines of 128, and of inputs that the GPU's L2 caches (32 MB)
  // cannot hold: smaller ones the projection may just have written.  Plain, stores and all past the caches:
  //   24000 tokens of 40 heads of 128, bf16 97.3, 93.2, 87.7 us      3000 of them (31 MB) 17.2, 13.0, 15.3; 6000 31.3, 29.9, 28.2
  //   100000 of 16 of 64, f16 83.2, 83.8, 92.4                       60000 of 8 of 64, float32 52.0, 52.3, 54.4
  //   and with 48 dims of 64 rotated 60.3, 117.4, 126.1              24000 of 40 with 112 of 128 rotated 102.9, 114.5, 130.0
  const int turned = a.rd, rest = HD - a.rd;  // bytes of a store: 16 for each 16 dims
  const bool far = (int64_t)a.tokens * a.rows * HD * (TYPE == MLCV_DTYPE_F32 ? 4 : 2) > (int64_t)40 << 20;
  if (!vec) qk_rope_kernel<TYPE, HD, NORM, RP_SINGLE><<<grid, RP_NT, 0, st>>>(a);
  else if (turned % 64 || rest % 64) qk_rope_kernel<TYPE, HD, NORM, RP_WIDE><<<grid, RP_NT, 0, st>>>(a);
  else if (!far || turned % 128 || rest % 128) qk_rope_kernel<TYPE, HD, NORM, RP_FAR_STORES><<<grid, RP_NT, 0, st>>>(a);
  else if constexpr (HD > 64) qk_rope_kernel<TYPE, HD, NORM, RP_FAR><<<grid, RP_NT, 0, st>>>(a);
  MLCV_HIP(hipGetLastError());
  return 0;
}
template <int TYPE>
int rope_launch(const RopeArgs& a, int hd, bool norm, bool vec, hipStream_t st) {
  if (hd == 64) return norm ? rope_launch<TYPE, 64, true>(a, vec, st) : rope_launch<TYPE, 64, false>(a, vec, st);
  if (hd == 128) return norm ? rope_launch<TYPE, 128, true>(a, vec, st) : rope_launch<TYPE, 128, false>(a, vec, st);
  return norm ? rope_launch<TYPE, 256, true>(a, vec, st) : rope_launch<TYPE, 256, false>(a, vec, st);
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
  // a token of the round behind the last still is an int
  static_assert(RP_ROUND == 40960, "in the message");
  MLCV_REQUIRE(tokens <= INT32_MAX - RP_ROUND, "more than 2^31 - 40961 tokens");
  auto in_place = [&](int64_t tok, int64_t otok, int64_t heads, int64_t head, int64_t ohead) {
    return (tokens == 1 || tok == otok) && (heads == 1 || head == ohead);
  };
  MLCV_REQUIRE((q != q_out || in_place(q_tok, qo_tok, H, q_head, qo_head)) &&
                   (k != k_out || in_place(k_tok, ko_tok, KV, k_head, ko_head)),
               "an out that is its input must have its strides");
  MLCV_REQUIRE(rows_apart(tokens, qo_tok, H, qo_head, hd) && rows_apart(tokens, ko_tok, KV, ko_head, hd),
               "rows of out overlap");
  const Rows::Int size = dtype == MLCV_DTYPE_F32 ? 4 : 2, w_size = w_dtype == MLCV_DTYPE_F32 ? 4 : 2;
  auto rows = [&](const void* p, int64_t tok, int64_t heads, int64_t head) {
    return Rows(p, tokens, tok * size, heads, head * size, hd * size);
  };
  const Rows arrays[] = {rows(q_out, qo_tok, H, qo_head), rows(k_out, ko_tok, KV, ko_head),
                         rows(q == q_out ? nullptr : q, q_tok, H, q_head), rows(k == k_out ? nullptr : k, k_tok, KV, k_head),
                         Rows(cu_seqlens, 4 * ((int64_t)B + 1)), Rows(kv_lens, 4 * (int64_t)B),
                         Rows(positions, 4 * (int64_t)tokens), Rows(q_weight, hd * w_size), Rows(k_weight, hd * w_size)};
  MLCV_REQUIRE(!any_meet(arrays, 2, 9), "an out overlaps an input or the other out");
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
