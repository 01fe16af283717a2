// Attention over the whole prompts of several requests, packed one after another (mlcv_prompt_attention):
// out_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys [0, limit_i) of the row's own prompt, with
//   limit_i = n (full), or max(i + 1, min(bidir, n)): causal behind a prefix whose tokens all see one another.
// Logits, softmax statistics and sums in float32; the weights are rounded to the tensors' type for the second
// matrix product, as its operands have to be.
//
// Bound by the matrix cores (4 hd flops per query head and visible pair, against 2 bytes per element read).
//
// A workgroup (4 waves) takes 128 rows of one query head of one prompt, 32 per wave, and streams the keys and
// values in tiles through two LDS buffers that global -> LDS DMA fills one tile ahead.  A wave computes
// S^T = K . Q^T and O^T = V^T . P^T on v_mfma_f32_32x32x16: with lane = 32 lh + r, S^T leaves keys
// 8 i + 4 lh + (0..3) of row r in a lane, and the second product contracts over keys in any order as long as
// both operands agree, so the weights go from the first product to the second without leaving their lanes: its
// k step kk takes keys 16 kk + 4 lh + (0..3) and 16 kk + 8 + 4 lh + (0..3) from lane half lh.  V's operand (one
// dim per lane, those 8 keys) is read from the row-major tile by the transposing LDS read, 4 keys x 16 dims per
// 16 lanes.  Everything of a query row (maximum, sum, output) stays in lanes r and 32 + r.
//
// The running maximum is only raised where it grew by more than 2^8: until then the weights, up to 2^8, are
// right under the old one, and the output needs no rescaling.
#include "kernels.h"
#include "mlcvla.h"

#include <algorithm>
#include <cmath>

namespace mlcv {

namespace {

constexpr int PR_NT = 256;    // threads per workgroup
constexpr int PR_ROWS = 128;  // query rows per workgroup

struct PromptArgs {
  const void *q, *k, *v;
  void* out;
  int64_t q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head;  // element strides
  const int32_t *cu, *bidir;
  int32_t tokens, B, H, grp, causal, items;
  float c;  // scale * log2(e)
};

template <bool BF>
struct Elem {
  typedef _Float16 T;
  typedef _Float16 V8 __attribute__((ext_vector_type(8)));
  typedef _Float16 V4 __attribute__((ext_vector_type(4)));
};
template <>
struct Elem<true> {
  typedef __bf16 T;
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
  typedef __bf16 V4 __attribute__((ext_vector_type(4)));
};
__device__ __forceinline__ f16v mfma32(Elem<false>::V8 a, Elem<false>::V8 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f16v mfma32(Elem<true>::V8 a, Elem<true>::V8 b, f16v c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// 16 bytes per lane from the buffer into LDS at lds + 16 lane (device pass only: in the host pass the builtin
// drops the kernel's launch stub)
__device__ __forceinline__ void pr_dma16(__amdgpu_buffer_rsrc_t r, char* lds, int voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, voff, 0, 0, 0);
#endif
}
// four 16-bit elements of one column: per 16 lanes a 4 x 16 block, lane i giving the address of row i / 4,
// columns 4 (i mod 4) .. + 3, and receiving column i
__device__ __forceinline__ u2v pr_read_tr(const char* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  typedef short s4 __attribute__((ext_vector_type(4)));
  return __builtin_bit_cast(u2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)lds));
#else
  return (u2v){0, 0};
#endif
}

// LDS slot of 16-byte piece p of key row r, K tile: the 16 rows that 16 lanes read at once in distinct slots of
// a 256-byte bank line
template <int HD>
__device__ __forceinline__ int k_slot(int r, int p) {
  return HD >= 128 ? p ^ (r & 15) : p ^ ((r >> 1) & 7);
}
// V tile: the transposing read takes 64 bytes of each of 8 rows (4 per lane half): rows 0..3 in distinct
// quarters of the bank line
template <int HD>
__device__ __forceinline__ int v_slot(int r, int p) {
  return HD >= 128 ? p ^ ((r & 3) << 2) : p ^ (((r >> 1) & 1) << 2);
}

// DMA of rows [row, row + NK) of one head of K or V into LDS; rows past the prompt's end become zeros (the
// buffer ends there)
template <int HD, int NK, bool V>
__device__ __forceinline__ void load_tile(const char* base, int64_t tok_bytes, int row, int n, char* lds, int w,
                                          int lane) {
  constexpr int PP = HD / 8, PER = NK * PP / PR_NT;  // 16-byte pieces per row, DMA instructions per wave
  const int have = min(n - row, NK);                 // >= 1
  const __amdgpu_buffer_rsrc_t r =
      dev_rsrc(base + (int64_t)row * tok_bytes, (uint32_t)((have - 1) * tok_bytes + HD * 2));
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int blk = 4 * i + w, slot = blk * 64 + lane, key = slot / PP, s = slot % PP;
    const int piece = V ? v_slot<HD>(key, s) : k_slot<HD>(key, s);  // both maps are their own inverse
    pr_dma16(r, lds + blk * 1024, key * (int)tok_bytes + piece * 16);
  }
}

template <bool BF, int HD, int NK>
__global__ __launch_bounds__(PR_NT, HD == 256 ? 1 : 2) void prompt_attn_kernel(const PromptArgs a) {
  typedef typename Elem<BF>::T T;
  typedef typename Elem<BF>::V8 V8;
  constexpr int TILE = NK * HD * 2, KS = HD / 16, ND = HD / 32, NS = NK / 32;
  // one LDS object, so that the compiler sees one thing that the DMA and the reads touch
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE + 64];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lh = lane >> 5;

  // request b has the work items [f(b), f(b + 1)), f(b) = floor(cu[b] / 128) + b, at least ceil(n / 128) of them
  const int h = blockIdx.x % a.H, item = a.items - 1 - blockIdx.x / a.H;
  int* sh = reinterpret_cast<int*>(lds + 4 * TILE);
  if (tid == 0) sh[0] = -1;
  __syncthreads();
  for (int b = tid; b < a.B; b += PR_NT) {
    const int c0 = min(max(a.cu[b], 0), a.tokens), c1 = min(max(a.cu[b + 1], 0), a.tokens);
    const int f0 = c0 / PR_ROWS + b, f1 = c1 / PR_ROWS + b + 1;
    if (f0 <= item && item < f1 && c1 > c0) {
      sh[0] = b;
      sh[1] = c0;
      sh[2] = c1 - c0;
      sh[3] = item - f0;
    }
  }
  __syncthreads();
  const int b = __builtin_amdgcn_readfirstlane(sh[0]), c0 = __builtin_amdgcn_readfirstlane(sh[1]);
  const int n = __builtin_amdgcn_readfirstlane(sh[2]);
  const int row0 = __builtin_amdgcn_readfirstlane(sh[3]) * PR_ROWS;
  if (b < 0 || row0 >= n) return;
  const int pre = a.causal ? (a.bidir ? min(max(load_global(a.bidir + b), 0), n) : 0) : n;
  const int most = max(min(row0 + PR_ROWS, n), pre);  // keys that some row sees
  const int tiles = (most + NK - 1) / NK;
  const int wrow = row0 + 32 * w, row = wrow + l32;
  const int lim = min(max(row + 1, pre), n);
  const int every = max(wrow + 1, pre), some = min(max(wrow + 32, pre), n);  // of this wave's rows

  const char* kb = reinterpret_cast<const char*>(a.k) + 2 * ((int64_t)c0 * a.k_tok + (int64_t)(h / a.grp) * a.k_head);
  const char* vb = reinterpret_cast<const char*>(a.v) + 2 * ((int64_t)c0 * a.v_tok + (int64_t)(h / a.grp) * a.v_head);
  load_tile<HD, NK, false>(kb, 2 * a.k_tok, 0, n, lds, w, lane);
  load_tile<HD, NK, true>(vb, 2 * a.v_tok, 0, n, lds + TILE, w, lane);

  V8 q[KS];  // row r, dims 16 ks + 8 lh .. + 7
  {
    const T* p = reinterpret_cast<const T*>(a.q) + (int64_t)(c0 + min(row, n - 1)) * a.q_tok + (int64_t)h * a.q_head +
                 8 * lh;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) q[ks] = load_global(reinterpret_cast<const V8*>(p + 16 * ks));
  }
  f16v o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float m = -INFINITY, l = 0.f;

  for (int t = 0; t < tiles; ++t) {
    char* cur = lds + (t & 1) * 2 * TILE;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the tile is in LDS
    __syncthreads();
    if (t + 1 < tiles) {
      char* nxt = lds + ((t + 1) & 1) * 2 * TILE;
      load_tile<HD, NK, false>(kb, 2 * a.k_tok, (t + 1) * NK, n, nxt, w, lane);
      load_tile<HD, NK, true>(vb, 2 * a.v_tok, (t + 1) * NK, n, nxt + TILE, w, lane);
    }
    const int key0 = t * NK;
    const bool edge = key0 + NK > every;  // some row of the wave does not see all of the tile
    // a tile that every row sees in part: a non-finite value behind a weight of 0 would reach rows that do not
    // see its key, so such a tile is looked through, by the whole workgroup
    bool apart = false;
    if (key0 + NK > max(row0 + 1, pre)) {
      int bad = 0;
      for (int i = tid; i < TILE / 16; i += PR_NT) {
        const u4 x = *reinterpret_cast<const u4*>(cur + TILE + 16 * i);
        const uint32_t ones = BF ? 0x7f80u : 0x7c00u;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          bad |= (x[j] & ones) == ones || ((x[j] >> 16) & ones) == ones;
      }
      apart = __syncthreads_or(bad);
    }
    if (key0 >= some) continue;  // nothing that this wave's rows see

    f16v s[NS];
#pragma unroll
    for (int u = 0; u < NS; ++u) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[u][e] = 0.f;
      const char* krow = cur + (32 * u + l32) * HD * 2;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        const V8 kf = *reinterpret_cast<const V8*>(krow + k_slot<HD>(32 * u + l32, 2 * ks + lh) * 16);
        s[u] = mfma32(kf, q[ks], s[u]);
      }
    }
    if (edge) {
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          if (key0 + 32 * u + 8 * (e >> 2) + 4 * lh + (e & 3) >= lim) s[u][e] = -INFINITY;
    }
    float top = -INFINITY;
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) top = fmaxf(top, s[u][e]);
    {
      const unsigned bits = __float_as_uint(top);
      const auto sw = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
      top = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * a.c;
    }
    if (__any(top > m + 8.0f)) {  // also where m is still -inf
      const float mn = fmaxf(m, top);
      const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
    }
    const float mu = m == -INFINITY ? 0.f : m;
    V8 p[2 * NS];
#pragma unroll
    for (int u = 0; u < NS; ++u)
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][e], a.c, -mu));
        l += x;
        p[2 * u + (e >> 3)][e & 7] = (T)x;
      }
    // V's operand of k step kk, dims 32 d + l32: rows 16 kk + 4 lh + (0..3) and 8 more
    const int vr = 4 * lh + ((lane & 15) >> 2);  // row of the 4 x 16 block this lane addresses
    const int vc = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);  // its 16-byte piece among the tile's 32 dims
    auto v_frag = [&](int d, int kk) {
      u4 x;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int r = 16 * kk + 8 * j + vr;
        const u2v y = pr_read_tr(cur + TILE + r * HD * 2 + v_slot<HD>(r, 4 * d + vc) * 16 + 8 * (lane & 1));
        x[2 * j] = y[0];
        x[2 * j + 1] = y[1];
      }
      return x;
    };
    if (!apart) {
#pragma unroll
      for (int kk = 0; kk < 2 * NS; ++kk)
#pragma unroll
        for (int d = 0; d < ND; ++d) o[d] = mfma32(__builtin_bit_cast(V8, v_frag(d, kk)), p[kk], o[d]);
    } else {
      // key by key: a product with that key alone, added to the rows that see it
#pragma unroll
      for (int kk = 0; kk < 2 * NS; ++kk)
        for (int i = 0; i < 16; ++i) {
          const int e = i & 7, half = i >> 3, key = key0 + 16 * kk + 8 * (e >> 2) + 4 * half + (e & 3);
          const uint32_t mine = lh == half ? (e & 1 ? 0xffff0000u : 0xffffu) : 0u;
#pragma unroll
          for (int d = 0; d < ND; ++d) {
            u4 x = v_frag(d, kk);
#pragma unroll
            for (int j = 0; j < 4; ++j) x[j] &= (e >> 1) == j ? mine : 0u;
            f16v z;
#pragma unroll
            for (int j = 0; j < 16; ++j) z[j] = 0.f;
            z = mfma32(__builtin_bit_cast(V8, x), p[kk], z);
            if (key < lim) o[d] += z;
          }
        }
    }
  }

  {
    const unsigned bits = __float_as_uint(l);
    const auto sw = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if (row < n) {
    const float f = 1.0f / l;  // every row sees its own key at least
    T* dst = reinterpret_cast<T*>(a.out) + (int64_t)(c0 + row) * a.o_tok + (int64_t)h * a.o_head;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        typename Elem<BF>::V4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (T)(o[d][4 * i + e] * f);
        *reinterpret_cast<typename Elem<BF>::V4*>(dst + 32 * d + 8 * i + 4 * lh) = x;
      }
  }
}

template <bool BF>
int prompt_launch(const PromptArgs& a, int hd, hipStream_t st) {
  const unsigned grid = (unsigned)((int64_t)a.items * a.H);
  if (hd == 64) prompt_attn_kernel<BF, 64, 64><<<grid, PR_NT, 0, st>>>(a);
  else if (hd == 128) prompt_attn_kernel<BF, 128, 64><<<grid, PR_NT, 0, st>>>(a);
  else prompt_attn_kernel<BF, 256, 32><<<grid, PR_NT, 0, st>>>(a);
  MLCV_HIP(hipGetLastError());
  return 0;
}

}  // namespace
}  // namespace mlcv

using namespace mlcv;

extern "C" int mlcv_prompt_attention(const void* q, int64_t q_tok, int64_t q_head, const void* k, int64_t k_tok,
                                     int64_t k_head, const void* v, int64_t v_tok, int64_t v_head, int32_t dtype,
                                     int32_t tokens, const int32_t* cu_seqlens, int32_t B, int32_t H, int32_t KV,
                                     int32_t hd, float scale, int32_t causal, const int32_t* bidir, void* out,
                                     int64_t o_tok, int64_t o_head, void* stream) {
  MLCV_REQUIRE(dtype == MLCV_DTYPE_F16 || dtype == MLCV_DTYPE_BF16, "q, k and v are float16 or bfloat16");
  MLCV_REQUIRE(tokens >= 0 && B >= 0, "negative size");
  MLCV_REQUIRE(H > 0 && KV > 0 && H % KV == 0, "query heads must be a multiple of the kv heads");
  MLCV_REQUIRE(hd == 64 || hd == 128 || hd == 256, "head_dim must be 64, 128 or 256");
  MLCV_REQUIRE(scale > 0.f && scale < INFINITY, "scale must be positive and finite");
  MLCV_REQUIRE(causal || !bidir, "bidir goes with causal attention");
  const int64_t items = (int64_t)tokens / PR_ROWS + B;
  MLCV_REQUIRE(items * H <= INT32_MAX, "too many workgroups");
  if (tokens == 0 || B == 0) return 0;
  MLCV_REQUIRE(q && k && v && cu_seqlens && out, "null pointer");
  auto fits = [](const void* p, int64_t tok, int64_t head) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && tok % 8 == 0 && head % 8 == 0;
  };
  MLCV_REQUIRE(fits(q, q_tok, q_head) && fits(k, k_tok, k_head) && fits(v, v_tok, v_head),
               "rows of q, k and v must be 16-byte aligned");
  MLCV_REQUIRE((reinterpret_cast<uintptr_t>(out) & 7) == 0 && o_tok % 4 == 0 && o_head % 4 == 0,
               "rows of out must be 8-byte aligned");
  // a tile of keys is addressed through one buffer with 32-bit offsets
  MLCV_REQUIRE(k_tok >= hd && v_tok >= hd && k_tok < (1 << 24) && v_tok < (1 << 24),
               "the tokens of k and v must be between head_dim and 2^24 elements apart");
  PromptArgs a{q, k, v, out, q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head, cu_seqlens, bidir, tokens, B,
               H, H / KV, causal != 0, (int32_t)items, scale * 1.4426950408889634f};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == MLCV_DTYPE_BF16 ? prompt_launch<true>(a, hd, st) : prompt_launch<false>(a, hd, st);
}
