// Attention over the whole prompts of several requests, packed one after another (mlcv_prompt_attention):
// out_i = sum_j softmax_j(scale * q_i . k_j) v_j over the keys [0, limit_i) of the row's own prompt, with
//   limit_i = n (full), or max(i + 1, min(bidir, n)): causal behind a prefix whose tokens all see one another.
// Logits, softmax statistics and sums in float32; the weights are rounded to the tensors' type for the second
// matrix product, as its operands have to be.
//
// Bound by the matrix cores (4 hd flops per query head and visible pair, against 2 bytes per element read) and by the
// softmax's vector work between their products: 2 x 4096 tokens of 16 heads, no mask, run at 1035 TFLOP/s (heads
// of 128), 917 (256) and 838 (64); two causal prompts, 12141
// tokens in all, at 980.  A large fp16 product of the library: 1311.
//
// A workgroup (4 waves) takes 128 rows of one query head of one prompt, 32 per wave (SP = 2: 64 rows, two waves of
// the same 32 rows each with half of a tile's keys, joined at the end), and streams the keys and
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

// 16 bytes per lane from the buffer into LDS at lds + 16 lane.  In assembly, because the compiler waits for every
// DMA in flight before a transposing LDS read, whose memory it does not know; it returns nothing into registers,
// and the loop waits for it before the barrier after which the tile is read.  M0, which holds the LDS address, has to
// be one wait state old.
__device__ __forceinline__ void pr_dma16(u4 r, char* lds, int voff) {
#if defined(__HIP_DEVICE_COMPILE__)
  const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(at), "v"(voff), "s"(r) : "m0");
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
// buffer ends there; a tile that lies behind it reads nothing)
template <int HD, int NK, bool V>
__device__ __forceinline__ void load_tile(const char* base, int64_t tok_bytes, int row, int n, char* lds, int w,
                                          int lane) {
  constexpr int PP = HD / 8, PER = NK * PP / PR_NT;  // 16-byte pieces per row, DMA instructions per wave
  const int have = min(n - row, NK);
  const uint64_t at = reinterpret_cast<uint64_t>(base) + (int64_t)row * tok_bytes;
  u4 r;  // a raw buffer
  r[0] = (uint32_t)at;
  r[1] = (uint32_t)(at >> 32) & 0xffffu;
  r[2] = have > 0 ? (uint32_t)((have - 1) * tok_bytes + HD * 2) : 0u;
  r[3] = 0x00020000u;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int blk = 4 * i + w, slot = blk * 64 + lane, key = slot / PP, s = slot % PP;
    const int piece = V ? v_slot<HD>(key, s) : k_slot<HD>(key, s);  // both maps are their own inverse
    pr_dma16(r, lds + blk * 1024, key * (int)tok_bytes + piece * 16);
  }
}

template <bool BF, int HD, int NK, int SP>
__global__ __launch_bounds__(PR_NT, HD == 256 ? 1 : 2) void prompt_attn_kernel(const PromptArgs a) {
  typedef typename Elem<BF>::T T;
  typedef typename Elem<BF>::V8 V8;
  constexpr int TILE = NK * HD * 2, KS = HD / 16, ND = HD / 32, NS = NK / 32 / SP, ROWS = PR_ROWS / SP;
  // one LDS object: with several, the compiler tags each access with its object and waits for every DMA in flight
  // before a read of the object that the DMA fills
  __shared__ __attribute__((aligned(1024))) char lds[4 * TILE + 64];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, lh = lane >> 5;
  const int part = SP == 1 ? 0 : w >> 1, rw = SP == 1 ? w : w & 1;  // this wave's keys of a tile, its rows

  // request b has the work items [f(b), f(b + 1)), f(b) = floor(cu[b] / 128) + b, at least ceil(n / 128) of them;
  // the long rows of a causal prompt first
  const int h = blockIdx.x % a.H, item = a.items - 1 - blockIdx.x / a.H;
  int* sh = reinterpret_cast<int*>(lds + 4 * TILE);
  if (tid == 0) {
    sh[0] = -1;
    sh[4] = 0;
  }
  __syncthreads();
  int mine = -1, mc0 = 0, mn = 0, mi = 0;
  for (int b = tid; b < a.B; b += PR_NT) {
    const int c0 = min(max(a.cu[b], 0), a.tokens), c1 = min(max(a.cu[b + 1], 0), a.tokens);
    const int f0 = c0 / ROWS + b, f1 = c1 / ROWS + b + 1;
    if (f0 <= item && item < f1 && c1 > c0) {
      mine = b;
      mc0 = c0;
      mn = c1 - c0;
      mi = item - f0;
    }
  }
  // offsets that do not ascend can put an item into several requests: one of them, whole
  if (mine >= 0) atomicMax(sh, mine);
  __syncthreads();
  if (mine >= 0 && mine == sh[0]) {
    sh[1] = mc0;
    sh[2] = mn;
    sh[3] = mi;
  }
  __syncthreads();
  const int b = __builtin_amdgcn_readfirstlane(sh[0]), c0 = __builtin_amdgcn_readfirstlane(sh[1]);
  const int n = __builtin_amdgcn_readfirstlane(sh[2]);
  const int row0 = __builtin_amdgcn_readfirstlane(sh[3]) * ROWS;
  if (b < 0 || row0 >= n) return;
  const int pre = a.causal ? (a.bidir ? min(max(load_global(a.bidir + b), 0), n) : 0) : n;
  const int most = max(min(row0 + ROWS, n), pre);  // keys that some row sees
  const int tiles = (most + NK - 1) / NK;
  const int wrow = row0 + 32 * rw, row = wrow + l32;
  const int lim = min(max(row + 1, pre), n);
  const int every = max(wrow + 1, pre), some = min(max(wrow + 32, pre), n);  // of this wave's rows

  const char* kb = reinterpret_cast<const char*>(a.k) + 2 * ((int64_t)c0 * a.k_tok + (int64_t)(h / a.grp) * a.k_head);
  const char* vb = reinterpret_cast<const char*>(a.v) + 2 * ((int64_t)c0 * a.v_tok + (int64_t)(h / a.grp) * a.v_head);
  // K tiles in buffers 0 and 1, V tiles in 2 and 3
  load_tile<HD, NK, false>(kb, 2 * a.k_tok, 0, n, lds, w, lane);
  load_tile<HD, NK, true>(vb, 2 * a.v_tok, 0, n, lds + 2 * TILE, w, lane);
  load_tile<HD, NK, false>(kb, 2 * a.k_tok, NK, n, lds + TILE, w, lane);

  V8 q[KS];  // row l32, dims 16 ks + 8 lh .. + 7
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

  // The operands of a tile's products in their order.  The next logits': K's row 32 u + l32, piece 2 ks + lh.  The
  // output's: of k step kk and dims 32 d + l32, V's rows 16 kk + 4 lh + (0..3) and 8 more.
  constexpr int NKF = NS * KS, NVF = 2 * NS * ND;
  const int kr = 32 * NS * part;                             // the wave's first key of a tile
  const int vr = 4 * lh + ((lane & 15) >> 2);                // row of the 4 x 16 block this lane addresses
  const int vc = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);  // its 16-byte piece among the tile's 32 dims
  auto k_frag = [&](const char* kt, int u, int ks) {
    return *reinterpret_cast<const V8*>(kt + (kr + 32 * u + l32) * HD * 2 +
                                        k_slot<HD>(kr + 32 * u + l32, 2 * ks + lh) * 16);
  };
  auto frag = [&](const char* kt, const char* vt, int i) {
    if (i < NKF) return k_frag(kt, i % NS, i / NS);
    const int d = (i - NKF) % ND, kk = (i - NKF) / ND;
    u4 x;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int r = kr + 16 * kk + 8 * j + vr;
      const u2v y = pr_read_tr(vt + r * HD * 2 + v_slot<HD>(r, 4 * d + vc) * 16 + 8 * (lane & 1));
      x[2 * j] = y[0];
      x[2 * j + 1] = y[1];
    }
    return __builtin_bit_cast(V8, x);
  };
  // the larger of a row's two lanes, times c
  auto row_top = [&](float x) {
    const unsigned bits = __float_as_uint(x);
    const auto sw = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    return fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * a.c;
  };

  bool poison = false;  // a non-finite value was taken out of a tile that not every row sees
  int poison0 = 0;      // the first key of such a tile
  float top;            // the tile's largest logit of the row, times c
  V8 ring[2];           // operands: the one in use and the next
  // Tile t, s its logits; P = t mod 2 (its buffers).  False: no row of this wave sees any of it.
  auto begin = [&](int t, int P, f16v (&s)[NS]) {
    const char *kt = lds + (P ^ 1) * TILE, *vt = lds + (2 + P) * TILE;
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): this wave's part of the tiles is in LDS
    __syncthreads();
    ring[0] = frag(kt, vt, 0);
    load_tile<HD, NK, false>(kb, 2 * a.k_tok, (t + 2) * NK, n, lds + P * TILE, w, lane);
    load_tile<HD, NK, true>(vb, 2 * a.v_tok, (t + 1) * NK, n, lds + (2 + (P ^ 1)) * TILE, w, lane);
    const int key0 = t * NK;
    // In a tile that not every row sees whole, a non-finite value behind a weight of 0 would reach rows that do
    // not see its key.  Such values are cleared here, and added at the end to the rows that see them.
    if (key0 + NK > max(row0 + 1, pre)) {
      for (int i = tid; i < TILE / 16; i += PR_NT) {
        u4* at = reinterpret_cast<u4*>(lds + (2 + P) * TILE + 16 * i);
        u4 x = *at;
        const uint32_t ones = BF ? 0x7f80u : 0x7c00u;
        bool hit = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool lo = (x[j] & ones) == ones, hi = ((x[j] >> 16) & ones) == ones;
          x[j] &= (lo ? 0u : 0xffffu) | (hi ? 0u : 0xffff0000u);
          hit = hit || lo || hi;
        }
        if (hit) {
          *at = x;
          sh[4] = 1;
        }
      }
      __syncthreads();
      if (!poison && sh[4]) {
        poison0 = key0;
        poison = true;
      }
    }
    if (key0 + kr >= some) return false;
    if (key0 + kr + 32 * NS > every) {  // some row of the wave does not see all of the tile
      float x = -INFINITY;
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          if (key0 + kr + 32 * u + 8 * (e >> 2) + 4 * lh + (e & 3) >= lim) s[u][e] = -INFINITY;
          x = fmaxf(x, s[u][e]);
        }
      top = row_top(x);
    }
    return true;
  };
  auto outgrown = [&] { return __any(top > m + 8.0f); };  // also where m is still -inf
  auto raise = [&] {
    const float mn = fmaxf(m, top);
    const float alpha = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= alpha;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[d] *= alpha;
  };
  // The rest of the tile; nx becomes the next tile's logits (of the last tile: not used).  The matrix products are
  // issued one by one, each behind the LDS read of the next one's operand and before a share of the softmax: the
  // next logits' between the exponentials, the output's between the comparisons of the next logits.
  auto finish = [&](int P, const f16v (&s)[NS], f16v (&nx)[NS]) {
    const char *kt = lds + (P ^ 1) * TILE, *vt = lds + (2 + P) * TILE;
    const float mu = m == -INFINITY ? 0.f : m;
    V8 p[2 * NS];
    float big = -INFINITY;
#pragma unroll
    for (int i = 0; i < NKF + NVF; ++i) {
      if (i + 1 < NKF + NVF) {
        ring[(i + 1) & 1] = frag(kt, vt, i + 1);
        __builtin_amdgcn_sched_barrier(0);
      }
      const V8 f = ring[i & 1];
      if (i < NKF) {
        const int u = i % NS, ks = i / NS;
        if (ks == 0) {
          f16v z;
#pragma unroll
          for (int e = 0; e < 16; ++e) z[e] = 0.f;
          nx[u] = mfma32(f, q[0], z);
        } else {
          nx[u] = mfma32(f, q[ks], nx[u]);
        }
        constexpr int EX = 16 / KS;  // exponentials per product
#pragma unroll
        for (int j = i * EX; j < (i + 1) * EX; ++j) {
          const int uu = j / 16, e = j & 15;
          const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(s[uu][e], a.c, -mu));
          l += x;
          p[2 * uu + (e >> 3)][e & 7] = (T)x;
        }
      } else {
        const int d = (i - NKF) % ND, kk = (i - NKF) / ND;
        o[d] = mfma32(f, p[kk], o[d]);
        constexpr int MX = 8 / ND;  // comparisons per product
#pragma unroll
        for (int j = (i - NKF) * MX; j < (i - NKF + 1) * MX; ++j) big = fmaxf(big, nx[j / 16][j & 15]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    top = row_top(big);
  };

  f16v s0[NS];
  __builtin_amdgcn_s_waitcnt(0x0f70);
  __syncthreads();
  {
    float x = -INFINITY;
#pragma unroll
    for (int u = 0; u < NS; ++u) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s0[u][e] = 0.f;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) s0[u] = mfma32(k_frag(lds, u, ks), q[ks], s0[u]);
#pragma unroll
      for (int e = 0; e < 16; ++e) x = fmaxf(x, s0[u][e]);
    }
    top = row_top(x);
  }
  if constexpr (HD < 256) {
    f16v s1[NS];
    auto step = [&](int t, int P, f16v (&s)[NS], f16v (&nx)[NS]) {
      if (!begin(t, P, s)) return;
      if (outgrown()) raise();
      finish(P, s, nx);
    };
    for (int t = 0; t < tiles; t += 2) {
      step(t, 0, s0, s1);
      if (t + 1 < tiles) step(t + 1, 1, s1, s0);
    }
  } else {
    // The output is rescaled outside the loop that the tiles usually stay in: with a multiply of it inside, the
    // compiler moves its 128 registers between the two kinds of them in every tile (816 instead of 924 TFLOP/s
    // over 2 x 4096 tokens of 16 heads; at the smaller head dims, where there is one kind, this form loses 4%).
    auto advance = [&](int t) {
      f16v s1[NS];
      finish(t & 1, s0, s1);
#pragma unroll
      for (int u = 0; u < NS; ++u) s0[u] = s1[u];
    };
    auto look = [&](int t) { return begin(t, t & 1, s0) ? 1 + outgrown() : 0; };
    for (int t = 0;;) {
      bool moved = false;
      for (; t < tiles; ++t) {
        const int how = look(t);
        if (how == 2) {
          moved = true;
          break;
        }
        if (how == 1) advance(t);
      }
      if (!moved) break;
      raise();
      advance(t);
      ++t;
    }
  }

  __builtin_amdgcn_s_waitcnt(0x0f70);  // no DMA outlives the loop
  {
    const unsigned bits = __float_as_uint(l);
    const auto sw = __builtin_amdgcn_permlane32_swap(bits, bits, false, false);
    l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
  }
  if constexpr (SP == 2) {
    // the two waves of the same rows meet: the second hands over its output (16 bytes per lane and instruction),
    // maximum and sum
    __syncthreads();
    f4* po = reinterpret_cast<f4*>(lds) + rw * (ND * 4 * 64 + 32) + lane;
    f2* pm = reinterpret_cast<f2*>(lds) + (rw * (ND * 4 * 64 + 32) + ND * 4 * 64) * 2 + l32;
    if (part == 1) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          po[(4 * d + i) * 64] = (f4){o[d][4 * i], o[d][4 * i + 1], o[d][4 * i + 2], o[d][4 * i + 3]};
      if (lh == 0) *pm = (f2){m, l};
    }
    __syncthreads();
    if (part == 1) return;
    const f2 ml = *pm;
    const float mn = fmaxf(m, ml[0]);  // finite: every row sees a key of its first tile
    const float f0 = __builtin_amdgcn_exp2f(m - mn), f1 = __builtin_amdgcn_exp2f(ml[0] - mn);
    l = l * f0 + ml[1] * f1;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f4 x = po[(4 * d + i) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[d][4 * i + e] = o[d][4 * i + e] * f0 + x[e] * f1;
      }
  }
  if (row >= n) return;
  if (poison)
    for (int key = poison0; key < lim; ++key) {
      const T* x = reinterpret_cast<const T*>(vb + (int64_t)key * 2 * a.v_tok) + 4 * lh;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float y = (float)load_global(x + 32 * d + 8 * (i >> 2) + (i & 3));
          if (!(fabsf(y) < INFINITY)) o[d][i] += y;
        }
    }
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

template <bool BF>
int prompt_launch(const PromptArgs& a, int hd, bool split, hipStream_t st) {
  const unsigned grid = (unsigned)((int64_t)a.items * a.H);
  if (split) {
    if (hd == 64) prompt_attn_kernel<BF, 64, 64, 2><<<grid, PR_NT, 0, st>>>(a);
    else if (hd == 128) prompt_attn_kernel<BF, 128, 64, 2><<<grid, PR_NT, 0, st>>>(a);
    else prompt_attn_kernel<BF, 256, 64, 2><<<grid, PR_NT, 0, st>>>(a);
  } else {
    if (hd == 64) prompt_attn_kernel<BF, 64, 64, 1><<<grid, PR_NT, 0, st>>>(a);
    else if (hd == 128) prompt_attn_kernel<BF, 128, 64, 1><<<grid, PR_NT, 0, st>>>(a);
    else prompt_attn_kernel<BF, 256, 32, 1><<<grid, PR_NT, 0, st>>>(a);
  }
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
  MLCV_REQUIRE(tokens <= INT32_MAX - 255, "more than 2^31 - 256 tokens");  // the last tile's rows and keys still are ints
  MLCV_REQUIRE(H > 0 && KV > 0 && H % KV == 0, "query heads must be a multiple of the kv heads");
  MLCV_REQUIRE(hd == 64 || hd == 128 || hd == 256, "head_dim must be 64, 128 or 256");
  const float c = scale * 1.4426950408889634f;
  MLCV_REQUIRE(c > 0.f && c < INFINITY, "scale must be positive and below 2.3e38");
  MLCV_REQUIRE(causal || !bidir, "bidir goes with causal attention");
  // Few rows: workgroups of 64 rows, whose waves share them by keys, while even those leave no CU two of them
  // (up to 128 workgroups of 128 rows).  One prompt of 968 tokens, 8 heads of 256: 43.9 -> 32.2 us; 16 heads of 128:
  // 24.5 -> 19.4, of 64: 17.6 -> 13.7.  At 256 workgroups it is level (heads of 64 and 128) or 1.28 times slower.
  // The sides cross between: ragged prompts of heads of 256 are 1.08 times faster with 64 rows at 160 workgroups, level at 184.
  const bool split = ((int64_t)tokens + PR_ROWS - 1) / PR_ROWS * H <= 128;
  const int64_t items = (int64_t)tokens / (split ? PR_ROWS / 2 : PR_ROWS) + B;
  MLCV_REQUIRE(items * H <= UINT32_MAX / PR_NT, "too many workgroups");  // a launch holds less than 2^32 threads
  if (tokens == 0 || B == 0) return 0;
  MLCV_REQUIRE(q && k && v && cu_seqlens && out, "null pointer");
  auto fits = [](const void* p, int64_t tok, int64_t head) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && tok % 8 == 0 && head % 8 == 0;
  };
  MLCV_REQUIRE(fits(q, q_tok, q_head) && fits(k, k_tok, k_head) && fits(v, v_tok, v_head),
               "rows of q, k and v must be 16-byte aligned");
  MLCV_REQUIRE((reinterpret_cast<uintptr_t>(out) & 7) == 0 && o_tok % 4 == 0 && o_head % 4 == 0,
               "rows of out must be 8-byte aligned");
  MLCV_REQUIRE(rows_apart(tokens, o_tok, H, o_head, hd), "rows of out overlap");
  // a tile of keys is addressed through one buffer with 32-bit offsets
  MLCV_REQUIRE(k_tok >= hd && v_tok >= hd && k_tok < (1 << 24) && v_tok < (1 << 24),
               "the tokens of k and v must be between head_dim and 2^24 elements apart");
  PromptArgs a{q, k, v, out, q_tok, q_head, k_tok, k_head, v_tok, v_head, o_tok, o_head, cu_seqlens, bidir, tokens, B,
               H, H / KV, causal != 0, (int32_t)items, c};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return dtype == MLCV_DTYPE_BF16 ? prompt_launch<true>(a, hd, split, st) : prompt_launch<false>(a, hd, split, st);
}
