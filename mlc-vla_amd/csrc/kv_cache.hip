// The paged 8-bit key/value cache of several requests: block tables and slot maps from request lengths
// (mlcv_kv_plan), the cache's writer (mlcv_kv_write) and the attention over it (mlcv_kv_attention).
//
// A page holds `page` tokens (16, 32, 64 or 128) of every kv head in e4m3 with one float32 scale per page, kv
// head and side:
//   keys   [pages][KV][page][hd]      values [pages][KV][hd][page] (token innermost)
// x is held as code * scale with scale = 2^e, the smallest e >= -64 with max|x| <= 448 * 2^e over the page's
// tokens.  A power of two loses nothing against any other scale (a floating-point code has the same relative
// step at every exponent), and it makes every rescaling exact but for the codes that fall below 2^-6: a page
// that grows token by token holds what one write of all its tokens would hold, to the subnormals' step.
// Values are held token-innermost because the attention's second product contracts over tokens: its matrix
// operand is then 16 contiguous bytes per lane, as is the first product's over the head dim.
#include "kernels.h"
#include "kv_args.h"
#include "mlcvla.h"

#include <algorithm>
#include <cmath>

namespace mlcv {

namespace {

constexpr int KV_NT = 256;         // threads per workgroup of every kernel here
constexpr int KV_RT = 16;          // query rows of an attention workgroup
constexpr float LOG2E = 1.4426950408889634f;

// ---- plan ------------------------------------------------------------------------------------------

// The last index b in [0, n) with a[b] <= v (a ascending, a[0] <= v).
__device__ __forceinline__ int last_le(const int* a, int n, int v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= v) lo = mid;
    else hi = mid;
  }
  return lo;
}

struct PlanArgs {
  const int32_t *past, *fresh, *free_pages, *free_count;
  int32_t *table, *cu, *kv_lens, *slots, *status;
  int32_t B, n_free, num_pages, psh, max_pages, tokens, slot_blocks;
};

// had = ceil(past / page), has = ceil((past + new) / page); request b takes the has - had pages from the free list that
// follow those of the requests before it, and slot = table[pos / page] * page + pos % page.
// Every workgroup runs the same scan over the requests (two loads and a prefix sum per 256 of them, which costs
// less than a second launch that waits for the first), then fills its own part of the slot map or of the table.
// Bound by launch and load latency: 3.1 us for 16 requests of one new token, 8.9 for 256 of up to 1168 (170000 tokens).
// The scan is the smaller part of that: 256 requests of one token take 0.3 us more than 16.  A thread's four slots cost 1.2
// us each, as their chains of search, length and page number run one after another.
__global__ __launch_bounds__(KV_NT) void kv_plan_kernel(const PlanArgs a) {
  extern __shared__ int sm[];
  __shared__ long long part[KV_NT / 64];
  __shared__ int sbad, sused;
  int* scu = sm;                // [B + 1] first token of each request
  int* sbase = sm + a.B + 1;    // [B + 1] first page it takes from the free list; ~base where it is refused
  const int tid = threadIdx.x, page = 1 << a.psh;
  const int n_free = a.free_count ? clamp_i(*a.free_count, 0, a.n_free) : a.n_free;
  if (tid == 0) sbad = sused = 0;
  __syncthreads();
  long long tok0 = 0, pg0 = 0;
  int bad = 0, used = 0;
  for (int b0 = 0; b0 < a.B; b0 += KV_NT) {
    const int b = b0 + tid;
    const bool in = b < a.B;
    const long long p = in ? a.past[b] : 0, q = in ? a.fresh[b] : 0;
    const long long qn = q > 0 ? q : 0;
    const long long end = block_scan<KV_NT>(qn, part) + tok0;
    const long long had = (p + page - 1) >> a.psh, has = (p + qn + page - 1) >> a.psh;
    const bool fits = in && p >= 0 && q >= 0 && has <= a.max_pages && end <= a.tokens;
    const long long need = fits ? has - had : 0;
    const long long pend = block_scan<KV_NT>(need, part) + pg0;
    const bool ok = fits && (need == 0 || pend <= n_free);
    if (in) {
      const long long first = end - qn;
      scu[b] = (int)(first < a.tokens ? first : a.tokens);
      // pages past the free list are never indexed: a refused request has no slots and no table entries
      const long long base = pend - need < n_free ? pend - need : n_free;
      sbase[b] = ok ? (int)base : ~(int)base;
      bad += !ok;
      if (ok && need > 0) used = (int)pend;  // granted: at most n_free; ascending over b
      if (blockIdx.x == 0) {
        a.cu[b] = scu[b];
        a.kv_lens[b] = ok ? (int)(p + q) : 0;
      }
    }
    // the last thread's sums carry over
    __shared__ long long carry[2];
    if (tid == KV_NT - 1) {
      carry[0] = end;
      carry[1] = pend;
    }
    __syncthreads();
    tok0 = carry[0];
    pg0 = carry[1];
    __syncthreads();
  }
  if (bad) atomicAdd(&sbad, bad);
  if (used) atomicMax(&sused, used);
  if (tid == 0) {
    scu[a.B] = (int)(tok0 < a.tokens ? tok0 : a.tokens);
    sbase[a.B] = (int)(pg0 < n_free ? pg0 : n_free);
  }
  __syncthreads();
  if ((int)blockIdx.x < a.slot_blocks) {  // slots
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const long long t = (long long)blockIdx.x * 4 * KV_NT + i * KV_NT + tid;
      if (t >= a.tokens) break;
      int slot = -1;
      if (t < scu[a.B]) {
        const int b = last_le(scu, a.B, (int)t), base = sbase[b];
        if (base >= 0) {
          const int p = a.past[b], had = (int)(((long long)p + page - 1) >> a.psh);
          const int pos = p + ((int)t - scu[b]), pg = pos >> a.psh;
          const int id = pg < had ? a.table[(size_t)b * a.max_pages + pg] : a.free_pages[base + pg - had];
          if (id >= 0 && id < a.num_pages) slot = (id << a.psh) + (pos & (page - 1));
        }
      }
      a.slots[t] = slot;
    }
    if (blockIdx.x == 0 && tid == 0) {
      a.cu[a.B] = scu[a.B];
      a.status[0] = sused;
      a.status[1] = sbad;
    }
  } else {  // table entries, one thread for each page taken
    const int f = ((int)blockIdx.x - a.slot_blocks) * KV_NT + tid;
    if (f >= sbase[a.B]) return;
    // the request that takes page f: the last whose base (refused or not) is <= f
    int lo = 0, hi = a.B;
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1, v = sbase[mid];
      if ((v >= 0 ? v : ~v) <= f) lo = mid;
      else hi = mid;
    }
    if (sbase[lo] < 0) return;
    const int had = (int)(((long long)a.past[lo] + page - 1) >> a.psh);
    a.table[(size_t)lo * a.max_pages + had + f - sbase[lo]] = a.free_pages[f];
  }
}

// ---- the page a workgroup works on ------------------------------------------------------------------

// Work items of a packed batch, without knowing its lengths on the host: request b takes the item numbers
// [f(b), f(b + 1)) with f(b) = floor(cu[b] * mul / div) + extra * b.  f grows by at least the request's
// ceil(n * mul / div) items (extra = 1), or one more for a first page that is not empty (extra = 2), so that
// floor(tokens * mul / div) + extra * B items always do; the few that are left over end at once.
// Every thread tests its own b: one round of loads instead of a chain of dependent ones.
struct Item {
  int b, c0, n;  // request, its first token and number of tokens; b = -1: none
  int i;         // the item's number within its request
  int len;       // its kv_lens entry, where the caller gives them
};
__device__ __forceinline__ Item find_item(const int32_t* cu, const int32_t* lens, int B, int tokens, long long item,
                                          int mul, int div, int extra, int* sh) {
  if (threadIdx.x == 0) sh[0] = -1;
  __syncthreads();
  int mine = -1, mc0 = 0, mn = 0, mi = 0, ml = 0;
  for (int b = threadIdx.x; b < B; b += KV_NT) {
    const int len = lens ? lens[b] : 0;
    const int c0 = clamp_i(cu[b], 0, tokens), c1 = clamp_i(cu[b + 1], 0, tokens);
    const long long f0 = (long long)c0 * mul / div + (long long)extra * b;
    const long long f1 = (long long)c1 * mul / div + (long long)extra * (b + 1);
    if (f0 <= item && item < f1 && c1 > c0) {
      mine = b;
      mc0 = c0;
      mn = c1 - c0;
      mi = (int)(item - f0);
      ml = len;
    }
  }
  // offsets that do not ascend can put an item into several requests: one of them, whole
  if (mine >= 0) atomicMax(sh, mine);
  __syncthreads();
  if (mine >= 0 && mine == sh[0]) {
    sh[1] = mc0;
    sh[2] = mn;
    sh[3] = mi;
    sh[4] = ml;
  }
  __syncthreads();
  Item r;
  r.b = __builtin_amdgcn_readfirstlane(sh[0]);
  r.c0 = __builtin_amdgcn_readfirstlane(sh[1]);
  r.n = __builtin_amdgcn_readfirstlane(sh[2]);
  r.i = __builtin_amdgcn_readfirstlane(sh[3]);
  r.len = __builtin_amdgcn_readfirstlane(sh[4]);
  return r;
}

// ---- write -----------------------------------------------------------------------------------------

struct WriteArgs {
  const void* x[2];       // keys, values
  int64_t tok[2], head[2];  // element strides
  uint8_t* cache[2];
  float* scale[2];
  const int32_t *cu, *slots;
  int32_t type[2], vec[2];  // vec: rows are 16-byte aligned
  int32_t tokens, B, num_pages, psh, KV;
};

// 8 elements as float32, from 16 (float32: 32) bytes
__device__ __forceinline__ void widen(int type, const u4* raw, float* out) {
  if (type == MLCV_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 8; ++i) out[i] = __uint_as_float(raw[i >> 2][i & 3]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t w = raw[0][i];
    if (type == MLCV_DTYPE_F16) {
      const h2 v = __builtin_bit_cast(h2, w);
      out[2 * i] = (float)v[0];
      out[2 * i + 1] = (float)v[1];
    } else {
      out[2 * i] = __uint_as_float(w << 16);
      out[2 * i + 1] = __uint_as_float(w & 0xffff0000u);
    }
  }
}
// N rows of 8 elements at p + at[n] (elements), those with on[n]; zeros elsewhere.  The type is settled outside of
// the loads, so that they are all in flight at once.
template <int TYPE, bool VEC, int N>
__device__ __forceinline__ void load_rows(const void* p, const int64_t* at, const bool* on, float (*out)[8]) {
  constexpr int W = TYPE == MLCV_DTYPE_F32 ? 2 : 1;
  u4 raw[N][W];
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      raw[n][w] = (u4){0, 0, 0, 0};
      if (!on[n]) continue;
      const char* x = reinterpret_cast<const char*>(p) + at[n] * (TYPE == MLCV_DTYPE_F32 ? 4 : 2) + 16 * w;
      if (VEC) {
        raw[n][w] = load_global(reinterpret_cast<const u4*>(x));
      } else if (TYPE == MLCV_DTYPE_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[n][w][i] = load_global(reinterpret_cast<const uint32_t*>(x) + i);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          raw[n][w][i] = load_global(reinterpret_cast<const uint16_t*>(x) + 2 * i) |
                         (uint32_t)load_global(reinterpret_cast<const uint16_t*>(x) + 2 * i + 1) << 16;
      }
    }
#pragma unroll
  for (int n = 0; n < N; ++n) widen(TYPE, raw[n], out[n]);
}

// four values as e4m3, rounded to nearest even; past the largest finite value (infinities among them) they
// saturate, NaN stays NaN
__device__ __forceinline__ float sat448(float x) { return x > 448.f ? 448.f : x < -448.f ? -448.f : x; }
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(sat448(a), sat448(b), 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(sat448(c), sat448(d), r, true);
}
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
  const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  return pack4(a[0] * ratio, a[1] * ratio, b[0] * ratio, b[1] * ratio);
}
// bytes [lo, hi) of a 4-byte word
__device__ __forceinline__ uint32_t byte_mask(int lo, int hi) {
  lo = clamp_i(lo, 0, 4);
  hi = clamp_i(hi, 0, 4);
  if (lo >= hi) return 0u;
  const uint32_t up = hi == 4 ? 0xffffffffu : (1u << (8 * hi)) - 1u;
  return up & ~((1u << (8 * lo)) - 1u);
}

// One workgroup: one page of one request, keys or values (blockIdx.z), and its share of the kv heads.  A unit of
// work is 4 positions of the page x 8 dims, UNITS of them per thread, held in registers from the maximum to the
// codes, so that the input is read once.  Where a head's page has fewer units than the workgroup threads, several
// heads go side by side.  Keys leave as 8 bytes per position; values go through LDS to be turned to [hd][page] and
// leave as 16-byte pieces.  A piece that is not wholly new is merged with what the page held.
// Bound by the chain of loads (cu, slots, tokens, the page's old codes), for few tokens (64 requests of one: 8.0 us) as
// for long prompts: 21447 tokens of 8 heads of 128 in pages of 32 take 40.7 us, 3.2 of the 5.2 TB/s of a copy, with the waves
// waiting 58% of their time.  The type is settled in the kernel, so that every type pays for float32's loads: 120
// registers and four waves a SIMD (UNITS = 2: 177, two waves; 4: 282, one).  The turn's stores meet on LDS banks (rows of
// page + 16 bytes: 8 to 32 lanes of a store on one), about a tenth of the time of those prompts.
template <int HD, int UNITS>
__global__ __launch_bounds__(KV_NT) void kv_write_kernel(const WriteArgs a) {
  constexpr int CH = HD / 8;                     // 8-dim pieces of a row
  constexpr int MOST = UNITS * KV_NT / CH * 4;   // positions that the workgroup covers, of all its heads
  __shared__ int sh[5], follow;
  __shared__ float smax[8];
  __shared__ __attribute__((aligned(16))) char turn[HD * 2 * MOST];
  const int tid = threadIdx.x, page = 1 << a.psh, z = blockIdx.z;
  const Item it = find_item(a.cu, nullptr, a.B, a.tokens, blockIdx.x, 1, page, 2, sh);
  if (it.b < 0) return;
  int o0 = a.slots[it.c0];  // the request's first slot: its place within the page says where the others begin
  if (o0 < 0) {
    // its first page is not there.  For a later one, any slot of the 2 page - 1 < KV_NT tokens that can lie on it,
    // wherever pages begin, says the same; if all are negative, there is nothing to be written.
    if (it.i == 0) return;
    if (tid == 0) follow = KV_NT;
    __syncthreads();
    const int near = (it.i - 1) * page + 1;
    if (tid < min(it.n - near, 2 * page - 1) && a.slots[it.c0 + near + tid] >= 0) atomicMin(&follow, tid);
    __syncthreads();
    const int first = follow;
    if (first == KV_NT) return;
    o0 = a.slots[it.c0 + near + first] - near - first;
    __syncthreads();  // follow is written again
  }
  o0 &= page - 1;
  const int start = it.i == 0 ? it.c0 : it.c0 + it.i * page - o0;
  const int stop = min(it.c0 + it.n, it.i == 0 ? it.c0 + page - o0 : start + page);
  if (start >= stop) return;
  const int mine = tid < stop - start ? a.slots[start + tid] : 0;
  const int slot = a.slots[start];
  const int id = slot >> a.psh, o = slot & (page - 1);
  // a page after the request's first is written from its beginning
  if (slot < 0 || id >= a.num_pages || (it.i > 0 && o > 0)) return;
  // positions [o, o + count) of the page are new: the group's tokens up to the first whose slot does not follow
  // its neighbour's
  const int span = min(stop - start, page - o);
  if (tid == 0) follow = span;
  __syncthreads();
  if (tid < span && mine != slot + tid) atomicMin(&follow, tid);

  // this thread's head of those side by side, and its place within the head's units
  const int per = min((page >> 2) * CH, KV_NT);  // threads of one head: 32 to 256
  const int sub = tid / per, lt = tid % per, abreast = KV_NT / per;
  const int wide = min(per, 64);                 // lanes that reduce together
  const void* x = a.x[z];
  char* tn = turn + sub * HD * (page + 16);
  const int row = page + 16;  // bytes of a row in LDS
  for (int h0 = blockIdx.y * abreast; h0 < a.KV; h0 += gridDim.y * abreast) {
    const int h = h0 + sub;
    const bool on = h < a.KV;
    const int64_t base = (int64_t)h * a.head[z];
    float v[UNITS][4][8];
    {
      int64_t at[UNITS * 4];
      bool there[UNITS * 4];
#pragma unroll
      for (int n = 0; n < UNITS * 4; ++n) {
        const int unit = lt + n / 4 * KV_NT, j = 4 * (unit / CH) + n % 4 - o;  // token within the group
        at[n] = (int64_t)(start + j) * a.tok[z] + base + 8 * (unit % CH);
        there[n] = on && j >= 0 && j < span;
      }
      float(*out)[8] = &v[0][0];
      const int type = a.type[z];
      if (!a.vec[z]) {
        if (type == MLCV_DTYPE_F32) load_rows<MLCV_DTYPE_F32, false, UNITS * 4>(x, at, there, out);
        else if (type == MLCV_DTYPE_F16) load_rows<MLCV_DTYPE_F16, false, UNITS * 4>(x, at, there, out);
        else load_rows<MLCV_DTYPE_BF16, false, UNITS * 4>(x, at, there, out);
      } else if (type == MLCV_DTYPE_F32) {
        load_rows<MLCV_DTYPE_F32, true, UNITS * 4>(x, at, there, out);
      } else if (type == MLCV_DTYPE_F16) {
        load_rows<MLCV_DTYPE_F16, true, UNITS * 4>(x, at, there, out);
      } else {
        load_rows<MLCV_DTYPE_BF16, true, UNITS * 4>(x, at, there, out);
      }
    }
    float* scale = a.scale[z] + (size_t)id * a.KV + h;
    const float old = on && o > 0 ? load_global(scale) : 0.f;
    __syncthreads();  // the count is known; the last round's maxima and codes in LDS are used
    const int count = follow;
    float big = 0.f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = 4 * ((lt + u * KV_NT) / CH) + i - o;
        if (j < count) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float m = fabsf(v[u][i][e]);
            big = m < INFINITY ? fmaxf(big, m) : big;
          }
        }
      }
    for (int s = wide >> 1; s > 0; s >>= 1) big = fmaxf(big, __shfl_xor(big, s));
    if (tid % wide == 0) smax[tid / wide] = big;
    __syncthreads();
    for (int i = 0; i < per / wide; ++i) big = fmaxf(big, smax[sub * (per / wide) + i]);
    // big = m * 2^E, 1 <= m < 2: 448 = 1.75 * 2^8, so e = E - 8, one more where m > 1.75
    const uint32_t bits = __float_as_uint(big);
    int e = (int)(bits >> 23) - 127 - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0);
    e = e < -64 ? -64 : e;
    const float need = __uint_as_float((uint32_t)(e + 127) << 23);
    const float now = fmaxf(need, old);  // a NaN that the page held counts as nothing
    const bool grown = o > 0 && now != old;
    const float inv = 1.0f / now;        // exact where the scale is a power of two, as this kernel's are
    const float ratio = old * inv;

    uint8_t* dst = a.cache[z] + ((size_t)id * a.KV + h) * (size_t)page * HD;
    if (z == 0) {  // keys [page][HD]
      if (on) {
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
          const int unit = lt + u * KV_NT, quad = unit / CH, ch = unit % CH;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int pos = 4 * quad + i, j = pos - o;
            if (j >= 0 && j < count) {
              u2v w;
              w[0] = pack4(v[u][i][0] * inv, v[u][i][1] * inv, v[u][i][2] * inv, v[u][i][3] * inv);
              w[1] = pack4(v[u][i][4] * inv, v[u][i][5] * inv, v[u][i][6] * inv, v[u][i][7] * inv);
              *reinterpret_cast<u2v*>(dst + (size_t)pos * HD + 8 * ch) = w;
            }
          }
        }
        if (grown)
          for (int i = lt; i < o * (HD / 4); i += per) {
            uint32_t* w = reinterpret_cast<uint32_t*>(dst) + i;
            *w = rescale4(*w, ratio);
          }
      }
    } else {  // values [HD][page]
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int unit = lt + u * KV_NT, quad = unit / CH, ch = unit % CH;
        if (4 * quad < page && 4 * quad + 4 > o && 4 * quad < o + count) {
#pragma unroll
          for (int d = 0; d < 8; ++d)
            *reinterpret_cast<uint32_t*>(tn + (8 * ch + d) * row + 4 * quad) =
                pack4(v[u][0][d] * inv, v[u][1][d] * inv, v[u][2][d] * inv, v[u][3][d] * inv);
        }
      }
      __syncthreads();
      const int segs = page >> 4;
      for (int i = on ? lt : HD * segs; i < HD * segs; i += per) {
        const int d = i / segs, s = i % segs;
        const int lo = o - 16 * s, hi = o + count - 16 * s;  // new bytes of this piece: [lo, hi)
        const bool fresh = lo < 16 && hi > 0;
        if (!fresh && !(grown && lo > 0)) continue;
        u4* g = reinterpret_cast<u4*>(dst + (size_t)d * page + 16 * s);
        u4 w = fresh ? *reinterpret_cast<const u4*>(tn + d * row + 16 * s) : (u4){0, 0, 0, 0};
        if (lo > 0 || hi < 16) {
          const u4 was = *g;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint32_t fm = byte_mask(lo - 4 * q, hi - 4 * q), km = byte_mask(0, lo - 4 * q);
            const uint32_t kept = grown ? rescale4(was[q], ratio) : was[q];
            w[q] = (w[q] & fm) | (kept & km) | (was[q] & ~(fm | km));
          }
        }
        *g = w;
      }
    }
    if (on && lt == 0 && now != old) *scale = now;
  }
}

// ---- attention -------------------------------------------------------------------------------------

struct KvAttnArgs {
  const void* q;
  int64_t q_tok, q_head, o_tok, o_head;  // element strides
  const int32_t *cu, *kv_lens, *table;
  const uint8_t *kc, *vc;
  const float *ks, *vs;
  void* out;
  float *part_o, *part_ml;  // of the splits: O [items][KV][S][16][HD], (m, l) [items][KV][S][16]
  int32_t tokens, B, H, KV, grp, max_pages, num_pages, psh, causal, q_vec;
  int32_t S, span;   // splits, tiles of 64 keys per split
  float c;           // scale * log2(e)
};

template <bool BF>
struct El {
  typedef _Float16 T;
  typedef h8 V8;
};
template <>
struct El<true> {
  typedef __bf16 T;
  typedef __bf16 V8 __attribute__((ext_vector_type(8)));
};
__device__ __forceinline__ f4 mfma16(h8 a, h8 b, f4 c) { return mfma16x16x32(a, b, c); }
__device__ __forceinline__ f4 mfma16(El<true>::V8 a, El<true>::V8 b, f4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// 8 codes as values of either type, exactly (both types hold every e4m3 value)
template <bool BF>
__device__ __forceinline__ typename El<BF>::V8 widen8(uint32_t lo, uint32_t hi) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  u4 w;
  if constexpr (BF) {
    w[0] = __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
    w[1] = __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
    w[2] = __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
    w[3] = __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
  } else {
    w[0] = __builtin_bit_cast(uint32_t, (h2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
    w[1] = __builtin_bit_cast(uint32_t, (h2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
    w[2] = __builtin_bit_cast(uint32_t, (h2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
    w[3] = __builtin_bit_cast(uint32_t, (h2)__builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
  }
  return __builtin_bit_cast(typename El<BF>::V8, w);
}

// keys that any row of [row0, row0 + rows) of a request sees
__device__ __forceinline__ int last_limit(const KvAttnArgs& a, const Item& it, int kv_len, int row0, int rt) {
  const int rows = it.n * a.grp, last = min(row0 + rt, rows) - 1;
  return a.causal ? kv_len - it.n + last / a.grp + 1 : kv_len;
}

// Global -> LDS DMA, one address per lane, to lds + 16 (4) lane.  In assembly: the compiler would wait for every DMA in
// flight before each read of LDS.  It returns nothing into registers; the loop waits for it.
__device__ __forceinline__ uint32_t lds_at(const char* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds;
#else
  return 0;
#endif
}
__device__ __forceinline__ void dma16(const void* base, int off, const char* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds_at(lds)), "v"(off), "s"(base)
               : "memory", "m0");
#endif
}
__device__ __forceinline__ void dma16(const void* p, const char* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds_at(lds)), "v"(p)
               : "memory", "m0");
#endif
}
__device__ __forceinline__ void dma4(const void* p, const char* lds) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" ::"s"(lds_at(lds)), "v"(p)
               : "memory", "m0");
#endif
}
// all but the last N DMA instructions have arrived
template <int N>
__device__ __forceinline__ void wait_dma() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
#endif
}
// LDS reads have arrived: their memory can be written again
__device__ __forceinline__ void wait_lds() {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#endif
}
// a value that was loaded is there
template <class T>
__device__ __forceinline__ void wait_value(T& v) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("" : "+v"(v));
#endif
}

// Piece p (16 bytes) of key row r lies at piece p ^ k_turn(r): the 16 rows that 16 lanes read at once fall into
// distinct pieces of a 256-byte bank line.  A field of r's bits, so that k_turn(a | b) = k_turn(a) ^ k_turn(b) for
// a & b = 0.
template <int HD>
__device__ constexpr int k_turn(int r) {
  return HD == 256 ? (r & 3) | (r >> 3 & 3) << 2 : HD == 128 ? (r >> 1 & 1) | (r >> 4 & 3) << 1 : r >> 4 & 3;
}

// Row r of a request is token r / grp of its n new tokens and head h * grp + r % grp: the query heads of a kv
// head share its keys.  A workgroup (NW waves) takes 16 such rows and one split of the keys; its waves take tiles
// of TK keys in turn, each with its own running maximum and sum, and meet in LDS at the end.
//
// No data is shuffled between lanes.  S^T = K . Q^T and O^T = V^T . P^T on
// v_mfma_f32_16x16x32: with lane = 16 g + r, S^T puts keys 4 g .. 4 g + 3 of each 16-key sub-tile and query row
// r into a lane, and the second product wants 8 keys of row r in it.  Both contractions may run in any order,
// so the order is chosen by the loads: with PL = TK / 4, sub-tile s's row 4 g + i is key PL g + 4 s + i of the
// tile; a lane then owns PL consecutive keys, which are PL contiguous bytes of the value page, lie in one page
// and have one scale of each side.  Dims likewise: a lane's 16 key bytes are two steps of the first contraction.
// A lane's neighbours hold other rows of the page, so that loads from the page into these registers would take a
// cache access per lane (1070 of a tile of 16 KB, which bound the many rows of action suffixes).  Each wave therefore
// fetches its tiles by DMA into a part of LDS of its own, lanes side by side along the rows (eight suffixes of 50
// tokens 25.4 -> 18.6 us), and reads the operands from there.  No barrier: as soon as a tile's keys (values) are in
// registers, the next tile's follow into the same place; its page numbers come a tile earlier.
//
// Bound by HBM: one token each of 96 requests that hold 4096, 8 kv heads of 128, takes 147 us (5.5 TB/s), of 48
// requests 84 (4.8); with lengths from 1 to 4096 the last workgroups run with the GPU half empty (48 requests, 64 us, 3.7
// TB/s).  More bytes in flight bring nothing there: two tiles of loads ahead 67 us, three waves a SIMD 79 and
// more (both before the DMA).
// Bound by the latency of a tile at few requests: 969 tokens of one kv head of 256, 6.8 us and 3.3 for the join.
//
// The value scale is folded into the weights before they are rounded to fp16: with x = logit * log2(e) the
// running maximum is that of x + log2(scale_v), so that w = 2^(x - m) * scale_v stays within [0, 2^12] whatever
// the pages' scales are; the sum of 2^(x - m) is kept in float32.  Weights and values are fp16 for either type
// of query (an e4m3 value is exact in it).  2^12 of headroom keeps weights down to 2^-26 of the largest above
// fp16's subnormals.
//
// A key or page that a row does not see has weight 0, which a NaN code behind it would turn into NaN.  In a tile
// that not every row sees whole such codes are cleared, and at the end the rows that do see one are set to NaN.
template <bool BF, int HD, int TK, int NW>
__global__ __launch_bounds__(64 * NW, 2) void kv_attn_kernel(const KvAttnArgs a) {
  typedef typename El<BF>::T T;
  typedef typename El<BF>::V8 V8;
  constexpr int NJ = HD / 64, ND = HD / 16, SUB = TK / 16, PL = TK / 4, VW = PL / 4;
  typedef uint32_t VWords __attribute__((ext_vector_type(VW)));
  __shared__ int sh[5];
  __shared__ float sm[NW][KV_RT], sl[NW][KV_RT];
  constexpr int HALF = TK * HD, AREA = 2 * HALF + 512, MEET = KV_RT * (HD + 4) * 4;  // bytes of a wave
  __shared__ __attribute__((aligned(1024))) char lds[NW * (AREA > MEET ? AREA : MEET)];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r16 = lane & 15, g = lane >> 4;
  const int item = blockIdx.x / (a.KV * a.S), rest = blockIdx.x % (a.KV * a.S);
  const int h = rest % a.KV, split = rest / a.KV;
  const Item it = find_item(a.cu, a.kv_lens, a.B, a.tokens, item, a.grp, KV_RT, 1, sh);
  if (it.b < 0) return;
  const int rows = it.n * a.grp, row0 = it.i * KV_RT, page = 1 << a.psh;
  if (row0 >= rows) return;
  const int kv_len = clamp_i(it.len, 0, a.max_pages << a.psh);
  const int most = last_limit(a, it, kv_len, row0, KV_RT);
  const int first = a.causal ? kv_len - it.n + row0 / a.grp + 1 : kv_len;  // keys that every row sees
  const int t_begin = split * a.span * (64 / TK), tiles = (most + TK - 1) / TK;
  const int t_end = split == a.S - 1 ? tiles : min(tiles, t_begin + a.span * (64 / TK));
  if (split > 0 && t_begin >= tiles) return;

  const int32_t* table = a.table + (size_t)it.b * a.max_pages;
  // A wave's part of LDS: its tile's keys, values, page numbers and scales.  A tile is NG groups of 16 keys, each in
  // one page.
  constexpr int NG = TK / 16, NI = HALF / 1024, RPI = 1024 / HD;  // DMA instructions, key rows of one
  char* const my_k = lds + w * AREA;
  char* const my_v = my_k + HALF;
  const int* const my_ids = reinterpret_cast<const int*>(my_v + HALF);
  const float* const my_scales = reinterpret_cast<const float*>(my_v + HALF + 256);
  const int vg = (lane & (NG - 1)) ^ (g & (NG - 1));  // the group whose numbers, scales and values this lane fetches
  const int ko = lane / (HD / 16) * HD + ((lane % (HD / 16)) ^ k_turn<HD>(lane / (HD / 16))) * 16;
  int ids[NG], id_mine = 0, id_own = 0;  // pages of the groups, of vg, of the lane's own keys; -1: none to be read
  auto fetch_ids = [&](int t) {
    t = min(t, t_end - 1);
    dma4(table + min((TK * t + 16 * vg) >> a.psh, a.max_pages - 1), reinterpret_cast<const char*>(my_ids));
  };
  auto read_ids = [&]() {
    auto sound = [&](int id) { return id >= 0 && id < a.num_pages ? id : -1; };
#pragma unroll
    for (int i = 0; i < NG; ++i) ids[i] = __builtin_amdgcn_readfirstlane(sound(my_ids[i]));  // lane i < NG has vg = i
    id_mine = sound(my_ids[lane]);
    id_own = sound(my_ids[PL * g >> 4]);
  };
  auto load_scales = [&]() {
    dma4((lane < 32 ? a.ks : a.vs) + (size_t)max(id_mine, 0) * a.KV + h, reinterpret_cast<const char*>(my_scales));
  };
  auto load_keys = [&](int t) {
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      const int grp = i * RPI / 16, pos = (TK * t + 16 * grp) & (page - 1);
      const uint8_t* p = a.kc + (((size_t)max(ids[grp], 0) * a.KV + h) * page + pos + (i * RPI & 15)) * HD;
      dma16(p, ko ^ 16 * k_turn<HD>(i * RPI), my_k + 1024 * i);
    }
  };
  auto load_values = [&](int t) {
    const uint8_t* p = a.vc + (((size_t)max(id_mine, 0) * a.KV + h) * HD + lane / NG) * page +
                       ((TK * t + 16 * vg) & (page - 1));
#pragma unroll
    for (int i = 0; i < NI; ++i) dma16(p + (size_t)(64 / NG * i) * page, my_v + 1024 * i);
  };
  int t = t_begin + w;
  if (t < t_end) fetch_ids(t);

  // the query operand: row r16, dims 64 j + 16 g + 8 s .. + 7 for step 2 j + s
  V8 q[2 * NJ];
  const int qrow = min(row0 + r16, rows - 1), qtok = qrow / a.grp;
  const int lim = a.causal ? kv_len - it.n + qtok + 1 : kv_len;  // keys that the row sees
  {
    const T* p = reinterpret_cast<const T*>(a.q) + (int64_t)(it.c0 + qtok) * a.q_tok +
                 (int64_t)(h * a.grp + qrow - qtok * a.grp) * a.q_head + 16 * g;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        if (a.q_vec) {
          q[2 * j + s] = load_global(reinterpret_cast<const V8*>(p + 64 * j + 8 * s));
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) q[2 * j + s][e] = load_global(p + 64 * j + 8 * s + e);
        }
      }
  }
#pragma unroll
  for (int i = 0; i < 2 * NJ; ++i) wait_value(q[i]);  // no load of the compiler's is in flight in the loop
  int own_page = 0;  // of the tile at hand
  if (t < t_end) {
    wait_dma<0>();
    read_ids();
    own_page = id_own;
    wait_lds();
    fetch_ids(t + NW);
    load_scales();
    load_keys(t);
    load_values(t);
  }
  f4 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = (f4){0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  bool poison = false;  // a NaN code was cleared
  for (; t < t_end; t += NW) {
    const int pv = TK * t + PL * g;
    const bool more = t + NW < t_end;
    wait_dma<NI>();  // in flight behind it: the values
    u4 kr[SUB][NJ];
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int row = PL * (r16 >> 2) + 4 * s + (r16 & 3);
        kr[s][j] = *reinterpret_cast<const u4*>(my_k + row * HD + (((4 * j + g) ^ k_turn<HD>(row)) * 16));
      }
    const int now = own_page;
    const int own = now < 0 ? 0 : clamp_i(kv_len - pv, 0, PL);  // the lane's keys that are the request's
    // the value scale of a page that holds none of them may be anything, NaN too: it would outlast the weight of 0
    const float vscale = my_scales[32 + ((PL * g >> 4) ^ (2 & (NG - 1)))];
    const float skc = my_scales[PL * g >> 4] * a.c, svc = own > 0 ? vscale : 0.f;
    if (more) {
      read_ids();
      own_page = id_own;
      wait_lds();
      fetch_ids(t + 2 * NW);
      load_scales();
      load_keys(t + NW);
    }
    f4 x[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      x[s] = (f4){0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        x[s] = mfma16(widen8<BF>(kr[s][j][0], kr[s][j][1]), q[2 * j], x[s]);
        x[s] = mfma16(widen8<BF>(kr[s][j][2], kr[s][j][3]), q[2 * j + 1], x[s]);
      }
    }
    const bool edge = TK * t + TK > first || __any(now < 0);
    const float lsv = __builtin_amdgcn_logf(fmaxf(svc, 0x1p-64f)) - 12.0f;
    h8 p[PL / 8];
    float top = -INFINITY;
    const int see = min(lim - pv, own);  // keys pv .. pv + see - 1 are visible
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v = x[s][i] * skc;
        if (edge && 4 * s + i >= see) v = -INFINITY;
        x[s][i] = v;
        top = fmaxf(top, v);
      }
    top = xor_max_16_32(top + lsv);
    const float mn = fmaxf(m, top), mu = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int s = 0; s < SUB; ++s)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(x[s][i] - mu);
        sum += e;
        p[s >> 1][4 * (s & 1) + i] = (_Float16)(e * svc);
      }
    l = l * alpha + sum;
    if (more) wait_dma<NI + 2>();  // behind the values: the next tile's keys, scales and page numbers
    else wait_dma<0>();
    VWords vr[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int dim = 16 * d + r16, piece = NG * dim + ((PL * g >> 4) ^ (dim * NG >> 4 & (NG - 1)));
      vr[d] = *reinterpret_cast<const VWords*>(my_v + 16 * piece + (PL * g & 15));
    }
    if (more) {
      wait_lds();
      load_values(t + NW);
    }
    if (edge) {
      bool nan = false;
#pragma unroll
      for (int i = 0; i < VW; ++i) {
        const uint32_t keep = byte_mask(0, own - 4 * i);
#pragma unroll
        for (int d = 0; d < ND; ++d) {
          vr[d][i] &= keep;
          // bytes that are NaN codes (0x7f or 0xff) to zero
          const uint32_t bad = ((((vr[d][i] & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7) * 0xffu;
          nan = nan || bad;
          vr[d][i] &= ~bad;
        }
      }
      poison = poison || __any(nan);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      o[d] *= alpha;
#pragma unroll
      for (int i = 0; i < PL / 8; ++i) o[d] = mfma16(widen8<false>(vr[d][2 * i], vr[d][2 * i + 1]), p[i], o[d]);
    }
  }
  if (poison)  // the tiles of this wave that hold keys from `first` on, or pages that are not there
    for (t = t_begin + w; t < t_end; t += NW) {
      const int pos = TK * t + PL * g, pg = pos >> a.psh;
      int idv = pg < a.max_pages ? load_global(table + pg) : -1;
      if (idv >= a.num_pages) idv = -1;
      if (!(TK * t + TK > first || __any(idv < 0))) continue;
      VWords vr[ND];
      const uint8_t* p = a.vc + (((size_t)max(idv, 0) * a.KV + h) * HD + r16) * page + (pos & (page - 1));
#pragma unroll
      for (int d = 0; d < ND; ++d) vr[d] = load_global(reinterpret_cast<const VWords*>(p + (size_t)16 * d * page));
      const int own = idv < 0 ? 0 : clamp_i(kv_len - pos, 0, PL);
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        int at = 0x7fffffff;  // the first of the lane's keys whose value at dim 16 d + r16 is NaN
        for (int i = PL - 1; i >= 0; --i)
          if (i < own && (vr[d][i >> 2] >> (8 * (i & 3)) & 0x7f) == 0x7f) at = TK * t + PL * g + i;
        at = min(at, __shfl_xor(at, 16));
        at = min(at, __shfl_xor(at, 32));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = __shfl(at, 4 * g + i);  // of dim 16 d + 4 g + i
          if (key < lim) o[d][i] = NAN;
        }
      }
    }

  const size_t part0 = (((size_t)item * a.KV + h) * a.S + split) * KV_RT;  // of the partial results' rows
  // ---- the waves meet ------------------------------------------------------------------------------
  float (*so)[KV_RT][HD + 4] = reinterpret_cast<float (*)[KV_RT][HD + 4]>(lds);  // once every wave is through its tiles
  l = xor_sum_16_32(l);
  if (g == 0) {
    sm[w][r16] = m;
    sl[w][r16] = l;
  }
  __syncthreads();
  float f;  // this wave's share of the workgroup's sum
  {
    float mx = sm[0][r16];
#pragma unroll
    for (int i = 1; i < NW; ++i) mx = fmaxf(mx, sm[i][r16]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    f = __builtin_amdgcn_exp2f(m - mu);
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) sum += sl[i][r16] * __builtin_amdgcn_exp2f(sm[i][r16] - mu);
    if (a.S > 1) {
      if (w == 0 && g == 0 && row0 + r16 < rows) reinterpret_cast<f2*>(a.part_ml)[part0 + r16] = (f2){mx, sum};
    } else {
      f = sum > 0.f ? f / sum : sum == 0.f ? 0.f : sum;  // nothing visible: zeros; NaN stays
    }
  }
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    *reinterpret_cast<f4*>(&so[w][r16][16 * d + 4 * g]) = o[d] * f;  // a NaN stays, even under a share of zero
  }
  __syncthreads();
#pragma unroll
  for (int i = tid; i < KV_RT * HD / 4; i += 64 * NW) {
    const int row = i / (HD / 4), d = 4 * (i % (HD / 4));
    if (row0 + row >= rows) continue;
    f4 v = *reinterpret_cast<const f4*>(&so[0][row][d]);
#pragma unroll
    for (int k = 1; k < NW; ++k) v += *reinterpret_cast<const f4*>(&so[k][row][d]);
    if (a.S > 1) {
      *reinterpret_cast<f4*>(a.part_o + (part0 + row) * HD + d) = v;
    } else {
      const int rr = row0 + row, tok = rr / a.grp;
      T* dst = reinterpret_cast<T*>(a.out) + (int64_t)(it.c0 + tok) * a.o_tok +
               (int64_t)(h * a.grp + rr - tok * a.grp) * a.o_head + d;
#pragma unroll
      for (int k = 0; k < 4; ++k) dst[k] = (T)v[k];
    }
  }
}

// The splits of one row: the partial results under their common maximum.  W waves take DC dims of one row, DC / 4
// lanes one split of it at a time.  Few splits: a wave takes a whole row.  Many: a workgroup takes 64 dims of one, so
// that the reads spread over the GPU (two rows of 8 heads and 128 splits: 5.2 us, with whole rows 8.1).
template <bool BF, int HD, int W, int DC>
__global__ __launch_bounds__(KV_NT) void kv_join_kernel(const KvAttnArgs a) {
  typedef typename El<BF>::T T;
  constexpr int LQ = DC / 4, NG = 64 * W / LQ, NC = HD / DC;  // lanes of a split, splits at once, pieces of a row
  __shared__ __attribute__((aligned(16))) float so[W][DC];
  __shared__ float sl[W];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const long long at = W == 1 ? (long long)blockIdx.x * 4 + w : blockIdx.x / NC;
  const int token = (int)(at / a.H), head = (int)(at % a.H), h = head / a.grp;
  // the token's request
  int b = -1, c0 = 0, n = 0, kv_len = 0;
  for (int b0 = 0; b0 < a.B && b < 0; b0 += 64) {
    const int i = min(b0 + lane, a.B - 1);
    const int x = clamp_i(a.cu[i], 0, a.tokens), y = clamp_i(a.cu[i + 1], 0, a.tokens), len = a.kv_lens[i];
    const unsigned long long hit = __ballot(x <= token && token < y);
    if (hit) {
      const int src = __ffsll(hit) - 1;
      b = min(b0 + src, a.B - 1);
      c0 = __builtin_amdgcn_readlane(x, src);
      n = __builtin_amdgcn_readlane(y, src) - c0;
      kv_len = clamp_i(__builtin_amdgcn_readlane(len, src), 0, a.max_pages << a.psh);
    }
  }
  if (token >= a.tokens || b < 0) return;
  Item it;
  it.n = n;
  const int rr = (token - c0) * a.grp + head - h * a.grp, tile = rr / KV_RT, row = rr % KV_RT;
  const long long item = (long long)c0 * a.grp / KV_RT + b + tile;
  const int tiles = (last_limit(a, it, kv_len, tile * KV_RT, KV_RT) + 63) >> 6;
  const int splits = clamp_i((tiles + a.span - 1) / a.span, 1, a.S);  // splits that there are
  const size_t p0 = ((size_t)item * a.KV + h) * a.S * KV_RT + row;
  const f2* ml = reinterpret_cast<const f2*>(a.part_ml) + p0;
  float mx = -INFINITY;
  for (int s = lane; s < splits; s += 64) mx = fmaxf(mx, load_global(ml + (size_t)s * KV_RT)[0]);
#pragma unroll
  for (int s = 32; s > 0; s >>= 1) mx = fmaxf(mx, __shfl_xor(mx, s));
  const float mu = mx == -INFINITY ? 0.f : mx;
  const int gq = (W == 1 ? lane : tid) / LQ, d = 4 * (lane % LQ), d0 = W == 1 ? 0 : (int)(blockIdx.x % NC) * DC;
  f4 v = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
#pragma unroll 4
  for (int s = gq; s < splits; s += NG) {
    const f2 e = load_global(ml + (size_t)s * KV_RT);
    const float f = __builtin_amdgcn_exp2f(e[0] - mu);
    const f4 u = load_global(reinterpret_cast<const f4*>(a.part_o + (p0 + (size_t)s * KV_RT) * HD + d0 + d));
    v += u * f;
    sum += e[1] * f;
  }
#pragma unroll
  for (int s = LQ; s < 64; s <<= 1) {  // the splits within a wave
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] += __shfl_xor(v[i], s);
    sum += __shfl_xor(sum, s);
  }
  if constexpr (W > 1) {
    if (lane < LQ) *reinterpret_cast<f4*>(&so[w][d]) = v;
    if (lane == 0) sl[w] = sum;
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int k = 1; k < W; ++k) {
      v += *reinterpret_cast<const f4*>(&so[k][d]);
      sum += sl[k];
    }
  }
  if (lane >= LQ) return;
  const float f = sum > 0.f ? 1.0f / sum : sum == 0.f ? 0.f : sum;
  T* dst = reinterpret_cast<T*>(a.out) + (int64_t)token * a.o_tok + (int64_t)head * a.o_head + d0 + d;
#pragma unroll
  for (int k = 0; k < 4; ++k) dst[k] = (T)(v[k] * f);
}

// How an attention call is cut: splits of the keys, from what the host knows.
struct KvAttnPlan {
  int S, span;
  bool wide;         // eight waves per workgroup
  long long items;  // tiles of 16 rows, at most
  size_t o_floats, bytes;
};
KvAttnPlan kv_attn_plan(int tokens, int B, int H, int KV, int hd, int max_kv) {
  KvAttnPlan p;
  const long long rows = (long long)tokens * (H / KV);
  p.items = rows / KV_RT + B;
  const long long busy = std::max({1ll, (rows + KV_RT - 1) / KV_RT, (long long)std::min(B, tokens)}) * KV;
  const int tiles = std::max(1, max_kv / 64 + (max_kv % 64 != 0));
  // What costs least: four or eight waves per workgroup, or splits, as many as make one or two workgroups per CU.  In
  // rounds of four waves' tiles a workgroup costs two more to begin with, all of it half as much again where eight
  // waves share a CU, and the join's launch 2.5 and its reads.  Heads of 256: 8 suffixes of 50 tokens over 1018 take
  // 18.7 us with four waves, 17.1 with eight, two suffixes 13.6 with four splits, 16.6 with eight and 16.2 with none;
  // 200 requests of 4096 tokens 126 with four waves, 80 with eight, 95 with two splits; 128 of them 67 with four
  // splits, 70 with none.  Heads of 128: 32 requests 43.6 with four waves, 38.4 with eight (24 of them 34.3 and 35.2);
  // 16 of them 33 with eight, 28 with four splits.  One workgroup per CU was never best there (8 requests 21.5, two
  // 17.4).  Above 256 workgroups eight waves are slower: 16 suffixes 31.7 us (26.2), 500 requests of up to 500 tokens,
  // heads of 64, 34 (25); though 96 long ones 58 (63).
  const int round = hd == 256 ? 2 : 4;  // tiles of 64 keys that four waves take at once
  auto cut = [&](long long n) {
    const long long want = std::max(1ll, std::min<long long>(n / busy, (tiles + round - 1) / round));
    return (int)((tiles + want - 1) / want);
  };
  auto cost = [&](int span, bool wide) {
    const long long S = (tiles + span - 1) / span, groups = busy * S, at_once = wide ? 2 * round : round;
    return (2 + (span + at_once - 1) / at_once) * (wide || groups > 256 ? 1.5 : 1.0) +
           (S > 1 ? 2.5 + groups * hd / 65536.0 : 0.0);
  };
  p.span = tiles;
  p.wide = busy <= 256 && cost(tiles, true) <= cost(tiles, false);
  for (const int n : {512, 256})
    if ((n == 512 || hd == 256) && cost(cut(n), false) < cost(p.span, p.wide)) {
      p.span = cut(n);
      p.wide = false;
    }
  p.S = (tiles + p.span - 1) / p.span;
  const size_t parts = (size_t)p.items * KV * p.S * KV_RT;
  p.o_floats = p.S > 1 ? parts * hd : 0;
  p.bytes = p.S > 1 ? (p.o_floats + parts * 2) * sizeof(float) : 0;
  return p;
}

template <int HD>
int kv_write_launch(const WriteArgs& a, hipStream_t st) {
  const int page = 1 << a.psh;
  constexpr int PER = 4 * KV_NT / (HD / 8);  // positions that one unit per thread covers
  // the heads over workgroups while there are fewer than 4096 of them, then in turn within one, whose first loads then
  // serve several heads: 21447 tokens of 8 heads of 128 in 40.7 us, with a workgroup for each round of heads 43.1
  const long long pages = a.tokens / page + a.B, abreast = std::max(1, PER / page);
  const long long groups = std::max(1ll, std::min((a.KV + abreast - 1) / abreast, 4096 / (2 * pages)));
  const dim3 grid(a.tokens / page + 2 * a.B, (unsigned)groups, 2);
  if (page <= PER) kv_write_kernel<HD, 1><<<grid, KV_NT, 0, st>>>(a);
  else if (page <= 2 * PER) kv_write_kernel<HD, (PER >= 128 ? 1 : 2)><<<grid, KV_NT, 0, st>>>(a);
  else kv_write_kernel<HD, (PER >= 64 ? 1 : 4)><<<grid, KV_NT, 0, st>>>(a);
  MLCV_HIP(hipGetLastError());
  return 0;
}

template <bool BF, int HD>
int kv_attn_launch(const KvAttnArgs& a, const KvAttnPlan& p, hipStream_t st) {
  const unsigned grid = (unsigned)(p.items * a.KV * p.S);
  // tiles of 32 keys at head_dim 256: two waves fit a SIMD (131072 tokens 52 -> 38 us)
  constexpr int TK = HD == 256 ? 32 : 64;
  if (p.wide) kv_attn_kernel<BF, HD, TK, 8><<<grid, 512, 0, st>>>(a);
  else kv_attn_kernel<BF, HD, TK, 4><<<grid, 256, 0, st>>>(a);
  MLCV_HIP(hipGetLastError());
  if (p.S > 1) {
    const long long rows = (long long)a.tokens * a.H;
    if (p.S <= 16) kv_join_kernel<BF, HD, 1, HD><<<(unsigned)((rows + 3) / 4), KV_NT, 0, st>>>(a);
    else kv_join_kernel<BF, HD, 4, 64><<<(unsigned)(rows * (HD / 64)), KV_NT, 0, st>>>(a);
    MLCV_HIP(hipGetLastError());
  }
  return 0;
}

}  // namespace
}  // namespace mlcv

using namespace mlcv;

extern "C" {

int mlcv_kv_plan_counted(const int32_t* past_lens, const int32_t* new_lens, int32_t B, const int32_t* free_pages,
                         int32_t n_free, const int32_t* free_count, int32_t num_pages, int32_t page,
                         int32_t* block_table, int32_t max_pages, int32_t* cu_seqlens, int32_t* kv_lens,
                         int32_t* slot_map, int32_t tokens, int32_t* status, void* stream) {
  MLCV_REQUIRE(B >= 0 && n_free >= 0 && num_pages >= 0 && max_pages >= 0 && tokens >= 0, "negative size");
  MLCV_REQUIRE(cu_seqlens && status, "null output");
  MLCV_REQUIRE(B == 0 || (past_lens && new_lens && kv_lens && (block_table || max_pages == 0)), "null request array");
  MLCV_REQUIRE(n_free == 0 || free_pages, "null free_pages");
  MLCV_REQUIRE(tokens == 0 || slot_map, "null slot_map");
  MLCV_REQUIRE(kv_page_ok(page), "page must be 16, 32, 64 or 128");
  MLCV_REQUIRE(B <= KV_MAX_REQ, "more than 4096 requests");
  MLCV_REQUIRE((int64_t)num_pages * page <= KV_MOST && (int64_t)max_pages * page <= KV_MOST,
               "more than 2^31 - 256 slots");
  // every workgroup reads the lengths, one writes kv_lens: a plan written over them would be read half new
  const Ints arrays[] = {{block_table, (int64_t)B * max_pages}, {cu_seqlens, (int64_t)B + 1}, {kv_lens, B}, {slot_map, tokens},
                         {status, 2}, {past_lens, B}, {new_lens, B}, {free_pages, n_free},
                         {free_count, free_count ? 1 : 0}};
  MLCV_REQUIRE(!overlap(arrays, 5, 9), "outputs overlap the inputs or one another");
  PlanArgs a{past_lens, new_lens, free_pages, free_count, block_table, cu_seqlens, kv_lens, slot_map, status, B, n_free,
             num_pages, log2_of(page), max_pages, tokens, 0};
  a.slot_blocks = std::max(1, (int)(((int64_t)tokens + 4 * KV_NT - 1) / (4 * KV_NT)));
  // a request takes at most new / page + 1 pages
  const int64_t pages = std::min<int64_t>(n_free, (int64_t)tokens / page + B);
  const unsigned grid = (unsigned)(a.slot_blocks + (pages + KV_NT - 1) / KV_NT);
  kv_plan_kernel<<<grid, KV_NT, (size_t)2 * (B + 1) * sizeof(int), reinterpret_cast<hipStream_t>(stream)>>>(a);
  MLCV_HIP(hipGetLastError());
  return 0;
}

int mlcv_kv_plan(const int32_t* past_lens, const int32_t* new_lens, int32_t B, const int32_t* free_pages,
                 int32_t n_free, int32_t num_pages, int32_t page, int32_t* block_table, int32_t max_pages,
                 int32_t* cu_seqlens, int32_t* kv_lens, int32_t* slot_map, int32_t tokens, int32_t* status,
                 void* stream) {
  return mlcv_kv_plan_counted(past_lens, new_lens, B, free_pages, n_free, nullptr, num_pages, page, block_table,
                              max_pages, cu_seqlens, kv_lens, slot_map, tokens, status, stream);
}

int mlcv_kv_write(const void* k, int32_t k_dtype, int64_t k_tok, int64_t k_head, const void* v, int32_t v_dtype,
                  int64_t v_tok, int64_t v_head, int32_t tokens, const int32_t* cu_seqlens, int32_t B,
                  const int32_t* slot_map, void* k_cache, float* k_scale, void* v_cache, float* v_scale,
                  int32_t num_pages, int32_t page, int32_t KV, int32_t hd, void* stream) {
  MLCV_REQUIRE(tokens >= 0 && B >= 0 && num_pages >= 0 && KV > 0, "bad size");
  if (tokens == 0 || B == 0 || num_pages == 0) return 0;
  MLCV_REQUIRE(k && v && cu_seqlens && slot_map && k_cache && k_scale && v_cache && v_scale, "null pointer");
  auto type_ok = [](int t) { return t == MLCV_DTYPE_F16 || t == MLCV_DTYPE_F32 || t == MLCV_DTYPE_BF16; };
  MLCV_REQUIRE(type_ok(k_dtype) && type_ok(v_dtype), "keys and values are float16, bfloat16 or float32");
  MLCV_REQUIRE(kv_page_ok(page), "page must be 16, 32, 64 or 128");
  MLCV_REQUIRE(kv_hd_ok(hd), "head_dim must be 64, 128 or 256");
  MLCV_REQUIRE(KV <= 65535, "more than 65535 kv heads");
  MLCV_REQUIRE((int64_t)num_pages * page <= KV_MOST, "more than 2^31 - 256 slots");
  MLCV_REQUIRE(tokens <= KV_MOST, "more than 2^31 - 256 tokens");
  MLCV_REQUIRE((int64_t)tokens / page + 2 * (int64_t)B <= UINT32_MAX / KV_NT, "too many requests");
  MLCV_REQUIRE(aligned16(k_cache) && aligned16(v_cache), "the cache must be 16-byte aligned");
  WriteArgs a{};
  a.x[0] = k;
  a.x[1] = v;
  a.tok[0] = k_tok;
  a.tok[1] = v_tok;
  a.head[0] = k_head;
  a.head[1] = v_head;
  a.cache[0] = static_cast<uint8_t*>(k_cache);
  a.cache[1] = static_cast<uint8_t*>(v_cache);
  a.scale[0] = k_scale;
  a.scale[1] = v_scale;
  a.cu = cu_seqlens;
  a.slots = slot_map;
  a.type[0] = k_dtype;
  a.type[1] = v_dtype;
  for (int z = 0; z < 2; ++z) {
    const int per = a.type[z] == MLCV_DTYPE_F32 ? 4 : 8;  // elements of 16 bytes
    a.vec[z] = aligned16(a.x[z]) && a.tok[z] % per == 0 && a.head[z] % per == 0;
  }
  a.tokens = tokens;
  a.B = B;
  a.num_pages = num_pages;
  a.psh = log2_of(page);
  a.KV = KV;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return hd == 64 ? kv_write_launch<64>(a, st) : hd == 128 ? kv_write_launch<128>(a, st) : kv_write_launch<256>(a, st);
}

static int kv_attn_sizes_ok(int32_t tokens, int32_t B, int32_t H, int32_t KV, int32_t hd, int32_t max_kv) {
  MLCV_REQUIRE(tokens >= 0 && B >= 0 && max_kv >= 0, "negative size");
  MLCV_REQUIRE(H > 0 && KV > 0 && H % KV == 0, "query heads must be a multiple of the kv heads");
  MLCV_REQUIRE(kv_hd_ok(hd), "head_dim must be 64, 128 or 256");
  MLCV_REQUIRE((int64_t)tokens * (H / KV) <= KV_MOST, "more than 2^31 - 256 query rows of a kv head");
  const KvAttnPlan p = kv_attn_plan(tokens, std::max(B, 1), H, KV, hd, max_kv);
  // a launch holds less than 2^32 threads
  MLCV_REQUIRE(p.items * KV * p.S <= UINT32_MAX / (p.wide ? 512 : 256) &&
                   (p.S == 1 || (int64_t)tokens * H * (hd / 64) <= UINT32_MAX / KV_NT), "too many workgroups");
  return 0;
}

int mlcv_kv_attention_workspace(int32_t tokens, int32_t B, int32_t H, int32_t KV, int32_t hd, int32_t max_kv,
                                size_t* bytes) {
  MLCV_REQUIRE(bytes, "null pointer");
  MLCV_TRY(kv_attn_sizes_ok(tokens, B, H, KV, hd, max_kv));
  *bytes = tokens == 0 || B == 0 ? 0 : kv_attn_plan(tokens, B, H, KV, hd, max_kv).bytes;
  return 0;
}

int mlcv_kv_attention_plan(int32_t tokens, int32_t B, int32_t H, int32_t KV, int32_t hd, int32_t max_kv, int32_t* splits,
                           int32_t* waves) {
  MLCV_REQUIRE(splits && waves, "null pointer");
  MLCV_TRY(kv_attn_sizes_ok(tokens, B, H, KV, hd, max_kv));
  const KvAttnPlan p = kv_attn_plan(tokens, std::max(B, 1), H, KV, hd, max_kv);
  *splits = p.S;
  *waves = p.wide ? 8 : 4;
  return 0;
}

int mlcv_kv_attention(const void* q, int32_t dtype, int64_t q_tok, int64_t q_head, int32_t tokens,
                      const int32_t* cu_seqlens, int32_t B, const int32_t* kv_lens, const int32_t* block_table,
                      int32_t max_pages, const void* k_cache, const float* k_scale, const void* v_cache,
                      const float* v_scale, int32_t num_pages, int32_t page, int32_t H, int32_t KV, int32_t hd,
                      float scale, int32_t causal, int32_t max_kv, void* out, int64_t o_tok, int64_t o_head,
                      void* workspace, size_t workspace_bytes, void* stream) {
  MLCV_REQUIRE(dtype == MLCV_DTYPE_F16 || dtype == MLCV_DTYPE_BF16, "queries are float16 or bfloat16");
  MLCV_TRY(kv_attn_sizes_ok(tokens, B, H, KV, hd, max_kv));
  MLCV_REQUIRE(kv_page_ok(page), "page must be 16, 32, 64 or 128");
  MLCV_REQUIRE(num_pages >= 0 && max_pages >= 0 && (int64_t)num_pages * page <= KV_MOST &&
                   (int64_t)max_pages * page <= KV_MOST, "more than 2^31 - 256 slots");
  MLCV_REQUIRE(scale > 0.f && scale * LOG2E < INFINITY, "scale must be positive and below 2.3e38");
  if (tokens == 0 || B == 0) return 0;
  MLCV_REQUIRE(q && cu_seqlens && kv_lens && out, "null pointer");
  MLCV_REQUIRE(max_pages == 0 || num_pages == 0 || (block_table && k_cache && k_scale && v_cache && v_scale),
               "null cache");
  MLCV_REQUIRE(aligned16(k_cache) && aligned16(v_cache), "the cache must be 16-byte aligned");
  MLCV_REQUIRE(rows_apart(tokens, o_tok, H, o_head, hd), "rows of out overlap");
  const KvAttnPlan p = kv_attn_plan(tokens, B, H, KV, hd, max_kv);
  MLCV_REQUIRE(p.bytes == 0 || (workspace && aligned16(workspace) && workspace_bytes >= p.bytes),
               "workspace missing, not 16-byte aligned or too small");
  KvAttnArgs a{};
  a.q = q;
  a.q_tok = q_tok;
  a.q_head = q_head;
  a.o_tok = o_tok;
  a.o_head = o_head;
  a.cu = cu_seqlens;
  a.kv_lens = kv_lens;
  a.table = block_table;
  a.kc = static_cast<const uint8_t*>(k_cache);
  a.vc = static_cast<const uint8_t*>(v_cache);
  a.ks = k_scale;
  a.vs = v_scale;
  a.out = out;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = a.part_o ? a.part_o + p.o_floats : nullptr;
  a.tokens = tokens;
  a.B = B;
  a.H = H;
  a.KV = KV;
  a.grp = H / KV;
  a.max_pages = num_pages > 0 ? max_pages : 0;  // a cache without pages holds nothing that could be read
  a.num_pages = num_pages;
  a.psh = log2_of(page);
  a.causal = causal != 0;
  a.q_vec = aligned16(q) && q_tok % 8 == 0 && q_head % 8 == 0;
  a.S = p.S;
  a.span = p.span;
  a.c = scale * LOG2E;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool bf = dtype == MLCV_DTYPE_BF16;
  if (hd == 64) return bf ? kv_attn_launch<true, 64>(a, p, st) : kv_attn_launch<false, 64>(a, p, st);
  if (hd == 128) return bf ? kv_attn_launch<true, 128>(a, p, st) : kv_attn_launch<false, 128>(a, p, st);
  return bf ? kv_attn_launch<true, 256>(a, p, st) : kv_attn_launch<false, 256>(a, p, st);
}

}  // extern "C"
