// The pages of the paged key/value cache change hands: which ones no request holds (mlcv_kv_free), requests that go on
// from another's tokens (mlcv_kv_fork), a pool made dense (mlcv_kv_compact), pages copied (mlcv_kv_copy).
//
// Nothing counts references: the pages in use are the ones that the block table's rows hold, and are found anew by each
// call.  Shared pages need no bookkeeping then, and nothing can drift.  Two requests may share a page as long as
// neither writes to it, which is so for pages that are full; a fork copies the one that is not.
#include "kernels.h"
#include "kv_args.h"
#include "mlcvla.h"

#include <algorithm>

namespace mlcv {

namespace {

constexpr int MK_NT = 1024;   // threads of a workgroup that marks or lists pages
constexpr int LS_BLOCK = 4096;  // pages that one lists: 64 groups of 64
constexpr int MK_PARTS = 4;     // parts of the table, where a pool has up to MK_FEW blocks
constexpr int MK_FEW = 64;
constexpr int CP_NT = 256;    // of one that copies
constexpr int FK_NT = 512;    // of one that forks

// ---- pages in use ------------------------------------------------------------------------------------

struct MarkArgs {
  const int32_t *table, *lens;
  uint32_t* words;   // a bit for each page in use, whole slices
  int32_t* counts;   // of the pages in use, per LS_BLOCK
  int32_t B, max_pages, psh, num_pages, slice, vec;  // vec: rows are 16-byte aligned
};
struct ListArgs {
  const uint32_t* words;
  const int32_t* counts;
  int32_t num_pages, blocks, parts;
  int32_t *free_pages, *free_count;       // the free list, or
  int32_t *to, *holes, *from, *status;    // a dense pool's moves: page from[r] goes to holes[r], to[from[r]] = r
};

// The wave's sum in every lane, in the registers
template <int CTRL>
__device__ __forceinline__ int dpp_add(int v) {
  return v + __builtin_amdgcn_update_dpp(0, v, CTRL, 0xf, 0xf, true);
}
__device__ __forceinline__ int wave_add(int v) {
  v = dpp_add<0xb1>(v);   // lane ^ 1
  v = dpp_add<0x4e>(v);   // ^ 2
  v = dpp_add<0x141>(v);  // the other four of eight
  v = dpp_add<0x140>(v);  // the other eight of sixteen
  const auto a = __builtin_amdgcn_permlane16_swap((uint32_t)v, (uint32_t)v, false, false);
  v = (int)(a[0] + a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap((uint32_t)v, (uint32_t)v, false, false);
  return (int)(b[0] + b[1]);
}

// before[q]: bits of the block's groups before group q
__device__ __forceinline__ void groups_before(const uint64_t* groups, int* before) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    int n = __popcll(groups[lane]), v = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int u = __shfl_up(v, o);
      if (lane >= o) v += u;
    }
    before[lane] = v - n;
  }
  __syncthreads();
}

// One block's pages, by a workgroup that has its groups of 64 bits in LDS.  With u(p) the pages in use before p: free page p is
// number p - u(p) of the list; with `live` of them in all, a page in use from there on is move number u(p) - u(live), and a
// free one before it hole number p - u(p).
template <bool MOVES>
__device__ __forceinline__ void list_block(const ListArgs& a, const uint64_t* groups, int* before, int mine, int base,
                                           int live, int used_low) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  groups_before(groups, before);
#pragma unroll
  for (int i = 0; i < LS_BLOCK / MK_NT; ++i) {
    const int q = w + i * (MK_NT / 64), p = mine * LS_BLOCK + 64 * q + lane;
    if (p >= a.num_pages) continue;
    const uint64_t g = groups[q];
    const bool used = (g >> lane) & 1;
    const int u = base + before[q] +
                  (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(g >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)g, 0));
    if constexpr (MOVES) {
      if (used && p >= live) {
        a.from[u - used_low] = p;
        a.to[p] = u - used_low;
      }
      if (!used && p < live) a.holes[p - u] = p;
    } else {
      if (!used) a.free_pages[p - u] = p;
      if (p >= a.num_pages - live) a.free_pages[p] = -1;
    }
  }
  if (mine == 0 && tid == 0) {
    if constexpr (MOVES) {
      a.status[0] = live;
      a.status[1] = live - used_low;
    } else {
      *a.free_count = a.num_pages - live;
    }
  }
}

// A workgroup reads the whole table, or one of MK_PARTS parts of it, and marks the pages of its slice in LDS: reading it over
// costs less than a pass that clears a bitmap in memory before another sets bits in it by atomics.  Bound by its own
// instructions, about 12 per 64 entries: 512 rows of 256 entries over 262144 pages take 18.3 us with the whole table for each of
// 64 workgroups, 9.0 in four parts, whose bits the listing workgroups put together.
// A pool of one block is listed by the same workgroup (THEN: 1 the free list, 2 the moves), a larger one by a second launch.
// bits [slice / 32] in LDS: the pages in use of the slice from p0 on, as far as the rows of this part of `parts` have them; held
// [B]: entries of each row in use
__device__ __forceinline__ void mark_slice_bits(const MarkArgs& a, uint32_t* bits, int* held, int p0, int part, int parts) {
  __shared__ int most;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (tid == 0) most = 0;
  for (int i = tid; i < a.slice >> 5; i += MK_NT) bits[i] = 0u;
  __syncthreads();
  int mine = 0;
  for (int b = tid; b < a.B; b += MK_NT) {
    const int len = clamp_i(a.lens[b], 0, a.max_pages << a.psh), n = (int)(((int64_t)len + (1 << a.psh) - 1) >> a.psh);
    held[b] = n;
    mine = max(mine, n);
  }
  if (mine) atomicMax(&most, mine);
  __syncthreads();
  // Items of 4 rows x 256 entries.  An item's loads are issued without branches (from within the table, used or not), and the
  // next one's before it is marked: with a branch around each load the compiler waits for all of them between items.
  const uint32_t many = (uint32_t)clamp_i(a.num_pages - p0, 0, a.slice);  // pages of the slice; a page before it wraps
  const int wide = (most + 255) >> 8, items = ((a.B + 3) >> 2) * wide;
  auto fetch = [&](int it, uint32_t (&v)[16]) {
    const int b0 = it / wide * 4, j0 = (it % wide) * 256;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int32_t* row = a.table + (int64_t)min(b0 + r, a.B - 1) * a.max_pages;
      if (a.vec) {
        const u4 x = load_global(reinterpret_cast<const u4*>(row + min(j0 + 4 * lane, a.max_pages - 4)));
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * r + i] = x[i];
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * r + i] = (uint32_t)load_global(row + min(j0 + lane + 64 * i, a.max_pages - 1));
      }
    }
  };
  auto mark = [&](int it, const uint32_t (&v)[16]) {
    const int b0 = it / wide * 4, j0 = (it % wide) * 256;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = b0 + r < a.B ? held[b0 + r] : 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int j = a.vec ? j0 + 4 * lane + i : j0 + lane + 64 * i;
        const uint32_t at = v[4 * r + i] - (uint32_t)p0;
        if (j < n && at < many) atomicOr(&bits[at >> 5], 1u << (at & 31));
      }
    }
  };
  const int begin = part * (MK_NT / 64) + w, step = parts * (MK_NT / 64);
  if (begin < items) {
    uint32_t one[16], two[16];
    fetch(begin, one);
    for (int it = begin; it < items; it += 2 * step) {
      fetch(min(it + step, items - 1), two);
      mark(it, one);
      fetch(min(it + 2 * step, items - 1), one);
      if (it + step < items) mark(it + step, two);
    }
  }
  __syncthreads();
}

// Of a pool of one block, whose groups of 64 bits are in LDS: pages in use, and those of them before page number `live`
__device__ __forceinline__ void count_block(const uint64_t* groups, int* sum) {
  const int lane = threadIdx.x & 63;
  if (threadIdx.x < 64) {
    const uint64_t g = groups[lane];
    const int live = wave_add(__popcll(g)), cut = clamp_i(live - 64 * lane, 0, 64);
    const int low = wave_add(__popcll(cut == 64 ? g : g & ((1ull << cut) - 1)));
    if (lane == 0) {
      sum[0] = live;
      sum[1] = low;
    }
  }
  __syncthreads();
}

template <int THEN>
__global__ __launch_bounds__(MK_NT) void mark_kernel(const MarkArgs a, const ListArgs l) {
  extern __shared__ __attribute__((aligned(16))) int dyn[];
  __shared__ int sum[2], before[LS_BLOCK / 64];
  uint32_t* bits = reinterpret_cast<uint32_t*>(dyn);  // [slice / 32]
  int* held = dyn + (a.slice >> 5);                   // [B]
  const int tid = threadIdx.x, lane = tid & 63;
  mark_slice_bits(a, bits, held, (int)blockIdx.x * a.slice, blockIdx.y, gridDim.y);
  if constexpr (THEN == 0) {
    // 128 words of a block: two waves' lanes
    for (int i = tid; i < a.slice >> 5; i += MK_NT) {
      const uint32_t v = bits[i];
      a.words[((size_t)blockIdx.y * gridDim.x + blockIdx.x) * (a.slice >> 5) + i] = v;
      const int n = wave_add(__popc(v));
      if (lane == 0) held[i >> 6] = n;  // the rows' numbers are not needed any more
    }
    if (gridDim.y > 1) return;
    __syncthreads();
    for (int i = tid; i < a.slice / LS_BLOCK; i += MK_NT)
      a.counts[(size_t)blockIdx.x * (a.slice / LS_BLOCK) + i] = held[2 * i] + held[2 * i + 1];
  } else {
    const uint64_t* groups = reinterpret_cast<const uint64_t*>(bits);
    count_block(groups, sum);
    list_block<THEN == 2>(l, groups, before, 0, 0, sum[0], sum[1]);
  }
}

// a word's bits for pages before p, its first page being at
__device__ __forceinline__ int used_before(uint32_t word, int at, int p) {
  const int cut = clamp_i(p - at, 0, 32);
  return __popc(cut == 32 ? word : word & ((1u << cut) - 1));
}

template <bool MOVES>
__global__ __launch_bounds__(MK_NT) void list_kernel(const ListArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t groups[LS_BLOCK / 32];
  __shared__ int before[LS_BLOCK / 64], sum[3];
  const int tid = threadIdx.x, lane = tid & 63, mine = blockIdx.x;
  if (tid < 3) sum[tid] = 0;
  __syncthreads();
  int lower = 0, all = 0, low = 0;  // pages in use: before this block, of the pool, before page number `live`
  if (a.parts > 1) {
    // few blocks: every workgroup puts the parts of the whole pool together, 8 words per thread at most
    constexpr int Q = MK_FEW * (LS_BLOCK / 128) / MK_NT;
    const int quads = a.blocks * (LS_BLOCK / 128);
    u4 v[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = min(tid + q * MK_NT, quads - 1);
      u4 x[MK_PARTS];
#pragma unroll
      for (int k = 0; k < MK_PARTS; ++k)
        x[k] = load_global(reinterpret_cast<const u4*>(a.words) + (size_t)k * quads + i);
      v[q] = x[0];
#pragma unroll
      for (int k = 1; k < MK_PARTS; ++k) v[q] |= x[k];
      if (tid + q * MK_NT >= quads) v[q] = (u4){0, 0, 0, 0};
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) {
      const int i = tid + q * MK_NT, n = __popc(v[q][0]) + __popc(v[q][1]) + __popc(v[q][2]) + __popc(v[q][3]);
      const int block = i / (LS_BLOCK / 128);
      all += n;
      lower += block < mine ? n : 0;
      if (block == mine) reinterpret_cast<u4*>(groups)[i % (LS_BLOCK / 128)] = v[q];
    }
    lower = wave_add(lower);
    all = wave_add(all);
    if (lane == 0 && all) {
      atomicAdd(&sum[0], lower);
      atomicAdd(&sum[1], all);
    }
    __syncthreads();
    if constexpr (MOVES) {
#pragma unroll
      for (int q = 0; q < Q; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) low += used_before(v[q][e], (tid + q * MK_NT) * 128 + 32 * e, sum[1]);
    }
  } else {
    if (tid < LS_BLOCK / 32) groups[tid] = a.words[(size_t)mine * (LS_BLOCK / 32) + tid];
    for (int i = tid; i < a.blocks; i += MK_NT) {
      const int n = a.counts[i];
      lower += i < mine ? n : 0;
      all += n;
    }
    lower = wave_add(lower);
    all = wave_add(all);
    if (lane == 0 && all) {
      atomicAdd(&sum[0], lower);
      atomicAdd(&sum[1], all);
    }
    __syncthreads();
    if constexpr (MOVES) {
      const int live = sum[1], lb = live / LS_BLOCK;
      for (int i = tid; i < lb; i += MK_NT) low += a.counts[i];
      if (tid < LS_BLOCK / 32 && lb < a.blocks)
        low += used_before(a.words[(size_t)lb * (LS_BLOCK / 32) + tid], lb * LS_BLOCK + 32 * tid, live);
    }
  }
  if constexpr (MOVES) {
    low = wave_add(low);
    if (lane == 0 && low) atomicAdd(&sum[2], low);
    __syncthreads();
  }
  list_block<MOVES>(a, reinterpret_cast<const uint64_t*>(groups), before, mine, sum[0], sum[1], sum[2]);
}

// Slices of the pages, one for each workgroup that marks: blocks of 4096 pages, more where there would be over 1024 of them
int mark_slice(int num_pages) {
  const int64_t blocks = std::max<int64_t>(1, ((int64_t)num_pages + LS_BLOCK - 1) / LS_BLOCK);
  return (int)((blocks + 1023) / 1024) * LS_BLOCK;
}
struct MarkSizes {
  int slice, slices, blocks, parts;
  size_t words, counts;  // ints
};
MarkSizes mark_sizes(int num_pages) {
  MarkSizes m;
  m.slice = mark_slice(num_pages);
  m.slices = std::max(1, (int)(((int64_t)num_pages + m.slice - 1) / m.slice));
  m.blocks = m.slices * (m.slice / LS_BLOCK);
  m.parts = m.blocks > 1 && m.blocks <= MK_FEW ? MK_PARTS : 1;
  m.words = (size_t)m.parts * m.slices * (m.slice / 32);
  m.counts = ((size_t)m.blocks + 3) / 4 * 4;
  return m;
}
// Finds the pages in use and lists the free ones, or a dense pool's moves; l: what is to be written
template <bool MOVES>
int list_launch(const int32_t* table, const int32_t* lens, int B, int max_pages, int page, int num_pages,
                const MarkSizes& m, int32_t* workspace, ListArgs l, hipStream_t st) {
  uint32_t* words = reinterpret_cast<uint32_t*>(workspace);
  int32_t* counts = workspace + m.words;
  const MarkArgs a{table, lens, words, counts, B, max_pages, log2_of(page), num_pages, m.slice,
                   aligned16(table) && max_pages % 4 == 0};
  const size_t lds = (size_t)(m.slice / 32 + std::max(B, m.slice / 2048)) * 4;
  l.words = words;
  l.counts = counts;
  l.num_pages = num_pages;
  l.blocks = m.blocks;
  l.parts = m.parts;
  if (m.blocks == 1) {
    mark_kernel<MOVES ? 2 : 1><<<1, MK_NT, lds, st>>>(a, l);
  } else {
    mark_kernel<0><<<dim3(m.slices, m.parts), MK_NT, lds, st>>>(a, l);
    MLCV_HIP(hipGetLastError());
    list_kernel<MOVES><<<(unsigned)m.blocks, MK_NT, 0, st>>>(l);
  }
  MLCV_HIP(hipGetLastError());
  return 0;
}

// ---- copying -----------------------------------------------------------------------------------------

struct Pool {
  uint8_t* data[2];  // keys, values [layers][pages][page_bytes]
  float* scale[2];   // [layers][pages][KV]
  int32_t pages;
};
struct CopyArgs {
  Pool from, into;
  const int32_t *src, *dst, *count;  // count: how many of them there are (null: most)
  int32_t most, layers, KV, page_bytes, pieces;
};
constexpr int CP_PIECE = 2048;  // bytes that a wave moves at a time: 2 loads of 16 per lane

// Units of one page, layer, side and piece; a wave takes one after another.  Bound by memory: 4001 pages of 32 KB of two layers
// take 105.7 us, 5.0 TB/s read and written.  Small units in many waves, and stores past the caches, which leaves those to pages that
// are read several times.  On end in a graph over three pools in turn: these copies, 431 pages forked from 64 in 6 layers, and a pool
// of 12000 pages of 32 KB made dense (2954 move) take 108.8, 22.8 and 43.5 us; with plain stores 110.7, 28.4 and 52.1, with 8 KB per
// wave 109.3, 27.5 and 48.0, with both 111.6, 29.5 and 56.1; with 1 KB per wave 113.6, 24.0 and 53.0.
// pair(i) gives pages (from, into) number i of n.
template <class Pair>
__device__ __forceinline__ void copy_pages(const CopyArgs& a, int n, long long unit, long long step, Pair pair) {
  const int lane = threadIdx.x & 63;
  const int per = a.layers * 2 * a.pieces;
  const long long units = (long long)n * per;
  for (; unit < units; unit += step) {
    const int i = (int)(unit / per), rest = (int)(unit - (long long)i * per);
    const int piece = rest % a.pieces, z = (rest / a.pieces) & 1, y = rest / a.pieces >> 1;
    const int2 p2 = pair(i);
    const int s = p2.x, d = p2.y;
    if (s < 0 || s >= a.from.pages || d < 0 || d >= a.into.pages) continue;
    const long long ps = (long long)y * a.from.pages + s, pd = (long long)y * a.into.pages + d;
    const u4* p = reinterpret_cast<const u4*>(a.from.data[z] + ps * a.page_bytes + piece * CP_PIECE) + lane;
    u4* q = reinterpret_cast<u4*>(a.into.data[z] + pd * a.page_bytes + piece * CP_PIECE) + lane;
    const int left = min(CP_PIECE, a.page_bytes - piece * CP_PIECE) / 16 - lane;
    u4 v[CP_PIECE / 1024];
#pragma unroll
    for (int k = 0; k < CP_PIECE / 1024; ++k)
      if (64 * k < left) v[k] = load_global(p + 64 * k);
#pragma unroll
    for (int k = 0; k < CP_PIECE / 1024; ++k)
      if (64 * k < left) __builtin_nontemporal_store(v[k], q + 64 * k);
    if (piece == 0)
      for (int h = lane; h < a.KV; h += 64) a.into.scale[z][pd * a.KV + h] = a.from.scale[z][ps * a.KV + h];
  }
}
// pairs from the lists
__device__ __forceinline__ void copy_listed(const CopyArgs& a, long long unit, long long step) {
  const int n = a.count ? clamp_i(*a.count, 0, a.most) : a.most;
  copy_pages(a, n, unit, step, [&](int i) { return make_int2(a.src[i], a.dst[i]); });
}

__global__ __launch_bounds__(CP_NT) void copy_kernel(const CopyArgs a) {
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  copy_listed(a, (long long)blockIdx.x * (CP_NT / 64) + w, (long long)gridDim.x * (CP_NT / 64));
}

struct RenameArgs {
  const int32_t *table, *lens, *to, *holes, *status;
  int32_t* out;
  int32_t B, max_pages, psh, num_pages, groups;
};
// The moves of a dense pool, and in the first `groups` workgroups the table's new page numbers: a row each, in turn
__global__ __launch_bounds__(CP_NT) void move_kernel(const CopyArgs a, const RenameArgs t) {
  if ((int)blockIdx.x >= t.groups) {
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    copy_listed(a, (long long)(blockIdx.x - t.groups) * (CP_NT / 64) + w, (long long)(gridDim.x - t.groups) * (CP_NT / 64));
    return;
  }
  const int live = t.status[0];
  for (int b = blockIdx.x; b < t.B; b += t.groups) {
    const int len = clamp_i(t.lens[b], 0, t.max_pages << t.psh), n = (int)(((int64_t)len + (1 << t.psh) - 1) >> t.psh);
    for (int j = threadIdx.x; j < t.max_pages; j += CP_NT) {
      const int64_t at = (int64_t)b * t.max_pages + j;
      int id = t.table[at];
      if (j < n && id >= live && id < t.num_pages) id = t.holes[t.to[id]];
      t.out[at] = id;
    }
  }
}

// A small pool made dense in one launch: every workgroup finds the moves for itself, keeps them in LDS, and does its share.  The
// new table must not be the old one, which others still read.  16 requests on 185 of 512 pages, 113 of which move, in 2 layers:
// 7.2 us on the GPU; a launch for the moves and another for the copies take 4.9 and 3.3, and the call 2.9 us longer.
__global__ __launch_bounds__(MK_NT) void dense_kernel(const MarkArgs a, const CopyArgs c, int32_t* out, int32_t* status) {
  extern __shared__ __attribute__((aligned(16))) int dyn[];
  __shared__ int sum[2], before[LS_BLOCK / 64];
  __shared__ uint16_t from[LS_BLOCK / 2], holes[LS_BLOCK / 2];
  uint32_t* bits = reinterpret_cast<uint32_t*>(dyn);  // [LS_BLOCK / 32]
  int* held = dyn + LS_BLOCK / 32;                    // [B]
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  mark_slice_bits(a, bits, held, 0, 0, 1);
  const uint64_t* groups = reinterpret_cast<const uint64_t*>(bits);
  count_block(groups, sum);
  groups_before(groups, before);
  const int live = sum[0], used_low = sum[1], moves = live - used_low;
  auto used = [&](int p) { return before[p >> 6] + __popcll(groups[p >> 6] & ((1ull << (p & 63)) - 1)); };  // before page p
#pragma unroll
  for (int i = 0; i < LS_BLOCK / MK_NT; ++i) {
    const int p = tid + i * MK_NT;
    if (p >= a.num_pages) continue;
    const bool in_use = (groups[p >> 6] >> (p & 63)) & 1;
    if (in_use && p >= live) from[used(p) - used_low] = (uint16_t)p;
    if (!in_use && p < live) holes[p - used(p)] = (uint16_t)p;
  }
  __syncthreads();
  if (blockIdx.x == 0 && tid == 0) {
    status[0] = live;
    status[1] = moves;
  }
  const int wave = blockIdx.x * (MK_NT / 64) + w, waves = gridDim.x * (MK_NT / 64);
  for (int b = wave; b < a.B; b += waves) {
    const int n = held[b];
    for (int j = lane; j < a.max_pages; j += 64) {
      const int64_t at = (int64_t)b * a.max_pages + j;
      int id = a.table[at];
      if (j < n && id >= live && id < a.num_pages) id = holes[used(id) - used_low];
      out[at] = id;
    }
  }
  copy_pages(c, moves, wave, waves, [&](int i) {
    return make_int2(__builtin_amdgcn_readfirstlane((int)from[i]), __builtin_amdgcn_readfirstlane((int)holes[i]));
  });
}

// Workgroups for `most` pages, of which there may be fewer: up to 16384.  With 2048 (about what the GPU holds at once) the
// copies above take 113.5, 22.7 and 46.0 us.
unsigned copy_groups(const CopyArgs& a) {
  const int64_t units = (int64_t)a.most * a.layers * 2 * a.pieces;
  return (unsigned)std::min<int64_t>((units + CP_NT / 64 - 1) / (CP_NT / 64), 16384);
}

// ---- forks -------------------------------------------------------------------------------------------

struct ForkArgs {
  const int32_t *parents, *table, *lens, *free_pages, *free_count;
  int32_t *out, *out_lens, *status;
  int32_t N, B, max_pages, psh, n_free;
};

// Row i of the new table goes on from row parents[i].  The first of a parent's rows keeps its last page, if that is not
// full; the others take a free one each, in their order.  Every workgroup finds this out for all rows (as the
// plan's do), then writes its own and copies its share of the pages: for few rows that takes as long as a second launch
// would, a call for 16 rows of 4 requests and 12 pages in 18 layers takes 13.4 us in one launch (5.9 on the GPU), 17.5 in two (3.0
// and 5.3); for 512 rows and 431 pages in 6 layers 22.5 and 20.3.
__global__ __launch_bounds__(FK_NT) void fork_kernel(const ForkArgs a, const CopyArgs c) {
  extern __shared__ int sm[];
  __shared__ long long part[FK_NT / 64], carry;
  __shared__ int lost;
  int* first = sm;              // [B] the first row of each parent
  int* fresh = sm + a.B;        // [N] number of the free page that a row takes; -1: none; -2: refused
  int* from = sm + a.B + a.N;   // [N] of each free page taken, the page that is copied there
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), page = 1 << a.psh;
  const int n_free = a.free_count ? clamp_i(*a.free_count, 0, a.n_free) : a.n_free;
  for (int b = tid; b < a.B; b += FK_NT) first[b] = INT32_MAX;
  if (tid == 0) lost = 0;
  __syncthreads();
  for (int i = tid; i < a.N; i += FK_NT) {
    const int p = a.parents[i];
    if (p >= 0 && p < a.B) atomicMin(&first[p], i);
  }
  __syncthreads();
  long long taken = 0;
  int refused = 0;
  for (int i0 = 0; i0 < a.N; i0 += FK_NT) {
    const int i = i0 + tid, p = i < a.N ? a.parents[i] : -1;
    const bool there = p >= 0 && p < a.B;
    const int len = there ? clamp_i(a.lens[p], 0, a.max_pages << a.psh) : 0;
    const bool need = there && (len & (page - 1)) && first[p] != i;
    const long long end = block_scan<FK_NT>(need, part) + taken;
    const bool ok = !need || end <= n_free;
    refused += !ok;
    if (i < a.N) fresh[i] = !ok ? -2 : need ? (int)end - 1 : -1;
    if (need && ok) from[end - 1] = a.table[(int64_t)p * a.max_pages + (len >> a.psh)];
    if (blockIdx.x == 0 && i < a.N) a.out_lens[i] = ok ? len : 0;
    if (tid == FK_NT - 1) carry = end;
    __syncthreads();
    taken = carry;
    __syncthreads();
  }
  const int got = (int)(taken < n_free ? taken : n_free);
  if (blockIdx.x == 0) {
    if (refused) atomicAdd(&lost, refused);
    __syncthreads();
    if (tid == 0) {
      a.status[0] = got;
      a.status[1] = lost;
    }
  }
  // a wave for each row
  for (int i = blockIdx.x * (FK_NT / 64) + w; i < a.N; i += gridDim.x * (FK_NT / 64)) {
    const int p = a.parents[i], f = fresh[i];
    const bool there = p >= 0 && p < a.B && f != -2;
    const int len = there ? clamp_i(a.lens[p], 0, a.max_pages << a.psh) : 0;
    const int n = (int)(((int64_t)len + page - 1) >> a.psh);
    for (int j = lane; j < a.max_pages; j += 64) {
      int id = j < n ? a.table[(int64_t)p * a.max_pages + j] : -1;
      if (f >= 0 && j == n - 1) id = a.free_pages[f];
      a.out[(int64_t)i * a.max_pages + j] = id;
    }
  }
  copy_pages(c, got, (long long)blockIdx.x * (FK_NT / 64) + w, (long long)gridDim.x * (FK_NT / 64),
             [&](int i) { return make_int2(__builtin_amdgcn_readfirstlane(from[i]), a.free_pages[i]); });
}

int pages_ok(int32_t num_pages, int32_t page, int32_t max_pages, int32_t B) {
  MLCV_REQUIRE(kv_page_ok(page), "page must be 16, 32, 64 or 128");
  MLCV_REQUIRE(num_pages >= 0 && max_pages >= 0 && B >= 0, "negative size");
  MLCV_REQUIRE((int64_t)num_pages * page <= KV_MOST && (int64_t)max_pages * page <= KV_MOST,
               "more than 2^31 - 256 slots");
  MLCV_REQUIRE(B <= KV_MAX_REQ, "more than 4096 requests");
  return 0;
}

// The copying part of a call; `a`'s lists are the caller's
int pool_ok(CopyArgs& a, void* k, float* ks, void* v, float* vs, int32_t num_pages, void* k2, float* ks2, void* v2,
            float* vs2, int32_t num_pages2, int32_t layers, int32_t page, int32_t KV, int32_t hd) {
  MLCV_REQUIRE(kv_page_ok(page), "page must be 16, 32, 64 or 128");
  MLCV_REQUIRE(kv_hd_ok(hd), "head_dim must be 64, 128 or 256");
  MLCV_REQUIRE(layers > 0 && layers <= 65535 && KV > 0 && KV <= 65535, "layers and kv heads must be 1 to 65535");
  MLCV_REQUIRE((num_pages == 0 || (k && ks && v && vs)) && (num_pages2 == 0 || (k2 && ks2 && v2 && vs2)), "null cache");
  MLCV_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k2) && aligned16(v2), "the cache must be 16-byte aligned");
  a.from = Pool{{static_cast<uint8_t*>(k), static_cast<uint8_t*>(v)}, {ks, vs}, num_pages};
  a.into = Pool{{static_cast<uint8_t*>(k2), static_cast<uint8_t*>(v2)}, {ks2, vs2}, num_pages2};
  MLCV_REQUIRE((int64_t)KV * page * hd <= 1 << 30, "a page of more than 2^30 bytes");
  a.layers = layers;
  a.KV = KV;
  a.page_bytes = KV * page * hd;
  a.pieces = (a.page_bytes + CP_PIECE - 1) / CP_PIECE;
  MLCV_REQUIRE((int64_t)a.layers * 2 * a.pieces <= INT32_MAX, "too many layers and heads");
  return 0;
}

size_t compact_ints(int32_t num_pages) {
  const MarkSizes m = mark_sizes(num_pages);
  return m.words + m.counts + 3 * (size_t)num_pages;
}

}  // namespace
}  // namespace mlcv

using namespace mlcv;

extern "C" {

int mlcv_kv_free_workspace(int32_t num_pages, size_t* bytes) {
  MLCV_REQUIRE(bytes, "null pointer");
  MLCV_REQUIRE(num_pages >= 0 && num_pages <= KV_MOST / 16, "bad num_pages");
  const MarkSizes m = mark_sizes(num_pages);
  *bytes = (m.words + m.counts) * 4;
  return 0;
}

int mlcv_kv_free(const int32_t* block_table, int32_t B, int32_t max_pages, const int32_t* kv_lens, int32_t num_pages,
                 int32_t page, int32_t* free_pages, int32_t* free_count, void* workspace, size_t workspace_bytes,
                 void* stream) {
  MLCV_TRY(pages_ok(num_pages, page, max_pages, B));
  MLCV_REQUIRE(free_count && (num_pages == 0 || free_pages), "null output");
  MLCV_REQUIRE(B == 0 || (kv_lens && (block_table || max_pages == 0)), "null request array");
  const MarkSizes m = mark_sizes(num_pages);
  MLCV_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= (m.words + m.counts) * 4,
               "workspace missing, not 16-byte aligned or too small");
  const Ints arrays[] = {{free_pages, num_pages}, {free_count, 1}, {workspace, (int64_t)(m.words + m.counts)},
                         {block_table, (int64_t)B * max_pages}, {kv_lens, B}};
  MLCV_REQUIRE(!overlap(arrays, 3, 5), "outputs overlap the inputs or one another");
  ListArgs l{};
  l.free_pages = free_pages;
  l.free_count = free_count;
  return list_launch<false>(block_table, kv_lens, B, max_pages, page, num_pages, m, static_cast<int32_t*>(workspace), l,
                            reinterpret_cast<hipStream_t>(stream));
}

int mlcv_kv_copy(const int32_t* src, const int32_t* dst, int32_t n, void* k_cache, float* k_scale, void* v_cache,
                 float* v_scale, int32_t num_pages, void* k_into, float* k_scale_into, void* v_into,
                 float* v_scale_into, int32_t pages_into, int32_t layers, int32_t page, int32_t KV, int32_t hd,
                 void* stream) {
  MLCV_REQUIRE(n >= 0, "negative size");
  MLCV_TRY(pages_ok(num_pages, page, 0, 0));
  MLCV_TRY(pages_ok(pages_into, page, 0, 0));
  CopyArgs a{};
  MLCV_TRY(pool_ok(a, k_cache, k_scale, v_cache, v_scale, num_pages, k_into, k_scale_into, v_into, v_scale_into,
                   pages_into, layers, page, KV, hd));
  if (n == 0 || num_pages == 0 || pages_into == 0) return 0;
  MLCV_REQUIRE(src && dst, "null pointer");
  a.src = src;
  a.dst = dst;
  a.most = n;
  copy_kernel<<<copy_groups(a), CP_NT, 0, reinterpret_cast<hipStream_t>(stream)>>>(a);
  MLCV_HIP(hipGetLastError());
  return 0;
}

int mlcv_kv_fork(const int32_t* parents, int32_t n, const int32_t* block_table, int32_t B, int32_t max_pages,
                 const int32_t* kv_lens, const int32_t* free_pages, int32_t n_free, const int32_t* free_count,
                 void* k_cache, float* k_scale, void* v_cache, float* v_scale, int32_t layers, int32_t num_pages,
                 int32_t page, int32_t KV, int32_t hd, int32_t* new_table, int32_t* new_lens, int32_t* status,
                 void* stream) {
  MLCV_TRY(pages_ok(num_pages, page, max_pages, B));
  MLCV_REQUIRE(n >= 0 && n_free >= 0, "negative size");
  MLCV_REQUIRE(n <= KV_MAX_REQ, "more than 4096 requests");
  CopyArgs a{};
  MLCV_TRY(pool_ok(a, k_cache, k_scale, v_cache, v_scale, num_pages, k_cache, k_scale, v_cache, v_scale, num_pages,
                   layers, page, KV, hd));
  MLCV_REQUIRE(status, "null output");
  MLCV_REQUIRE(n == 0 || (parents && new_lens && (new_table || max_pages == 0)), "null row array");
  MLCV_REQUIRE(B == 0 || (kv_lens && (block_table || max_pages == 0)), "null request array");
  MLCV_REQUIRE(n_free == 0 || free_pages, "null free_pages");
  const Ints arrays[] = {{new_table, (int64_t)n * max_pages}, {new_lens, n}, {status, 2},
                         {parents, n}, {block_table, (int64_t)B * max_pages}, {kv_lens, B}, {free_pages, n_free},
                         {free_count, free_count ? 1 : 0}};
  MLCV_REQUIRE(!overlap(arrays, 3, 8), "outputs overlap the inputs or one another");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const ForkArgs f{parents, block_table, kv_lens, free_pages, free_count, new_table, new_lens, status, n, B, max_pages,
                   log2_of(page), n_free};
  // a wave for each row, and for each unit of the pages as far as the GPU holds them at once
  const int64_t units = num_pages ? (int64_t)std::min(n, n_free) * layers * 2 * a.pieces : 0;
  const int64_t waves = std::max<int64_t>({1, std::min(n, 2048), std::min<int64_t>(units, 8192)});
  fork_kernel<<<(unsigned)((waves + FK_NT / 64 - 1) / (FK_NT / 64)), FK_NT, (size_t)(B + 2 * n) * 4, st>>>(f, a);
  MLCV_HIP(hipGetLastError());
  return 0;
}

int mlcv_kv_compact_workspace(int32_t num_pages, size_t* bytes) {
  MLCV_REQUIRE(bytes, "null pointer");
  MLCV_REQUIRE(num_pages >= 0 && num_pages <= KV_MOST / 16, "bad num_pages");
  *bytes = compact_ints(num_pages) * 4;
  return 0;
}

int mlcv_kv_compact(const int32_t* block_table, int32_t B, int32_t max_pages, const int32_t* kv_lens, void* k_cache,
                    float* k_scale, void* v_cache, float* v_scale, int32_t layers, int32_t num_pages, int32_t page,
                    int32_t KV, int32_t hd, int32_t* new_table, int32_t* status, void* workspace,
                    size_t workspace_bytes, void* stream) {
  MLCV_TRY(pages_ok(num_pages, page, max_pages, B));
  CopyArgs a{};
  MLCV_TRY(pool_ok(a, k_cache, k_scale, v_cache, v_scale, num_pages, k_cache, k_scale, v_cache, v_scale, num_pages,
                   layers, page, KV, hd));
  MLCV_REQUIRE(status, "null output");
  MLCV_REQUIRE(B == 0 || (kv_lens && ((block_table && new_table) || max_pages == 0)), "null request array");
  const size_t ints = compact_ints(num_pages);
  MLCV_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= ints * 4,
               "workspace missing, not 16-byte aligned or too small");
  // the table may become the new one in place
  const int64_t entries = (int64_t)B * max_pages;
  const Ints arrays[] = {{new_table, entries}, {status, 2}, {workspace, (int64_t)ints}, {kv_lens, B},
                         {block_table, new_table == block_table ? 0 : entries}};
  MLCV_REQUIRE(!overlap(arrays, 3, 5), "outputs overlap the inputs or one another");
  const MarkSizes m = mark_sizes(num_pages);
  // every move has a hole: at most half of the pages move
  a.most = num_pages / 2;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (m.blocks == 1 && new_table != block_table && ((int64_t)B + 3) / 4 * ((max_pages + 255) / 256) <= 2 * (MK_NT / 64)) {
    // the table is marked in two rounds of a workgroup's waves at most
    const MarkArgs k{block_table, kv_lens, nullptr, nullptr, B, max_pages, log2_of(page), num_pages, m.slice,
                     aligned16(block_table) && max_pages % 4 == 0};
    const int64_t waves = std::max<int64_t>({1, B, std::min<int64_t>((int64_t)a.most * layers * 2 * a.pieces, 8192)});
    dense_kernel<<<(unsigned)((waves + MK_NT / 64 - 1) / (MK_NT / 64)), MK_NT, (size_t)(LS_BLOCK / 32 + B) * 4, st>>>(
        k, a, new_table, status);
    MLCV_HIP(hipGetLastError());
    return 0;
  }
  ListArgs l{};
  l.to = static_cast<int32_t*>(workspace) + m.words + m.counts;
  l.holes = l.to + num_pages;
  l.from = l.holes + num_pages;
  l.status = status;
  MLCV_TRY(list_launch<true>(block_table, kv_lens, B, max_pages, page, num_pages, m, static_cast<int32_t*>(workspace), l, st));
  a.src = l.from;
  a.dst = l.holes;
  a.count = status + 1;
  const RenameArgs t{block_table, kv_lens, l.to, l.holes, status, new_table, B, max_pages, log2_of(page), num_pages,
                     std::min(B, 256)};
  const unsigned grid = t.groups + (a.most ? copy_groups(a) : 0);
  if (grid == 0) return 0;
  move_kernel<<<grid, CP_NT, 0, st>>>(a, t);
  MLCV_HIP(hipGetLastError());
  return 0;
}

}  // extern "C"
