// fa_pages.hip — what a serving program does to the pages of the paged key/value cache (gfx950):
// sequences that fork, change places and end (fork_*_kernel), pages that are copied
// (page_copy_kernel), and a cache that is compacted (compact_*_kernel).
//
// A page may be held by several entries of the page table; shares[p] counts those beyond the
// first. What tables, lengths, parents and lists hold is checked entry by entry, as in fa_paged.hip.
#include <algorithm>

#include "fa_common.hpp"
#include "fa_layer.hpp"

namespace fa {

namespace {

__global__ __launch_bounds__(256) void zero_words_kernel(unsigned* words, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    words[i] = 0;
}

hipError_t zero_words(unsigned* words, int64_t n, hipStream_t stream) {
  const int64_t blocks = std::min<int64_t>((n + 255) / 256, 1024);
  hipLaunchKernelGGL(zero_words_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, words, n);
  return hipGetLastError();
}

// Sum, and smallest value, over a block of 256 threads; `scratch` holds 4 ints each.
__device__ __forceinline__ void block_sum_min(int& sum, int& low, int (*scratch)[4]) {
#pragma unroll
  for (int i = 32; i > 0; i >>= 1) {
    sum += __shfl_xor(sum, i, 64);
    low = min(low, __shfl_xor(low, i, 64));
  }
  if ((threadIdx.x & 63) == 0) {
    scratch[0][threadIdx.x >> 6] = sum;
    scratch[1][threadIdx.x >> 6] = low;
  }
  __syncthreads();
  sum = scratch[0][0] + scratch[0][1] + scratch[0][2] + scratch[0][3];
  low = min(min(scratch[1][0], scratch[1][1]), min(scratch[1][2], scratch[1][3]));
  __syncthreads();
}

}  // namespace

// ---- fork -------------------------------------------------------------------------------
// Row b of the new table is row parents[b] of the old one (none: empty). A row's whole pages are
// held by all its children, so shares[p] grows by the children less one at every entry; its last
// page, where it has begun, goes on with one of them, the keeper (itself, or else the first), and
// each other child takes a page from the free list to copy it to. A page whose count falls below
// zero is held by nobody and returns to the list.
//
// Two launches and more, since a row is read by blocks that write others: fork_count_kernel counts and
// puts the new rows aside, fork_finish_kernel writes them; in between lies the order of all atomics.
// Counts do not depend on it. The released pages return in ascending order, so that the result does
// not either: one block looks through the counts for them or, in a large cache, through a bitmap
// that is marked beside the counts. What bounds it is the chain behind each launch.
//
// Up to kForkCounted rows each block of fork_count_kernel looks through all parents for its row's
// children, which saves a launch; that work grows with the square of the rows, so for more of them
// fork_children_kernel counts the children of all. (Rows of a page, any parents: 4096 rows 29 us without
// the counts, 4097 30 with them, 8192 58 and 45, 32768 413 and 140, 131071 4520 and 521.)

// A row's pages, and the tokens of the last one if it has begun (0: it is full).
__device__ __forceinline__ int fork_held(const ForkArgs& a, int len, int* begun) {
  len = max(len, 0);
  const int held = (int)(((unsigned)len + a.S - 1) / a.S);
  *begun = held <= a.M ? len % a.S : 0;
  return min(held, a.M);
}
__device__ __forceinline__ bool fork_page(const ForkArgs& a, int p) { return p >= 0 && p < a.pages; }

// Each row's children, and the one that comes first: B + 1 for the row itself, B - x for child x, so
// that the largest is the keeper and 0 stands for none. The first lane adds for all of its wave that
// have the same parent, since atomics on one address follow one another: many rows with one parent are
// the samples of a prompt.
__global__ __launch_bounds__(256) void fork_children_kernel(ForkArgs a) {
  const int x = blockIdx.x * 256 + threadIdx.x;
  if (x >= a.B) return;
  const int par = a.parents[x];
  if (par < 0 || par >= a.B) return;
  const bool same = par == __builtin_amdgcn_readfirstlane(par);
  const int n = __popcll(__builtin_amdgcn_ballot_w64(same));
  const bool itself = __builtin_amdgcn_ballot_w64(same && x == par) != 0;
  const bool first = x == __builtin_amdgcn_readfirstlane(x);  // of those with a parent: of `same` too
  if (same && !first) return;
  atomicAdd(a.children + par, first ? n : 1);
  atomicMax(a.children + a.B + par, (first ? itself : x == par) ? a.B + 1 : a.B - x);
}

// Block (b, y): part y of row b's columns.
template <bool COUNTED>
__global__ __launch_bounds__(256) void fork_count_kernel(ForkArgs a) {
  __shared__ int scratch[2][4];
  const int b = blockIdx.x, tid = threadIdx.x;
  int children = 0, keeper = INT32_MAX;
  if constexpr (COUNTED) {
    children = a.children[b];
    const int first = a.children[a.B + b];
    if (first > 0) keeper = first > a.B ? b : a.B - first;
  } else {
    for (int x = tid; x < a.B; x += 256)
      if (a.parents[x] == b) {
        ++children;
        keeper = min(keeper, x == b ? -1 : x);
      }
    block_sum_min(children, keeper, scratch);
    if (keeper == -1) keeper = b;
  }
  if (blockIdx.y == 0 && tid == 0) a.keeper[b] = keeper;
  const int step = (int)gridDim.y * 256;
  int begun;
  const int held = fork_held(a, a.lengths[b], &begun);
  const int* const row = a.table + b * a.table_stride;
  for (int j = (int)blockIdx.y * 256 + tid; j < held; j += step) {
    const int n = begun && j == held - 1 ? min(children, 1) : children;
    if (n == 1) continue;
    const int p = row[j];
    if (!fork_page(a, p)) continue;
    const bool gone = atomicAdd(a.shares + p, n - 1) + n - 1 < 0;
    if (gone && a.bits) atomicOr(a.bits + (p >> 5), 1u << (p & 31));
  }
  const int par = a.parents[b];
  if (par < 0 || par >= a.B || par == b) return;
  const int taken = fork_held(a, a.lengths[par], &begun);
  const int* const from = a.table + par * a.table_stride;
  int* const to = a.rows + (int64_t)b * a.M;
  for (int j = (int)blockIdx.y * 256 + tid; j < taken; j += step) to[j] = from[j];
}

// Whether sequence b copies its parent's begun page: then `last` is its column.
__device__ __forceinline__ bool fork_copies(const ForkArgs& a, int b, int* last, int* begun) {
  const int par = a.parents[b];
  if (par < 0 || par >= a.B || par == b) return false;
  *last = fork_held(a, a.lengths[par], begun) - 1;
  return *begun > 0 && a.keeper[par] != b && fork_page(a, a.rows[(int64_t)b * a.M + *last]);
}

// The pages that nobody holds any more go back to the list, whose first `copies` pages from `start` on
// are taken. A block of 1024 threads finds them: in a small cache in the counts, from which it makes a
// bitmap in LDS with the released pages in front of each of its words; in a large one each thread
// looks through a run of the call's bitmap of candidates.
// (1500 rows of 8: the counts 14.5 us at 5000 pages and 15.6 at 8192, the bitmap 14.5 and 15.1; at 16384
// 18.5 and 15.0.)
constexpr int kForkPages = 1 << 13;  // of a small cache
struct ForkFound {
  unsigned bits[kForkPages / 32];
  int fronts[kForkPages / 32], sums[16][1];
};
__device__ __forceinline__ void fork_release(const ForkArgs& a, int start, int copies, ForkFound& f) {
  constexpr int W = 16, T = 64 * W, WORDS = kForkPages / 32;
  static_assert(WORDS <= T, "a word a thread");
  const int tid = threadIdx.x;
  int n[1] = {0}, before[1], released[1];
  if (!a.bits) {
#pragma unroll
    for (int i = 0; i < kForkPages / T; ++i) {
      const int p = T * i + tid;
      const uint64_t m = __builtin_amdgcn_ballot_w64(p < a.pages && a.shares[p] < 0);
      if ((tid & 31) == 0) f.bits[p / 32] = (unsigned)(tid & 32 ? m >> 32 : m);
    }
    __syncthreads();
    if (tid < WORDS) n[0] = __popc(f.bits[tid]);
    block_scan<W>(n, f.sums, before, released);
    if (tid < WORDS) f.fronts[tid] = before[0];
    __syncthreads();
  } else {
    const int words = (a.pages + 31) / 32, per = (words + T - 1) / T;
    const int w0 = min(words, tid * per), w1 = min(words, w0 + per);
    auto each_released = [&](auto&& found) __attribute__((always_inline)) {
      for (int w = w0; w < w1; ++w)
        for (unsigned m = a.bits[w]; m != 0; m &= m - 1) {
          const int p = 32 * w + __builtin_ctz(m);
          if (a.shares[p] < 0) found(p);
        }
    };
    each_released([&](int) { ++n[0]; });
    block_scan<W>(n, f.sums, before, released);
    int at = start + min(copies, a.F - start) - released[0] + before[0];
    each_released([&](int p) {
      a.shares[p] = 0;
      if (at >= 0) a.free_pages[at] = p;
      ++at;
    });
  }
  const int first = start + min(copies, a.F - start) - released[0];
  if (tid == 0) a.free_out[0] = max(first, 0);
  if (a.bits) return;
#pragma unroll
  for (int i = 0; i < kForkPages / T; ++i) {
    const int p = T * i + tid;
    if (p >= a.pages) break;
    const unsigned word = f.bits[p / 32];
    if (!(word >> (p & 31) & 1)) continue;
    const int k = first + f.fronts[p / 32] + __popc(word & ((1u << (p & 31)) - 1));
    a.shares[p] = 0;
    if (k >= 0) a.free_pages[k] = p;
  }
}

// Block 0: the copies and the lists. Block 1 + b + B y: part y of row b's columns.
__global__ __launch_bounds__(1024) void fork_finish_kernel(ForkArgs a) {
  constexpr int W = 16, T = 64 * W;
  __shared__ int sums[2][W][1];
  __shared__ ForkFound found;
  const int tid = threadIdx.x;
  int last, begun;
  if (blockIdx.x > 0) {
    const int b = (int)((blockIdx.x - 1) % a.B), y = (int)((blockIdx.x - 1) / a.B);
    const int par = a.parents[b];
    if (par < 0 || par >= a.B || par == b) return;
    const int skip = fork_copies(a, b, &last, &begun) ? last : -1;
    const int held = fork_held(a, a.lengths[par], &begun);
    const int* const from = a.rows + (int64_t)b * a.M;
    int* const to = a.table + b * a.table_stride;
    for (int j = y * T + tid; j < held; j += a.parts * T)
      if (j != skip) to[j] = from[j];
    return;
  }
  int start = a.free_start ? a.free_start[0] : 0;
  start = min(max(start, 0), a.F);
  int copies = 0;  // so far
  for (int b0 = 0; b0 < a.B; b0 += T) {
    const int b = b0 + tid;
    const bool copy = b < a.B && fork_copies(a, b, &last, &begun);
    int one[1] = {copy}, before[1], all[1];
    block_scan<W>(one, sums[(b0 / T) & 1], before, all);
    if (b < a.B) {
      int source = -1, target = -1;
      if (copy) {
        const int64_t at = (int64_t)start + copies + before[0];
        source = a.rows[(int64_t)b * a.M + last];
        if (at < a.F) target = a.free_pages[at];
        a.table[b * a.table_stride + last] = target;
      }
      a.sources[b] = source;
      a.targets[b] = target;
      a.tokens[b] = copy ? begun : 0;
      const int par = a.parents[b];
      a.lengths_out[b] = par < 0 || par >= a.B ? 0 : max(a.lengths[par], 0);
    }
    copies += all[0];
  }
  __syncthreads();  // the list's pages are read
  fork_release(a, start, copies, found);
}

// All of it in one block, where that has few entries to walk over. (One launch and two: 64 rows of beams,
// 112 to 1086 tokens in tables of 68 pages, 6.8 us and 9.6. Rows x pages, three quarters full:
// 64 x 16 6.5 and 9.7, 64 x 64 10.5 and 11.3, 1024 x 2 9.3 and 13.0; 64 x 128 13.6 and 11.3.)
constexpr int kForkSmall = 1 << 13;  // most table entries
constexpr int kForkRows = 1024;      // and rows, one a thread
constexpr int kForkCounted = 1 << 12;

__global__ __launch_bounds__(1024) void fork_small_kernel(ForkArgs a) {
  constexpr int W = 16, T = 64 * W;
  __shared__ int parent[kForkRows], children[kForkRows], keeper[kForkRows], rows[kForkSmall];
  __shared__ int held_s[kForkRows], begun_s[kForkRows], sums[W][1];
  __shared__ ForkFound found;
  const int tid = threadIdx.x, entries = a.B * a.M;
  int len = 0;
  if (tid < a.B) {
    const int x = a.parents[tid];
    len = a.lengths[tid];
    parent[tid] = x >= 0 && x < a.B ? x : -1;
    held_s[tid] = fork_held(a, len, &begun_s[tid]);
    children[tid] = 0;
    keeper[tid] = INT32_MAX;
  }
#pragma unroll
  for (int i = 0; i < kForkSmall / T; ++i) {
    const int t = T * i + tid, b = t / a.M;
    if (t < entries) rows[t] = a.table[b * a.table_stride + (t - b * a.M)];
  }
  int start = a.free_start ? a.free_start[0] : 0;
  start = min(max(start, 0), a.F);
  __syncthreads();
  const int par = tid < a.B ? parent[tid] : -1;
  if (par >= 0) {
    atomicAdd(children + par, 1);
    atomicMin(keeper + par, par == tid ? -1 : tid);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kForkSmall / T; ++i) {
    const int t = T * i + tid, b = t / a.M, j = t - b * a.M;
    if (t >= entries || j >= held_s[b]) continue;
    const int n = begun_s[b] && j == held_s[b] - 1 ? min(children[b], 1) : children[b];
    if (n != 1 && fork_page(a, rows[t])) atomicAdd(a.shares + rows[t], n - 1);
  }
  // The copies: child tid of par.
  const int last = par >= 0 ? held_s[par] - 1 : -1;
  const int source = last >= 0 ? rows[par * a.M + last] : -1;
  const int kept_by = par >= 0 && keeper[par] != -1 ? keeper[par] : par;
  const bool copy = par >= 0 && begun_s[par] > 0 && kept_by != tid && fork_page(a, source);
  int x[1] = {copy}, before[1], copies[1];
  block_scan<W>(x, sums, before, copies);
  int target = -1;
  if (copy && (int64_t)start + before[0] < a.F) target = a.free_pages[start + before[0]];
  if (tid < a.B) {
    a.sources[tid] = copy ? source : -1;
    a.targets[tid] = target;
    a.tokens[tid] = copy ? begun_s[par] : 0;
    a.lengths_out[tid] = par >= 0 ? max(a.lengths[par], 0) : 0;
  }
#pragma unroll
  for (int i = 0; i < kForkSmall / T; ++i) {
    const int t = T * i + tid, b = t / a.M, j = t - b * a.M;
    if (t >= entries) break;
    const int p = parent[b];
    if (p >= 0 && p != b && j < held_s[p]) a.table[b * a.table_stride + j] = rows[p * a.M + j];
  }
  __syncthreads();  // the counts are whole, and the copied pages' entries come last
  if (copy) a.table[tid * a.table_stride + last] = target;
  fork_release(a, start, copies[0], found);
}

int64_t fork_workspace_bytes(int64_t B, int64_t M, int64_t pages) {
  return 4 * (3 * B + (pages + 31) / 32 + B * M);
}

hipError_t launch_fork(const ForkArgs& args, void* workspace, hipStream_t stream) {
  ForkArgs a = args;
  const int64_t words = (a.pages + 31) / 32;
  a.keeper = static_cast<int*>(workspace);
  a.bits = reinterpret_cast<unsigned*>(a.keeper + a.B);
  a.children = reinterpret_cast<int*>(a.bits + words);
  a.rows = a.children + 2 * a.B;
  a.parts = std::min((a.M + 1023) / 1024, 16);  // four entries a thread, one
  if (a.pages <= kForkPages && a.B <= kForkRows && (int64_t)a.B * a.M <= kForkSmall) {
    a.bits = nullptr;
    hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(1024), 0, stream, a);
    return hipGetLastError();
  }
  // A few counts a thread are read sooner than the bitmap is cleared by a launch of its own.
  const bool marked = a.pages > kForkPages, counted = a.B > kForkCounted;
  hipError_t e = hipSuccess;
  if (marked || counted) {
    unsigned* const from = marked ? a.bits : reinterpret_cast<unsigned*>(a.children);
    e = zero_words(from, (marked ? words : 0) + (counted ? 2 * (int64_t)a.B : 0), stream);
    if (e != hipSuccess) return e;
  }
  if (!marked) a.bits = nullptr;
  if (a.B > 0) {
    const dim3 grid((unsigned)a.B, (unsigned)a.parts), block(256);
    if (counted) {
      hipLaunchKernelGGL(fork_children_kernel, dim3((unsigned)(a.B + 255) / 256), block, 0, stream, a);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
      hipLaunchKernelGGL(fork_count_kernel<true>, grid, block, 0, stream, a);
    } else {
      hipLaunchKernelGGL(fork_count_kernel<false>, grid, block, 0, stream, a);
    }
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fork_finish_kernel, dim3((unsigned)(1 + a.B * a.parts)), dim3(1024), 0, stream, a);
  return hipGetLastError();
}

// ---- copy -------------------------------------------------------------------------------
// Rows 0 .. tokens[i] - 1 of page targets[i] become those of page sources[i], keys and values,
// in 16-byte pieces: bound by memory. A pair's pieces are numbered along the memory, heads of a
// row or rows of a head inside, whichever lie closer; a thread takes one, past the caches. (More a
// thread, or through the caches, are slower: 1792 pages of 64 tokens, H8 D128, 0.94 GB in all.)
__global__ __launch_bounds__(256) void page_copy_kernel(CopyArgs a) {
  const unsigned pair = blockIdx.x / a.blocks;
  const int from = a.sources[pair], to = a.targets[pair];
  if (from < 0 || to < 0 || from >= a.pages || to >= a.pages) return;
  const int rows = a.tokens ? min(max(a.tokens[pair], 0), a.S) : a.S;
  const unsigned inner = a.rows_inside ? rows : a.H, outer = a.rows_inside ? a.H : rows;
  const unsigned run = inner * a.chunks;  // pieces that lie together
  const unsigned t = (blockIdx.x - pair * a.blocks) * 256 + threadIdx.x;
  if (t >= 2 * run * outer) return;
  const unsigned r = t / run, x = t - r * run, side = r >= outer, y = a.together ? 0 : x / a.chunks;
  const int64_t in = a.rows_inside ? a.ks[2] : a.ks[1], out = a.rows_inside ? a.ks[1] : a.ks[2];
  half_t* const base = (side ? a.v : a.k) + (side ? r - outer : r) * out + y * in +
                       8 * (int64_t)(x - y * a.chunks);
  const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(base + from * a.ks[0]));
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(base + to * a.ks[0]));
}

hipError_t launch_page_copy(const CopyArgs& args, hipStream_t stream) {
  CopyArgs a = args;
  a.rows_inside = a.ks[2] <= a.ks[1];
  a.together = (a.rows_inside ? a.ks[2] : a.ks[1]) == 8 * a.chunks;
  const int64_t pieces = 2 * (int64_t)a.H * a.S * a.chunks;
  a.blocks = (unsigned)((pieces + 255) / 256);
  const int64_t most = kMostBlocks / a.blocks;
  for (int64_t i = 0; i < args.n; i += most) {  // pairs past one grid's blocks: another launch
    a.n = std::min(most, args.n - i);
    a.sources = args.sources + i;
    a.targets = args.targets + i;
    if (args.tokens) a.tokens = args.tokens + i;
    const dim3 grid((unsigned)(a.n * a.blocks)), block(256);
    hipLaunchKernelGGL(page_copy_kernel, grid, block, 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---- compact ----------------------------------------------------------------------------
// Pages that the list does not name as free are held: with `used` of them, the k-th held page from
// place `used` on moves to the k-th free page in front of it. compact_mark_kernel marks the free
// pages in a bitmap, compact_rank_kernel counts along it, compact_apply_kernel renumbers the table,
// the counts and the list; compact_small_kernel does it all for a small cache.
//
// Up to kCompactCounted pages each block of compact_rank_kernel counts the whole bitmap for itself,
// which saves two launches; that work grows with the square of the pages, so in larger caches
// compact_count_kernel counts it once, by chunks of 1024 pages, and compact_scan_kernel sums the counts.
// (Half of the pages free, in any order: 2^19 pages 36 us without the counts and 39 with them, 2^20
// 52 and 48, 2^22 259 and 131, 2^26 44600 and 1800.)
constexpr int kChunk = 1024;  // pages of a chunk
constexpr int kCompactCounted = 1 << 19;

__global__ __launch_bounds__(256) void compact_mark_kernel(CompactArgs a) {
  const int start = a.free_start ? min(max(a.free_start[0], 0), a.F) : 0;
  for (int64_t i = start + (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.F; i += (int64_t)gridDim.x * 256) {
    const int p = a.free_pages[i];
    if (p >= 0 && p < a.pages) atomicOr(a.bits + (p >> 5), 1u << (p & 31));
  }
}

// Free pages of each chunk, 32 threads a chunk.
__global__ __launch_bounds__(256) void compact_count_kernel(CompactArgs a) {
  static_assert(kChunk == 32 * 32, "a word a thread");
  const int w = blockIdx.x * 256 + threadIdx.x;
  int n = w < (a.pages + 31) / 32 ? __popc(a.bits[w]) : 0;
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) n += __shfl_xor(n, i, 32);
  if (w % 32 == 0 && w / 32 < (a.pages + kChunk - 1) / kChunk) a.chunks[w / 32] = n;
}

// Free pages of the chunks in front of each, and of all behind the last.
__global__ __launch_bounds__(1024) void compact_scan_kernel(CompactArgs a) {
  constexpr int W = 16, T = 64 * W;
  __shared__ int sums[W][1];
  const int tid = threadIdx.x, n = (a.pages + kChunk - 1) / kChunk;
  const int per = (n + T - 1) / T, c0 = min(n, tid * per), c1 = min(n, c0 + per);
  int x[1] = {0}, before[1], all[1];
  for (int c = c0; c < c1; ++c) x[0] += a.chunks[c];
  block_scan<W>(x, sums, before, all);
  int front = before[0];
  for (int c = c0; c < c1; ++c) {
    const int here = a.chunks[c];
    a.chunks[c] = front;
    front += here;
  }
  if (tid == 0) a.chunks[n] = all[0];
}

// The bits of word w whose pages lie in front of page p.
__device__ __forceinline__ unsigned bits_before(int w, int p) {
  return p >= 32 * w + 32 ? ~0u : p <= 32 * w ? 0u : (1u << (p - 32 * w)) - 1;
}

// Where page p >= used or free moves, or comes from: its place among the moves, given the free pages
// in front of its word, its word of the bitmap and the moves.
__device__ __forceinline__ int compact_place(int p, int free_before, unsigned word, int used, int moves) {
  const int free = free_before + __popc(word & ((1u << (p & 31)) - 1));
  return p < used ? free : p - free - (used - moves);
}

// Block i: pages 1024 i to 1024 i + 1023, four a thread.
template <bool COUNTED>
__global__ __launch_bounds__(256) void compact_rank_kernel(CompactArgs a) {
  __shared__ int scratch[2][4], fronts[32];
  const int tid = threadIdx.x, words = (a.pages + 31) / 32;
  const int w0 = blockIdx.x * 32;
  int all = 0, front = 0, moves = 0, low = 0, used;  // moves: free pages in front of `used`
  if constexpr (COUNTED) {
    all = a.chunks[gridDim.x];
    front = a.chunks[blockIdx.x];
    used = a.pages - all;
    const int c = used / kChunk, w = c * (kChunk / 32) + tid;  // of the chunk that `used` lies in
    if (tid < kChunk / 32 && w < words) moves = __popc(a.bits[w] & bits_before(w, used));
    block_sum_min(moves, low, scratch);
    moves += a.chunks[c];
  } else {
    // (the words behind the last page's, up to a multiple of 4, are cleared as well)
    const u32x4* const bits4 = reinterpret_cast<const u32x4*>(a.bits);
#pragma unroll 4
    for (int w = 4 * tid; w < words; w += 1024) {
      const u32x4 m = bits4[w / 4];
      const int n = __popc(m[0]) + __popc(m[1]) + __popc(m[2]) + __popc(m[3]);
      all += n;
      if (w < w0) front += n;  // w0 is a multiple of 4
    }
    block_sum_min(all, low, scratch);
    block_sum_min(front, low, scratch);
    used = a.pages - all;
#pragma unroll 4
    for (int w = 4 * tid; w < words && 32 * w < used; w += 1024) {
      const u32x4 m = bits4[w / 4];
#pragma unroll
      for (int i = 0; i < 4; ++i) moves += __popc(m[i] & bits_before(w + i, used));
    }
    block_sum_min(moves, low, scratch);
  }
  if (blockIdx.x == 0 && tid == 0) {
    a.used[0] = used;
    a.counts[0] = moves;
  }
  if (tid < 64) {
    const int n = tid < 32 && w0 + tid < words ? __popc(a.bits[w0 + tid]) : 0;
    const int incl = wave_scan(n);
    if (tid < 32) fronts[tid] = front + incl - n;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = blockIdx.x * 1024 + 256 * i + tid;
    if (p >= a.pages) break;
    const unsigned word = a.bits[p >> 5];
    const bool free = word >> (p & 31) & 1;
    if (free != (p < used)) continue;
    const int k = compact_place(p, fronts[(p >> 5) - w0], word, used, moves);
    if (free) {
      a.targets[k] = p;
    } else {
      a.sources[k] = p;
      a.place[p] = k;
    }
  }
}

__global__ __launch_bounds__(256) void compact_apply_kernel(CompactArgs a) {
  const int used = a.used[0], moves = a.counts[0];
  const int start = a.free_start ? min(max(a.free_start[0], 0), a.F) : 0;
  const int64_t entries = (int64_t)a.B * a.M, all = entries + a.pages + a.F;
  auto moved = [&](int p) __attribute__((always_inline)) {
    return p >= used && p < a.pages && !(a.bits[p >> 5] >> (p & 31) & 1);
  };
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < all; t += (int64_t)gridDim.x * 256) {
    if (t < entries) {
      const int64_t b = t / a.M;
      const int p = a.table[b * a.table_stride + (t - b * a.M)];
      a.table_out[t] = moved(p) ? a.targets[a.place[p]] : p;
    } else if (t < entries + a.pages) {
      const int p = (int)(t - entries);
      const bool free = a.bits[p >> 5] >> (p & 31) & 1;
      if (p >= used) {
        a.shares_out[p] = 0;
        if (!free) a.shares_out[a.targets[a.place[p]]] = a.shares[p];
      } else if (!free) {
        a.shares_out[p] = a.shares[p];
      }
    } else {
      const int i = (int)(t - entries - a.pages);
      const int64_t p = (int64_t)used + (i - start);
      a.free_pages_out[i] = i < start ? a.free_pages[i] : p < a.pages ? (int)p : -1;
      if (i >= moves) a.sources[i] = a.targets[i] = -1;
    }
  }
}

// All of it in one block, the bitmap and the free pages in front of each of its words in LDS. (4.5 thousand
// items 7.2 us in one launch and 16 in four, 16 thousand 9.7 and 16.3, 26 thousand 15.2 and 16.4.)
constexpr int kCompactSmall = 1 << 14;  // most pages, and table entries, pages and list entries

__global__ __launch_bounds__(1024) void compact_small_kernel(CompactArgs a) {
  constexpr int W = 16, T = 64 * W, WORDS = kCompactSmall / 32;
  static_assert(WORDS <= T, "a word a thread");
  __shared__ unsigned bits[WORDS];
  __shared__ int fronts[WORDS], sums[2][W][1];
  const int tid = threadIdx.x;
  if (tid < WORDS) bits[tid] = 0;
  const int start = a.free_start ? min(max(a.free_start[0], 0), a.F) : 0;
  __syncthreads();
  for (int i = start + tid; i < a.F; i += T) {
    const int p = a.free_pages[i];
    if (p >= 0 && p < a.pages) atomicOr(bits + (p >> 5), 1u << (p & 31));
  }
  __syncthreads();
  const unsigned mine = tid < WORDS ? bits[tid] : 0u;
  int x[1] = {(int)__popc(mine)}, before[1], all[1];
  block_scan<W>(x, sums[0], before, all);
  if (tid < WORDS) fronts[tid] = before[0];
  const int used = a.pages - all[0];
  x[0] = __popc(mine & bits_before(tid, used));
  block_scan<W>(x, sums[1], before, all);
  const int moves = all[0];
  if (tid == 0) a.used[0] = used;
  auto is_free = [&](int p) __attribute__((always_inline)) { return bits[p >> 5] >> (p & 31) & 1; };
  auto place = [&](int p) __attribute__((always_inline)) {
    return compact_place(p, fronts[p >> 5], bits[p >> 5], used, moves);
  };
  for (int p = tid; p < a.pages; p += T) {
    const bool free = is_free(p);
    if (free && p < used) a.targets[place(p)] = p;
    else if (!free && p >= used) a.sources[place(p)] = p;
  }
  __syncthreads();
  auto moved = [&](int p) __attribute__((always_inline)) { return p >= used && p < a.pages && !is_free(p); };
  for (int t = tid; t < a.B * a.M; t += T) {
    const int b = t / a.M, p = a.table[b * a.table_stride + (t - b * a.M)];
    a.table_out[t] = moved(p) ? a.targets[place(p)] : p;
  }
  for (int p = tid; p < a.pages; p += T) {
    if (p >= used) a.shares_out[p] = 0;
    if (moved(p)) a.shares_out[a.targets[place(p)]] = a.shares[p];
    else if (p < used && !is_free(p)) a.shares_out[p] = a.shares[p];
  }
  for (int i = tid; i < a.F; i += T) {
    const int p = used + (i - start);
    a.free_pages_out[i] = i < start ? a.free_pages[i] : p < a.pages ? p : -1;
    if (i >= moves) a.sources[i] = a.targets[i] = -1;
  }
}

static int64_t compact_words(int64_t pages) { return (pages + 127) / 128 * 4; }
static int64_t compact_chunks(int64_t pages) { return (pages + kChunk - 1) / kChunk; }
int64_t compact_workspace_bytes(int64_t pages) {
  return 4 * (4 + compact_words(pages) + compact_chunks(pages) + 1 + pages);
}

hipError_t launch_compact(const CompactArgs& args, void* workspace, hipStream_t stream) {
  CompactArgs a = args;
  const int64_t words = compact_words(a.pages);
  const int64_t items = (int64_t)a.B * a.M + a.pages + a.F;
  if (items <= kCompactSmall) {
    hipLaunchKernelGGL(compact_small_kernel, dim3(1), dim3(1024), 0, stream, a);
    return hipGetLastError();
  }
  a.counts = static_cast<int*>(workspace);
  a.bits = reinterpret_cast<unsigned*>(a.counts + 4);
  a.chunks = reinterpret_cast<int*>(a.bits + words);
  a.place = a.chunks + compact_chunks(a.pages) + 1;
  const bool counted = a.pages > kCompactCounted;
  const dim3 block(256), chunks((unsigned)compact_chunks(a.pages));
  hipError_t e = zero_words(a.bits, words, stream);
  if (e != hipSuccess) return e;
  if (a.F > 0) {
    const dim3 grid((unsigned)std::min<int64_t>(((int64_t)a.F + 255) / 256, 2048));
    hipLaunchKernelGGL(compact_mark_kernel, grid, block, 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (counted) {
    hipLaunchKernelGGL(compact_count_kernel, dim3((chunks.x + 7) / 8), block, 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(compact_scan_kernel, dim3(1), dim3(1024), 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(compact_rank_kernel<true>, chunks, block, 0, stream, a);
  } else {
    hipLaunchKernelGGL(compact_rank_kernel<false>, chunks, block, 0, stream, a);
  }
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t blocks = std::min<int64_t>((items + 255) / 256, 4096);
  hipLaunchKernelGGL(compact_apply_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace fa
