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
// Three launches, since a row is read by blocks that write others: fork_count_kernel counts and
// puts the new rows aside, fork_finish_kernel writes them; in between lies the order of all atomics.
// Counts do not depend on it. The released pages are marked in a bitmap and return in ascending
// order, so that the result does not either. What bounds it is the chain behind each launch.

// A row's pages, and the tokens of the last one if it has begun (0: it is full).
__device__ __forceinline__ int fork_held(const ForkArgs& a, int len, int* begun) {
  len = max(len, 0);
  const int held = (int)(((unsigned)len + a.S - 1) / a.S);
  *begun = held <= a.M ? len % a.S : 0;
  return min(held, a.M);
}
__device__ __forceinline__ bool fork_page(const ForkArgs& a, int p) { return p >= 0 && p < a.pages; }

// Block (b, y): part y of row b's columns.
__global__ __launch_bounds__(256) void fork_count_kernel(ForkArgs a) {
  __shared__ int scratch[2][4];
  const int b = blockIdx.x, tid = threadIdx.x;
  int children = 0, keeper = INT32_MAX;
  for (int x = tid; x < a.B; x += 256)
    if (a.parents[x] == b) {
      ++children;
      keeper = min(keeper, x == b ? -1 : x);
    }
  block_sum_min(children, keeper, scratch);
  if (keeper == -1) keeper = b;
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
    if (atomicAdd(a.shares + p, n - 1) + n - 1 < 0) atomicOr(a.bits + (p >> 5), 1u << (p & 31));
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

// Block 0: the copies and the lists. Block 1 + b + B y: part y of row b's columns.
__global__ __launch_bounds__(1024) void fork_finish_kernel(ForkArgs a) {
  constexpr int W = 16, T = 64 * W;
  __shared__ int sums[2][W][1];
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
  __syncthreads();  // the list's pages are read; scratch is free
  // The released pages, a run of the bitmap's words a thread.
  const int words = (a.pages + 31) / 32, per = (words + T - 1) / T;
  const int w0 = min(words, tid * per), w1 = min(words, w0 + per);
  int count[1] = {0}, before[1], released[1];
  for (int w = w0; w < w1; ++w)
    for (unsigned m = a.bits[w]; m != 0; m &= m - 1)
      count[0] += a.shares[32 * w + __builtin_ctz(m)] < 0;
  block_scan<W>(count, sums[0], before, released);
  const int first = start + min(copies, a.F - start) - released[0];
  int at = first + before[0];
  for (int w = w0; w < w1; ++w)
    for (unsigned m = a.bits[w]; m != 0; m &= m - 1) {
      const int p = 32 * w + __builtin_ctz(m);
      if (a.shares[p] >= 0) continue;
      a.shares[p] = 0;
      if (at >= 0) a.free_pages[at] = p;
      ++at;
    }
  if (tid == 0) a.free_out[0] = max(first, 0);
}

int64_t fork_workspace_bytes(int64_t B, int64_t M, int64_t pages) {
  return 4 * (B + (pages + 31) / 32 + B * M);
}

hipError_t launch_fork(const ForkArgs& args, void* workspace, hipStream_t stream) {
  ForkArgs a = args;
  const int64_t words = (a.pages + 31) / 32;
  a.keeper = static_cast<int*>(workspace);
  a.bits = reinterpret_cast<unsigned*>(a.keeper + a.B);
  a.rows = reinterpret_cast<int*>(a.bits + words);
  a.parts = std::min((a.M + 1023) / 1024, 16);  // four entries a thread, one
  hipError_t e = zero_words(a.bits, words, stream);
  if (e != hipSuccess) return e;
  if (a.B > 0) {
    hipLaunchKernelGGL(fork_count_kernel, dim3((unsigned)a.B, (unsigned)a.parts), dim3(256), 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fork_finish_kernel, dim3((unsigned)(1 + a.B * a.parts)), dim3(1024), 0, stream, a);
  return hipGetLastError();
}

// ---- copy -------------------------------------------------------------------------------
// Rows 0 .. tokens[i] - 1 of page targets[i] become those of page sources[i], keys and values,
// in 16-byte pieces: bound by memory. A pair's pieces are numbered along the memory, heads of a
// row or rows of a head inside, whichever lie closer; a block takes 256 U of them.

template <int U>
__global__ __launch_bounds__(256) void page_copy_kernel(CopyArgs a) {
  const unsigned pair = blockIdx.x / a.blocks;
  const int from = a.sources[pair], to = a.targets[pair];
  if (from < 0 || to < 0 || from >= a.pages || to >= a.pages) return;
  const int rows = a.tokens ? min(max(a.tokens[pair], 0), a.S) : a.S;
  const unsigned inner = a.rows_inside ? rows : a.H, outer = a.rows_inside ? a.H : rows;
  const unsigned run = inner * a.chunks;  // pieces that lie together
  const unsigned all = 2 * run * outer;
  const unsigned first = (blockIdx.x - pair * a.blocks) * (256 * U) + threadIdx.x;
  if (first >= all) return;
  const int64_t in = a.rows_inside ? a.ks[2] : a.ks[1], out = a.rows_inside ? a.ks[1] : a.ks[2];
  u32x4 v[U];
  half_t* dst[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const unsigned t = first + 256 * i;
    if (t >= all) continue;
    const unsigned r = t / run, side = r >= outer, o = side ? r - outer : r, x = t - r * run;
    const unsigned y = a.together ? 0 : x / a.chunks;
    const int64_t off = o * out + y * in + 8 * (int64_t)(x - y * a.chunks);
    half_t* const base = (side ? a.v : a.k) + off;
    dst[i] = base + to * a.ks[0];
    v[i] = *reinterpret_cast<const u32x4*>(base + from * a.ks[0]);
  }
#pragma unroll
  for (int i = 0; i < U; ++i)
    if (first + 256 * i < all) __builtin_nontemporal_store(v[i], reinterpret_cast<u32x4*>(dst[i]));
}

hipError_t launch_page_copy(const CopyArgs& args, hipStream_t stream) {
  CopyArgs a = args;
  a.rows_inside = a.ks[2] <= a.ks[1];
  a.together = (a.rows_inside ? a.ks[2] : a.ks[1]) == 8 * a.chunks;
  const int64_t pieces = 2 * (int64_t)a.H * a.S * a.chunks;
  const bool small = a.n * pieces <= 256 * 2048;
  const int64_t each = small ? 256 : 256 * 8;
  a.blocks = (unsigned)((pieces + each - 1) / each);
  const int64_t most = kMostBlocks / a.blocks;
  for (int64_t i = 0; i < args.n; i += most) {  // pairs past one grid's blocks: another launch
    a.n = std::min(most, args.n - i);
    a.sources = args.sources + i;
    a.targets = args.targets + i;
    if (args.tokens) a.tokens = args.tokens + i;
    const dim3 grid((unsigned)(a.n * a.blocks)), block(256);
    if (small) hipLaunchKernelGGL(page_copy_kernel<1>, grid, block, 0, stream, a);
    else hipLaunchKernelGGL(page_copy_kernel<8>, grid, block, 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---- compact ----------------------------------------------------------------------------
// Pages that the list does not name as free are held: with `used` of them, the k-th held page from
// place `used` on moves to the k-th free page in front of it. compact_mark_kernel marks the free
// pages in a bitmap, compact_rank_kernel counts along it (every block for itself, over the words in
// front of its own), compact_apply_kernel renumbers the table, the counts and the list.

__global__ __launch_bounds__(256) void compact_mark_kernel(CompactArgs a) {
  const int start = a.free_start ? min(max(a.free_start[0], 0), a.F) : 0;
  for (int64_t i = start + (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.F; i += (int64_t)gridDim.x * 256) {
    const int p = a.free_pages[i];
    if (p >= 0 && p < a.pages) atomicOr(a.bits + (p >> 5), 1u << (p & 31));
  }
}

// The bits of word w whose pages lie in front of page p.
__device__ __forceinline__ unsigned bits_before(int w, int p) {
  return p >= 32 * w + 32 ? ~0u : p <= 32 * w ? 0u : (1u << (p - 32 * w)) - 1;
}

// Block i: words 256 i to 256 i + 255, one a thread.
__global__ __launch_bounds__(256) void compact_rank_kernel(CompactArgs a) {
  __shared__ int scratch[2][4], sums[4][1];
  const int tid = threadIdx.x, words = (a.pages + 31) / 32;
  const int w0 = blockIdx.x * 256;
  int all = 0, front = 0, moves = 0, low = 0;
  for (int w = tid; w < words; w += 256) {
    const int n = __popc(a.bits[w]);
    all += n;
    if (w < w0) front += n;
  }
  block_sum_min(all, low, scratch);
  block_sum_min(front, low, scratch);
  const int used = a.pages - all;
  for (int w = tid; w < words && 32 * w < used; w += 256) moves += __popc(a.bits[w] & bits_before(w, used));
  block_sum_min(moves, low, scratch);  // free pages in front of `used`, held ones behind it
  if (blockIdx.x == 0 && tid == 0) {
    a.used[0] = used;
    a.counts[0] = moves;
  }
  const int w = w0 + tid;
  const unsigned free = w < words ? a.bits[w] : 0u;
  int x[1] = {(int)__popc(free)}, before[1], total[1];
  block_scan<4>(x, sums, before, total);
  if (w >= words) return;
  const int free_before = front + before[0];
  const unsigned in = bits_before(w, used);
  int k = free_before;
  for (unsigned m = free & in; m != 0; m &= m - 1) a.targets[k++] = 32 * w + __builtin_ctz(m);
  for (unsigned m = ~free & ~in & bits_before(w, a.pages); m != 0; m &= m - 1) {
    const int bit = __builtin_ctz(m), p = 32 * w + bit;
    // held pages in front of p, less those that stay
    k = p - free_before - __popc(free & ((1u << bit) - 1)) - (used - moves);
    a.sources[k] = p;
    a.place[p] = k;
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

int64_t compact_workspace_bytes(int64_t pages) { return 4 * (1 + (pages + 31) / 32 + pages); }

hipError_t launch_compact(const CompactArgs& args, void* workspace, hipStream_t stream) {
  CompactArgs a = args;
  const int64_t words = ((int64_t)a.pages + 31) / 32;
  a.counts = static_cast<int*>(workspace);
  a.bits = reinterpret_cast<unsigned*>(a.counts + 1);
  a.place = reinterpret_cast<int*>(a.bits + words);
  hipError_t e = zero_words(a.bits, words, stream);
  if (e != hipSuccess) return e;
  if (a.F > 0) {
    const int64_t blocks = std::min<int64_t>(((int64_t)a.F + 255) / 256, 2048);
    hipLaunchKernelGGL(compact_mark_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(compact_rank_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, stream, a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t items = (int64_t)a.B * a.M + a.pages + a.F;
  const int64_t blocks = std::min<int64_t>((items + 255) / 256, 4096);
  hipLaunchKernelGGL(compact_apply_kernel, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

}  // namespace fa
