// fa_paged.hip — the paged key/value cache (gfx950): pages and slots of a step's new tokens
// (paged_plan_kernel), their keys and values into the cache (paged_store_kernel), and the
// attention of new tokens over it (paged_fwd_kernel, paged_join_kernel).
//
// The cache holds pages of S tokens (a multiple of 16), [pages, Hkv, S, d]; a sequence's tokens
// 0, 1, ... lie in the pages that its row of the page table names. What the tables, lengths,
// slots and positions hold is on the GPU and is checked here, entry by entry, before an address
// is made of it.
#include <algorithm>
#include <type_traits>

#include "fa_common.hpp"
#include "fa_layer.hpp"

namespace fa {

namespace {

// Inclusive sum over the lanes of a wave, up to this one.
template <class T>
__device__ __forceinline__ T wave_scan(T x, int lane) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const T y = __shfl_up(x, d, 64);
    if (lane >= d) x += y;
  }
  return x;
}

// Two sums over the threads before this one of a block of 256, and the block's totals, behind
// one barrier.
__device__ __forceinline__ void block_scan2(int64_t x, int64_t y, int64_t (*sums)[4],
                                            int64_t* x_before, int64_t* y_before, int64_t* x_all,
                                            int64_t* y_all) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t xi = wave_scan(x, lane), yi = wave_scan(y, lane);
  if (lane == 63) {
    sums[0][wave] = xi;
    sums[1][wave] = yi;
  }
  __syncthreads();
  *x_before = xi - x;
  *y_before = yi - y;
  *x_all = *y_all = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if (w < wave) {
      *x_before += sums[0][w];
      *y_before += sums[1][w];
    }
    *x_all += sums[0][w];
    *y_all += sums[1][w];
  }
}

}  // namespace

// ---- plan -------------------------------------------------------------------------------
// Sequence b holds len_b tokens in ceil(len_b / S) pages and gets new_b more: the pages that
// these need come from the list of free ones, in the order of the sequences, so two running
// sums over the sequences place everything: of new tokens (a token's row in the step) and of
// new pages. Every block takes kPlanTokens tokens and computes the running sums itself, 1024
// sequences at a time in LDS: one launch, and no block waits for another. A thread has OWN
// tokens, 256 apart, whose sequences it finds by bisections side by side. The first token on a
// new page writes the page's table entry. What bounds it is the chain of loads (lengths, then
// page ids) behind the launch: 64 sequences with a token each 4.2 us, 509 with 520 thousand 9.4.
constexpr int kPlanSeqs = 1024;
constexpr int kPlanMost = (1 << 30) - 1;  // largest length and number of new tokens

template <int OWN>
__global__ __launch_bounds__(256) void paged_plan_kernel(PlanArgs a) {
  // Of the group's sequences: the first token in the step, from the group's on; the first new
  // page's place in the free list; the tokens held. Sums past 2^31 - 1 stop there, behind every
  // token and every free page.
  __shared__ int first[kPlanSeqs], place[kPlanSeqs], length[kPlanSeqs];
  __shared__ int64_t sums[2][4];
  const int tid = threadIdx.x;
  const bool head = blockIdx.x == 0;
  const int64_t t0 = (int64_t)blockIdx.x * (256 * OWN);
  const int64_t t1 = min(a.T, t0 + 256 * OWN);
  int64_t tokens = 0;                                  // before this group of sequences
  int64_t pages = a.free_start ? a.free_start[0] : 0;  // place of its first new page
  auto capped = [](int64_t x) { return (int)max(min(x, (int64_t)INT32_MAX), (int64_t)INT32_MIN); };
  for (int b0 = 0; b0 < a.B; b0 += kPlanSeqs) {
    if (tokens >= t1 && !head) return;  // the rest belongs to later blocks
    int len[4], add[4], need[4];
    int64_t n = 0, g = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = b0 + 4 * tid + i;
      len[i] = add[i] = need[i] = 0;
      if (b < a.B) {
        len[i] = min(max(a.lengths[b], 0), kPlanMost);
        add[i] = min(max(a.new_tokens[b], 0), kPlanMost);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int held = (int)(((unsigned)len[i] + a.S - 1) / a.S);
      const int then = (int)(((unsigned)(len[i] + add[i]) + a.S - 1) / a.S);
      need[i] = max(min(then, a.M) - held, 0);  // a row of the table holds M pages
      n += add[i];
      g += need[i];
    }
    int64_t n_all, g_all, n_at, g_at;
    block_scan2(n, g, sums, &n_at, &g_at, &n_all, &g_all);
    g_at += pages;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int b = b0 + 4 * tid + i;
      first[4 * tid + i] = capped(n_at);
      place[4 * tid + i] = capped(g_at);
      length[4 * tid + i] = len[i];
      if (head && b < a.B) {
        a.starts[b] = capped(tokens + n_at);
        a.lengths_out[b] = len[i] + add[i];
      }
      n_at += add[i];
      g_at += need[i];
    }
    __syncthreads();
    // The thread's tokens, from the group's first on, and the last sequence with first <= t,
    // which holds token t.
    const int from = (int)(max(t0, tokens) - tokens) + tid;
    // (none in block 0's later groups, whose distance from its tokens may pass 32 bits)
    const int to = (int)(max(min(t1, tokens + n_all), tokens) - tokens);
    const int count = min(kPlanSeqs, a.B - b0);
    int seq[OWN], pos[OWN], page[OWN], in_page[OWN], entry[OWN];
#pragma unroll
    for (int i = 0; i < OWN; ++i) seq[i] = 0;
    for (int step = kPlanSeqs / 2; step > 0; step >>= 1) {
      if (step >= count) continue;
#pragma unroll
      for (int i = 0; i < OWN; ++i)
        if (seq[i] + step < count && first[seq[i] + step] <= from + 256 * i) seq[i] += step;
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      const int t = from + 256 * i;
      page[i] = entry[i] = -1;
      if (t >= to) continue;
      const int held_tokens = length[seq[i]];
      pos[i] = held_tokens + (t - first[seq[i]]);
      const int j = pos[i] / a.S, held = (int)(((unsigned)held_tokens + a.S - 1) / a.S);
      in_page[i] = pos[i] - j * a.S;
      if (j >= a.M) continue;
      if (j < held) {
        page[i] = a.table[(int64_t)(b0 + seq[i]) * a.table_stride + j];
      } else {
        const int64_t at = (int64_t)place[seq[i]] + (j - held);
        if (at >= 0 && at < a.F) page[i] = a.free_pages[at];
        if (in_page[i] == 0) entry[i] = j;  // the page's first token
      }
    }
#pragma unroll
    for (int i = 0; i < OWN; ++i) {
      if (from + 256 * i >= to) continue;
      const int64_t t = tokens + from + 256 * i;
      if (entry[i] >= 0) a.table[(int64_t)(b0 + seq[i]) * a.table_stride + entry[i]] = page[i];
      a.slots[t] = page[i] < 0 ? -1 : (int64_t)page[i] * a.S + in_page[i];
      a.positions[t] = pos[i];
    }
    tokens += n_all;
    pages += g_all;
    __syncthreads();
  }
  for (int64_t t = max(t0, tokens) + tid; t < t1; t += 256) {  // padding
    a.slots[t] = -1;
    a.positions[t] = 0;
  }
  if (head && tid == 0) {
    a.starts[a.B] = capped(tokens);
    a.free_out[0] = max(capped(pages), 0);
  }
}

template <int OWN>
hipError_t paged_plan_start(const PlanArgs& a, hipStream_t stream) {
  const int64_t blocks = std::max<int64_t>(1, (a.T + 256 * OWN - 1) / (256 * OWN));
  if (blocks > 0x7fffffff) return hipErrorInvalidConfiguration;
  hipLaunchKernelGGL(paged_plan_kernel<OWN>, dim3((unsigned)blocks), dim3(256), 0, stream, a);
  return hipGetLastError();
}

// Two tokens a thread once the blocks of one would not run at once (520 thousand tokens: 9.4 us
// against 11.4; four 10.3); fewer steps behind each other before (64 tokens: 4.2 against 4.5).
hipError_t launch_paged_plan(const PlanArgs& a, hipStream_t stream) {
  return a.T <= 256 * 1024 ? paged_plan_start<1>(a, stream) : paged_plan_start<2>(a, stream);
}

// ---- store ------------------------------------------------------------------------------
// Row t of the keys and values to slot t's row of every head: a copy in 16-byte pieces, bound
// by memory. W neighbouring threads share a token and walk over its 2 H chunks pieces; each
// thread has kStoreTokens tokens in flight. Slots outside the cache are left out. The rows are
// written past the caches: a prompt's attention reads its own keys and values, and until the
// next step reads the cache, the other layers' have passed through (16381 tokens, 14334 of them
// stored, H8 D128: 26.2 -> 19.4 us, 6.0 TB/s; 16384 tokens and at once a step's attention over
// these alone 48.0 -> 51.2). A step's 32 tokens: 3.0 us, with four tokens a thread 3.6.
constexpr int kStoreTokens = 2;

template <int W>
__global__ __launch_bounds__(256) void paged_store_kernel(StoreArgs a) {
  constexpr int TPP = 256 / W;  // tokens of a pass
  const int item = threadIdx.x % W;
  const int64_t t0 = (int64_t)blockIdx.x * (TPP * kStoreTokens) + threadIdx.x / W;
  int64_t page[kStoreTokens];
  int row[kStoreTokens];
#pragma unroll
  for (int i = 0; i < kStoreTokens; ++i) {
    const int64_t t = t0 + i * TPP;
    const int64_t slot = t < a.T ? a.slots[t] : -1;
    page[i] = slot < 0 || slot >= a.pages * a.S ? -1 : slot / a.S;
    row[i] = (int)(slot - page[i] * a.S);
  }
  const int per_side = a.H * a.chunks;
  for (int p = item; p < 2 * per_side; p += W) {
    const int side = p >= per_side;
    const int r = p - side * per_side;
    const int h = r / a.chunks, c = r - h * a.chunks;
    const half_t* src = a.src[side] + h * a.ss[side][1] + 8 * c;
    half_t* dst = a.dst[side] + h * a.ds[1] + 8 * c;
    u32x4 v[kStoreTokens];
#pragma unroll
    for (int i = 0; i < kStoreTokens; ++i)
      if (page[i] >= 0)
        v[i] = *reinterpret_cast<const u32x4*>(src + (t0 + i * TPP) * a.ss[side][0]);
#pragma unroll
    for (int i = 0; i < kStoreTokens; ++i)
      if (page[i] >= 0)
        __builtin_nontemporal_store(
            v[i], reinterpret_cast<u32x4*>(dst + page[i] * a.ds[0] + row[i] * a.ds[2]));
  }
}

hipError_t launch_paged_store(const StoreArgs& args, hipStream_t stream) {
  const int pieces = 2 * args.H * args.chunks;
  const int W = pieces > 128 ? 256 : pieces > 64 ? 128 : pieces > 32 ? 64 : 32;
  const int64_t tokens = 256 / W * kStoreTokens, most = kMostBlocks * tokens;
  for (int64_t t = 0; t < args.T; t += most) {  // tokens past one grid's blocks: another launch
    StoreArgs a = args;
    a.T = std::min(most, args.T - t);
    a.slots += t;
    for (int i = 0; i < 2; ++i) a.src[i] += t * a.ss[i][0];
    const dim3 grid((unsigned)((a.T + tokens - 1) / tokens)), block(256);
    switch (W) {
      case 256: hipLaunchKernelGGL(paged_store_kernel<256>, grid, block, 0, stream, a); break;
      case 128: hipLaunchKernelGGL(paged_store_kernel<128>, grid, block, 0, stream, a); break;
      case 64: hipLaunchKernelGGL(paged_store_kernel<64>, grid, block, 0, stream, a); break;
      default: hipLaunchKernelGGL(paged_store_kernel<32>, grid, block, 0, stream, a); break;
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// ---- attention --------------------------------------------------------------------------
// o = softmax(scale q K^T) V of the group * N query rows that read one key/value head, in
// blocks of 16 rows (one MFMA block) or, where there are more, of 32: query n of a sequence of
// len keys sees keys j <= len - N + n. K and V are read once a row block and next to nothing is
// computed, so what bounds the kernel is reading them: 8 sequences of 32768 keys (Hq32 Hkv8
// D128, 1.07 GB) take 184 us, 5.8 TB/s with the launch in it.
//
// Work is dealt by units of 32 keys. The units of all (sequence, head, row block) triples lie
// on one line, each triple's together; the grid is what the chip holds at once, and every
// work-group takes an equal stretch of that line, found from the lengths on the GPU (the call
// reads no length on the host, so it can be captured). A stretch covers whole triples, which
// are written as they end, and at most one piece at each end of a triple that it shares with
// its neighbours: those go to the workspace as a normalised partial O and a base-2 log-sum-exp,
// and paged_join_kernel joins them. Sequences of any mix of lengths load the chip evenly (Hkv8
// D128, pages that hold head by head: 32 of 17 to 8192 keys, 554 MB, 101 us, where 32 of 4096,
// 537 MB, take 96).
//
// Each row block walks over the keys for itself, also over those that a long chunk's early queries
// do not see: rows past 32 a head are served, far below the matrix unit's rate (4 sequences of 4000
// keys, 64 queries, Hq16 Hkv2 D128 bf16: 40 us).
//
// Within a stretch a work-group's four waves take every fourth unit, each on its own, and
// merge through LDS at the end of a piece. K and V of the next unit are on their way to a
// wave's registers while it works on one (16 KiB a wave at D = 128); K rows come in the layout
// of the MFMA operand, V rows go through a tile in LDS for the transposing reads. Two
// work-groups a CU saturate the memory; a third, for which D = 128 would have to spill, eight
// waves a work-group, a barrier a unit or more work-groups are no faster. A page holds a
// multiple of 16 tokens, so each half unit of 16 keys lies in one page and is read through a
// buffer descriptor of its own, made of its page's 64-bit address, with the half's rows that
// exist as its range: rows past the length read zeros and never reach memory. The pages of a
// wave's next 32 units are kept one a lane.
//
// MFMA layouts (16x16x32, lane l, c16 = l % 16, G = l / 16) as in fa_fwd_decode.hip:
//   S^T block kb: lane holds row c16 and keys 16 kb + 4 G + j of the unit;
//   O^T block dd: lane holds row c16, d = 16 dd + 4 G + j.
// Row r of the triple is query r % N of the group's head r / N.

// A row's probabilities are taken against a reference that moves only when they outgrow a limit.
// fp16 ends at 2^16 and rounds to zero below 2^-25: there the reference is 2^7 below the max, so
// that the many small ones of a long row (2^-26 of the largest, a million times) still count, and
// moves when a lane's eight of a unit sum to more than the type holds. bf16 has room at both ends,
// but values up to 2^128, whose sums in float32 have none: there all probabilities so far are held
// to a sum of 2^-5 a lane, 2^-3 a wave, 1/2 with the four waves, so that no sum of values passes
// the largest of them. The reference moves to 2^16 above the max, or above the sum where many keys
// alike have filled it (8 thousand keys a wave, then once in 2^11 times as many); a weight below
// 2^-110 of the largest is zero. It costs nothing (32 sequences of 17 to 8192 keys 106.3 us with
// sums that are not held).
// The probabilities are rounded to the type for the product with V, as in the dense forward; their
// sums are of the unrounded ones, in float32. Against 64 bits that makes 2.9e-4 (fp16) and 2.2e-3
// (bf16) rel-L2 of what one rounding of the output alone would leave at 2.1e-4 and 1.6e-3; the
// alternative is two products, of a high and a low part.
template <class E>
constexpr bool kPagedWide = std::is_same_v<E, BF16>;
template <class E>
constexpr float kPagedShift = kPagedWide<E> ? -16.f : 7.f;
template <class E>
constexpr float kPagedSumLimit = kPagedWide<E> ? 0.03125f : 32768.f;

constexpr int kPagedWaves = 4;  // of a work-group

template <int D>
struct PagedTile {
  static constexpr int KD = D / 32, DD = D / 16;
  static constexpr int TILE = kPagedUnit * D;          // halves of a unit's K (or V) rows
  static constexpr int VI = TILE * 2 / 1024;           // 1 KiB loads of a unit's V
  static constexpr int VROWS = 512 / D;                // rows of one of them
};

namespace {

// Units of one (head, row block) of a sequence: at least one, which writes the rows of an
// empty sequence. A length that the table cannot hold has one unit too, marked bad.
__device__ __forceinline__ int paged_units(const PagedArgs& a, int len) {
  return len > 0 && len <= a.M * a.S ? (len + kPagedUnit - 1) / kPagedUnit : 1;
}

// Empty units in front of a triple on the line: about what opening and closing a piece takes
// (4 us), in units of the memory's rate. Without them the stretches that cover many short
// sequences end last: 32 sequences of 17 to 8192 keys 110 us (D = 128, none), 106 (3 units),
// 102 (6), 102 (10); where all triples and stretches are equal they cost up to 2 % (95.5 / 96.4).
template <int D>
constexpr int kPagedLead = 768 / D;

// The line of units, cut into stretches of `stretch` units, one a work-group. A triple has its
// own units on the line behind `lead` empty ones, which stand for what opening and closing a
// piece takes; or, in a launch too small to fill the grid (`padded`), its own and empty ones up
// to a whole number of stretches, so that no work-group has two short pieces.
struct PagedLine {
  int total, stretch, lead;
  bool padded;
  __device__ __forceinline__ int units(int own) const {
    return padded ? (own + stretch - 1) / stretch * stretch : lead + own;
  }
};

// A place on it: unit `unit` of triple `triple` (head-major) of sequence `b`, of `len` keys.
struct PagedPlace {
  int b, triple, unit, len;
};

// The line, and its place at stretch `s`, which is defined where the line reaches it. For
// blocks of W waves.
template <int D, int W>
__device__ __forceinline__ PagedLine paged_find(const PagedArgs& a, int s, PagedPlace* place) {
  __shared__ int sums[W][3], found[4];
  const int HB = a.Hkv * a.blocks;
  const int per = (a.B + 64 * W - 1) / (64 * W);
  const int b0 = threadIdx.x * per, b1 = min(a.B, b0 + per);
  constexpr int S1 = kPagedWaves, S2 = 2 * kPagedWaves;  // stretches of padded lines
  // Of the thread's sequences: units on a line that is not padded, stretches on the padded ones.
  int own[3] = {0, 0, 0}, first[3], all[3];
  for (int b = b0; b < b1; ++b) {
    const int u = paged_units(a, a.lengths[b]);
    own[0] += (u + kPagedLead<D>) * HB;
    own[1] += (u + S1 - 1) / S1 * HB;
    own[2] += (u + S2 - 1) / S2 * HB;
  }
  block_scan<W>(own, sums, first, all);
  PagedLine line;
  line.padded = all[2] <= a.grid;
  int before, mine;
  if (line.padded) {
    const int i = all[1] <= a.grid ? 1 : 2;
    line.lead = 0;
    line.stretch = i == 1 ? S1 : S2;
    line.total = (i == 1 ? all[1] : all[2]) * line.stretch;
    before = (i == 1 ? first[1] : first[2]) * line.stretch;
    mine = (i == 1 ? own[1] : own[2]) * line.stretch;
  } else {
    line.lead = kPagedLead<D>;
    line.total = all[0];
    line.stretch = (line.total + a.grid - 1) / a.grid;
    before = first[0];
    mine = own[0];
  }
  const int64_t at = (int64_t)s * line.stretch;
  if (at >= before && at < (int64_t)before + mine) {
    int rest = (int)(at - before), b = b0, len = 0, units = 1;
    for (; b < b1; ++b) {
      len = a.lengths[b];
      units = line.units(paged_units(a, len));
      if (rest < units * HB) break;
      rest -= units * HB;
    }
    found[0] = b;
    found[1] = rest / units;
    found[2] = rest % units;
    found[3] = len;
  }
  __syncthreads();
  place->b = uniform(found[0]);
  place->triple = uniform(found[1]);
  place->unit = uniform(found[2]);
  place->len = uniform(found[3]);
  return line;
}

// The triple that the end of a work-group's stretch cuts, where that is the triple's first cut:
// `more` pieces follow the work-group's own, which is in its slot `slot`; more = 0 where there
// is no such triple. The workspace holds one of these for each work-group, then two partials
// for each: a row block's rows of O, then their log-sum-exps.
struct PagedCut {
  int b, triple, more, slot;
};
template <int D>
__device__ __forceinline__ float* paged_part(const PagedArgs& a, int64_t slot) {
  return a.part + a.grid * (sizeof(PagedCut) / 4) + slot * (a.rows * (D + 1));
}

// A row of a triple: query n of the group's head h, if it exists; and its row of the output.
struct PagedRow {
  bool ok;
  int h, n;
};
__device__ __forceinline__ int64_t paged_out_row(const PagedArgs& a, int b, int kvh,
                                                 const PagedRow& r) {
  return ((int64_t)(b * (int64_t)a.Hkv + kvh) * a.group + r.h) * a.N + r.n;
}

}  // namespace

template <int D, class E, int RB, bool SHORT>
__global__ __launch_bounds__(64 * kPagedWaves, 2) void paged_fwd_kernel(PagedArgs a) {
  using T = PagedTile<D>;
  constexpr int KD = T::KD, DD = T::DD, NW = kPagedWaves;
  constexpr int ROWS = 16 * RB;
  constexpr int LDS_FLOATS = NW * RB * DD * 256 + 2 * NW * ROWS;
  static_assert(NW * T::TILE * 2 <= LDS_FLOATS * 4, "the V tiles and the merge share it");
  __shared__ __attribute__((aligned(16))) float lds[LDS_FLOATS];
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int c16 = lane & 15;
  const int G = lane >> 4;

  // The work-group's stretch. Where the rows of neighbouring heads share 128-byte lines, an XCD
  // takes consecutive stretches, so that its L2 holds a line for both (39 sequences of 1710 to
  // 3420 keys, Hkv8 D32, pages that hold token by token: 38.9 -> 32.0 us); elsewhere those are
  // better spread (32 sequences of 4096 keys, Hkv8 D128, token by token: 99.3 against 103.7).
  const bool lines_shared = D <= 64 && !SHORT && a.Hkv > 1 && a.ks[1] < 64 && a.grid % 8 == 0;
  const int s_at = lines_shared ? (int)(blockIdx.x % 8) * (a.grid / 8) + (int)(blockIdx.x / 8)
                                : (int)blockIdx.x;
  // It is `left` units from the place on. In a SHORT launch a triple of its own.
  PagedPlace at;
  int left;
  int lead = 0, stretch = 0;
  bool padded = true;
  PagedCut* const cut = reinterpret_cast<PagedCut*>(a.part) + s_at;
  if constexpr (SHORT) {
    at.b = blockIdx.x / (a.Hkv * a.blocks);
    at.triple = blockIdx.x - at.b * (a.Hkv * a.blocks);
    at.unit = 0;
    at.len = uniform(a.lengths[at.b]);
    left = INT32_MAX;
  } else {
    const PagedLine line = paged_find<D, NW>(a, s_at, &at);
    const int64_t from = (int64_t)s_at * line.stretch;
    if (tid == 0) cut->more = 0;
    if (from >= line.total) return;
    left = min(line.stretch, (int)(line.total - from));
    stretch = line.stretch;
    padded = line.padded;
    lead = line.lead;
  }
  bool opening = true;  // the stretch's first piece

  half_t* const vt = reinterpret_cast<half_t*>(lds) + wave * T::TILE;
  const int row_bytes = (int)a.ks[2] * 2;
  uint32_t k_off[KD], v_off[T::VI], v_at[T::VI];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    const int col = 32 * kd + 8 * G;
    k_off[kd] = col < a.d ? (uint32_t)(c16 * row_bytes + col * 2) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < T::VI; ++i) {
    const int row = i * T::VROWS + lane / (D / 8), chunk = lane % (D / 8);
    v_off[i] = 8 * chunk < a.d ? (uint32_t)((row & 15) * row_bytes + chunk * 16) : kOutOfRange;
    v_at[i] = (uint32_t)swz_offset<D>(row, chunk);
  }
  int t_off[DD];
#pragma unroll
  for (int dd = 0; dd < DD; ++dd) {
    const int row = 4 * G + (c16 >> 2), col = 16 * dd + 4 * (c16 & 3);
    t_off[dd] = row * D + 8 * swz_chunk<D>(row, col >> 3) + (col & 7);
  }

  while (true) {
    const int len = at.len;
    const bool fits = len >= 0 && len <= a.M * a.S;
    const int keys = fits ? len : 0;
    const int units = paged_units(a, len);
    const int u0 = max(at.unit - lead, 0);
    const int line_units = lead + units;
    const int u1 = left < line_units - at.unit ? max(at.unit + left - lead, 0) : units;
    if (u1 <= u0) return;  // the stretch ends before the triple's first unit
    const int kvh = at.triple / a.blocks, block = at.triple - kvh * a.blocks;
    const int rows = a.group * a.N;

    // The lane's rows. Each sees the keys below see[]; rows that do not exist score 0
    // everywhere: masked, they would move the reference max in every unit.
    auto row_of = [&](int rb) __attribute__((always_inline)) {
      const int r = block * ROWS + 16 * rb + c16;
      return PagedRow{r < rows, r / a.N, r % a.N};
    };
    const int all_see = keys - a.N + 1;  // every row sees the keys below this
    int see[RB];
    half8 qf[RB][KD];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const PagedRow r = row_of(rb);
      see[rb] = r.ok ? all_see + r.n : INT32_MAX;
      const half_t* q = a.q + at.b * a.qs[0] + (int64_t)(kvh * a.group + r.h) * a.qs[1] + r.n * a.qs[2];
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) {
        u32x4 v = {0u, 0u, 0u, 0u};
        const int col = 32 * kd + 8 * G;
        if (r.ok && col < a.d) v = *reinterpret_cast<const u32x4*>(q + col);
        qf[rb][kd] = __builtin_bit_cast(half8, v);
      }
    }

    // Unit i of the wave is u0 + wave + 4 i.
    const int mine = u1 - u0 > wave ? (u1 - u0 - wave + NW - 1) / NW : 0;
    const half_t* const k_head = a.k + kvh * a.ks[1];
    const half_t* const v_head = a.v + kvh * a.ks[1];
    bool bad = !fits;
    // The page of half unit lane & 1 of unit i0 + lane / 2, and its first row there.
    auto half_key = [&](int i0) __attribute__((always_inline)) {
      return (u0 + wave + NW * (i0 + (lane >> 1))) * kPagedUnit + 16 * (lane & 1);
    };
    auto half_page = [&](int i0) __attribute__((always_inline)) {
      const int key = half_key(i0);
      return i0 + (lane >> 1) < mine && key < keys
                 ? a.table[at.b * a.table_stride + key / a.S] : 0;
    };
    int page = half_page(0), row = half_key(0) % a.S;  // of the units from i & ~31 on
    int next_page = half_page(32);

    u32x4 kx[2][KD], vx[T::VI];
    int64_t off[2];
    uint32_t bytes[2];
    // Where unit i lies; its K and its V on their way to the registers. Past the wave's last
    // unit, and in pages that do not exist, no rows.
    auto turn_to = [&](int i) __attribute__((always_inline)) {
      if ((i & 31) == 0 && i > 0) {
        page = next_page;
        row = half_key(i) % a.S;
        next_page = half_page(i + 32);
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int there = keys - ((u0 + wave + NW * i) * kPagedUnit + 16 * e);
        const int pg = __builtin_amdgcn_readlane(page, 2 * (i & 31) + e);
        const bool any = i < mine && there > 0, known = pg >= 0 && pg < a.pages;
        bad |= any && !known;
        off[e] = pg * a.ks[0] + __builtin_amdgcn_readlane(row, 2 * (i & 31) + e) * a.ks[2];
        bytes[e] = any && known ? (uint32_t)((min(there, 16) - 1) * row_bytes + a.d * 2) : 0u;
      }
    };
    auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const rsrc_t r_k = make_rsrc(k_head + off[e], bytes[e]);
#pragma unroll
        for (int kd = 0; kd < KD; ++kd) kx[e][kd] = buf_load_b128(r_k, k_off[kd]);
      }
    };
    auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int j = 0; j < T::VI; ++j) {
        const int e = j * T::VROWS / 16;
        const rsrc_t r_v = make_rsrc(v_head + off[e], bytes[e]);
        vx[j] = buf_load_b128(r_v, v_off[j]);
      }
    };

    float4v o[RB][DD];
    float m[RB], l[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
      for (int dd = 0; dd < DD; ++dd) o[rb][dd] = {0.f, 0.f, 0.f, 0.f};
      m[rb] = -INFINITY;
      l[rb] = 0.f;
    }
    const float c = a.c;

    turn_to(0);
    load_k();
    load_v();
    for (int i = 0; i < mine; ++i) {
      const int ka = (u0 + wave + NW * i) * kPagedUnit;
      float4v s[RB][2];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          s[rb][kb] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int kd = 0; kd < KD; ++kd)
            s[rb][kb] = mma16<E>(__builtin_bit_cast(half8, kx[kb][kd]), qf[rb][kd], s[rb][kb]);
        }
      turn_to(i + 1);  // past the last unit: no rows
      load_k();
#pragma unroll
      for (int j = 0; j < T::VI; ++j) *reinterpret_cast<u32x4*>(vt + v_at[j]) = vx[j];
      load_v();
      half8 pa[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        if (ka + kPagedUnit > all_see) {
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (ka + 16 * kb + 4 * G + j >= see[rb]) s[rb][kb][j] = -INFINITY;
        }
        auto probs = [&](float ref) __attribute__((always_inline)) {
          float sum = 0.f;
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float p = exp2_fast(fmaf(s[rb][kb][j], c, -ref));
              sum += p;
              pa[rb][4 * kb + j] = to_elem<E>(p);
            }
          return sum;
        };
        // The probabilities' sum, and what the limit holds: this unit's, or all so far.
        float l_u = probs(m[rb]);
        const float held = kPagedWide<E> ? l[rb] + l_u : l_u;
        if (__builtin_amdgcn_ballot_w64(!(held <= kPagedSumLimit<E>)) != 0) {
          float mt = s[rb][0][0];
#pragma unroll
          for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int j = 0; j < 4; ++j) mt = __builtin_fmaxf(mt, s[rb][kb][j]);
          float m_new = __builtin_fmaxf(m[rb], quarters_max(mt) * c - kPagedShift<E>);
          if constexpr (kPagedWide<E>)
            m_new = __builtin_fmaxf(m_new, m[rb] + log2_fast(quarters_max(l[rb])) - kPagedShift<E>);
          const float ref = exp_reference(m_new);
          const float alpha = exp2_fast(m[rb] - ref);
          l[rb] *= alpha;
#pragma unroll
          for (int dd = 0; dd < DD; ++dd) o[rb][dd] *= alpha;
          m[rb] = m_new;
          l_u = probs(ref);
        }
        l[rb] += l_u;
      }
#pragma unroll
      for (int dd = 0; dd < DD; ++dd) {
        const half4 lo = __builtin_bit_cast(
            half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vt + t_off[dd])));
        const half4 hi = __builtin_bit_cast(
            half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vt + t_off[dd] + 16 * D)));
        half8 va;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          va[e] = lo[e];
          va[4 + e] = hi[e];
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) o[rb][dd] = mma16<E>(va, pa[rb], o[rb][dd]);
      }
    }

    // Merge of the waves' results: O, and per row m and l.
    __syncthreads();
    float* const xo = lds;                        // [wave][row block][dd][lane][4]
    float* const xm = lds + NW * RB * DD * 256;   // [wave][row], m then l
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float lw = quarters_sum(l[rb]), mw = m[rb];
      if (bad) {  // NaN, whatever the other waves and pieces hold
        lw = __builtin_nanf("");
        mw = mw == -INFINITY ? 0.f : mw;
      }
#pragma unroll
      for (int dd = 0; dd < DD; ++dd)
        *reinterpret_cast<float4v*>(xo + (((wave * RB + rb) * DD + dd) * 64 + lane) * 4) = o[rb][dd];
      if (G == 0) {
        xm[wave * ROWS + 16 * rb + c16] = mw;
        xm[(NW + wave) * ROWS + 16 * rb + c16] = lw;
      }
    }
    __syncthreads();
    const bool whole = SHORT || (u0 == 0 && u1 == units);
    float* const part = paged_part<D>(a, (int64_t)s_at * 2 + (opening ? 0 : 1));
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const int x = 16 * rb + c16;
      float mt = -INFINITY;
#pragma unroll
      for (int w = 0; w < NW; ++w) mt = __builtin_fmaxf(mt, xm[w * ROWS + x]);
      float wt[NW], lt = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const float mw = xm[w * ROWS + x];
        wt[w] = mw == -INFINITY ? 0.f : exp2_fast(mw - mt);  // a wave that saw no key weighs 0
        lt += wt[w] * xm[(NW + w) * ROWS + x];
      }
      const float inv = lt == 0.f ? 0.f : 1.0f / lt;  // a row that saw no key is 0
      const PagedRow r = row_of(rb);
      half_t* const out = a.o + paged_out_row(a, at.b, kvh, r) * a.d;
#pragma unroll
      for (int dd = wave; dd < DD; dd += NW) {
        float4v v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w)
          v += *reinterpret_cast<const float4v*>(xo + (((w * RB + rb) * DD + dd) * 64 + lane) * 4) *
               wt[w];
        v *= inv;
        const int col = 16 * dd + 4 * G;
        if (!r.ok) continue;
        if (!whole) *reinterpret_cast<float4v*>(part + x * D + col) = v;
        else if (col < a.d)
          *reinterpret_cast<u32x2*>(out + col) = pack4<E>(v[0], v[1], v[2], v[3]);
      }
      if (!whole && wave == 0 && G == 0 && r.ok)
        part[ROWS * D + x] = lt == 0.f ? -INFINITY : mt + log2_fast(lt);
    }
    __syncthreads();

    left -= line_units - at.unit;
    if (!SHORT && tid == 0 && u0 == 0 && u1 < units)  // the triple goes on in other stretches
      *cut = {at.b, at.triple, (stretch - 1 - left) / stretch, opening ? 0 : 1};
    if (padded || left <= 0) return;
    opening = false;
    at.unit = 0;
    if (++at.triple == a.Hkv * a.blocks) {
      at.triple = 0;
      ++at.b;
      at.len = uniform(a.lengths[at.b]);
    }
  }
}

// Joins the pieces of the triples that the ends of the stretches cut: block (w, y) rows of the
// triple that work-group w's cut names. Piece p of a row weighs exp2(lse_p) against the others'.
// A lane holds four columns of a row, a wave RPP rows; of a block's four waves `groups` take
// different rows, and the 4 / groups waves that share theirs take every (4 / groups)-th piece
// and merge through LDS, in a fixed order. Most blocks have two pieces to join or none, and all
// is latency: each wave asks for its first piece beside the cut that says whether it exists.
constexpr int kJoinWaves = 4;
template <int D>
constexpr int kJoinRows = 64 / (D / 4);  // of a wave
// The weight of a row's largest piece: those of 512 pieces, the most there are, sum to 1/2, so
// that sums of values near 2^128 stay in float32.
constexpr float kJoinWeight = 0x1p-10f;

inline __host__ __device__ int join_groups(int rows, int wave_rows) {
  return rows <= wave_rows ? 1 : rows <= 2 * wave_rows ? 2 : 4;
}

template <int D, class E>
__global__ __launch_bounds__(64 * kJoinWaves) void paged_join_kernel(PagedArgs a) {
  constexpr int W = kJoinWaves;
  constexpr int COLS = D / 4;           // 4-column pieces of a row
  constexpr int RPP = kJoinRows<D>;
  constexpr int AHEAD = 8;              // pieces of a wave asked for at once
  __shared__ __attribute__((aligned(16))) float acc_s[W][64][4];
  __shared__ float m_s[W][64], l_s[W][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int w = blockIdx.x;
  const int groups = join_groups(min(a.rows, a.group * a.N), RPP);
  const int group = wave % groups, part0 = wave / groups, step = W / groups;
  const int row = (blockIdx.y * groups + group) * RPP + lane / COLS, col = 4 * (lane % COLS);
  struct Piece {
    float lse;
    float4v o;
  };
  const bool held = row < a.rows;  // the partials hold such a row
  auto load = [&](int64_t slot) __attribute__((always_inline)) {
    Piece p = {-INFINITY, {0.f, 0.f, 0.f, 0.f}};
    if (held) {
      const float* part = paged_part<D>(a, slot);
      p.lse = part[a.rows * D + row];
      p.o = *reinterpret_cast<const float4v*>(part + row * D + col);
    }
    return p;
  };
  // Slot 0 of the work-group part0 behind w (of w itself also slot 1): inside the workspace,
  // and unused unless the cut says that it was written.
  const int64_t ahead = min(w + part0, a.grid - 1);
  const PagedCut cut = reinterpret_cast<const PagedCut*>(a.part)[w];
  Piece p0 = load(2 * ahead);
  if (part0 == 0) {
    const Piece p1 = load(2 * ahead + 1);
    if (cut.slot != 0) p0 = p1;
  }
  if (cut.more == 0) return;
  const int kvh = cut.triple / a.blocks, block = cut.triple - kvh * a.blocks;
  const int rows = min(a.rows, a.group * a.N - block * a.rows);
  float m = -INFINITY, l = 0.f;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  if (part0 <= cut.more) {
    m = p0.lse;
    l = m == -INFINITY ? 0.f : kJoinWeight;
    acc = p0.o * kJoinWeight;
    for (int at = part0 + step; at <= cut.more; at += step * AHEAD) {
      Piece p[AHEAD];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        p[i] = at + step * i <= cut.more ? load(2 * ((int64_t)w + at + step * i))
                                         : Piece{-INFINITY, {0.f, 0.f, 0.f, 0.f}};
      float mx = m;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) mx = __builtin_fmaxf(mx, p[i].lse);
      const float ref = exp_reference(mx);
      const float keep = m == -INFINITY ? 0.f : exp2_fast(m - ref);
      l *= keep;
      acc *= keep;
#pragma unroll
      for (int i = 0; i < AHEAD; ++i) {
        const float f = p[i].lse == -INFINITY ? 0.f : exp2_fast(p[i].lse - ref) * kJoinWeight;
        l += f;
        acc += p[i].o * f;
      }
      m = mx;
    }
  }
  *reinterpret_cast<float4v*>(acc_s[wave][lane]) = acc;
  m_s[wave][lane] = m;
  l_s[wave][lane] = l;
  __syncthreads();
  if (part0 != 0 || row >= rows || col >= a.d) return;
  float mx = -INFINITY;
  for (int i = group; i < W; i += groups) mx = __builtin_fmaxf(mx, m_s[i][lane]);
  float lt = 0.f;
  float4v v = {0.f, 0.f, 0.f, 0.f};
  for (int i = group; i < W; i += groups) {
    const float f = m_s[i][lane] == -INFINITY ? 0.f : exp2_fast(m_s[i][lane] - mx);
    lt += f * l_s[i][lane];
    v += *reinterpret_cast<const float4v*>(acc_s[i][lane]) * f;
  }
  v *= lt == 0.f ? 0.f : 1.0f / lt;
  const int r = block * a.rows + row;
  half_t* out = a.o + paged_out_row(a, cut.b, kvh, {true, r / a.N, r % a.N}) * a.d;
  *reinterpret_cast<u32x2*>(out + col) = pack4<E>(v[0], v[1], v[2], v[3]);
}

// Where a sequence's row of the table holds few keys, a work-group takes a whole triple: no
// line, no partials and no second launch. It reads at most 61 bytes a ns, what one CU draws
// from HBM (four units in 1.07 us at D = 128; eight waves are no faster), so the bound is about
// where that takes as long as a second launch saves: D = 128, B x Hkv 8 / 64 / 256 triples, us,
// this / split and joined (kernels alone; the second launch adds about 1.5):
//   512 keys   8.9 / 11.3   9.3 / 13.2  13.6 / 20.2
//   1024 keys 13.5 / 10.4  13.8 / 16.3  25.8 / 34.3
//   2048 keys 21.1 / 11.0  21.9 / 20.1  47.7 / 57.3
// At 1024 keys the bound favours the 64 triples and more of a batch: 8 triples would end 1.6 us
// earlier split. A longer row may hold one long sequence among short ones, whose time the split
// shares out. The lengths are on the GPU, so the table's width decides: sequences that are short
// for their table take the split, 257 keys in a table of 8192 (8, 64, 256 triples) 7.7 + 3.6,
// 8.4 + 3.5 and 13.7 + 4.0 us, against 6.9, 7.2 and 9.7 in a table of 272.
// More triples than a grid has blocks take the split launch, whose work-groups walk over them.
bool paged_short(int64_t triples, int64_t keys) {
  return triples <= kMostBlocks && (keys <= 1024 || (keys <= 2048 && triples >= 256));
}

// Two work-groups a CU, at most one for each four units that the tables could hold; 0: a
// work-group for each triple.
int paged_grid(int64_t B, int64_t Hkv, int64_t blocks, int64_t keys) {
  const int64_t triples = B * Hkv * blocks;
  if (paged_short(triples, keys)) return 0;
  const int64_t units = triples * ((keys + kPagedUnit - 1) / kPagedUnit);
  return (int)std::min<int64_t>((units + 3) / 4, 512);
}

template <int D, class E, int RB>
hipError_t paged_start(const PagedArgs& a, hipStream_t stream) {
  if (a.grid == 0) {
    const int64_t triples = (int64_t)a.B * a.Hkv * a.blocks;
    hipLaunchKernelGGL((paged_fwd_kernel<D, E, RB, true>), dim3((unsigned)triples),
                       dim3(64 * kPagedWaves), 0, stream, a);
    return hipGetLastError();
  }
  hipLaunchKernelGGL((paged_fwd_kernel<D, E, RB, false>), dim3((unsigned)a.grid),
                     dim3(64 * kPagedWaves), 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int rows = std::min(a.rows, a.group * a.N);
  const int block_rows = kJoinRows<D> * join_groups(rows, kJoinRows<D>);
  const dim3 grid((unsigned)(a.grid - 1), (unsigned)((rows + block_rows - 1) / block_rows));
  hipLaunchKernelGGL((paged_join_kernel<D, E>), grid, dim3(64 * kJoinWaves), 0, stream, a);
  return hipGetLastError();
}

template <int D, class E>
hipError_t paged_start(const PagedArgs& a, hipStream_t stream) {
  return a.rows == 16 ? paged_start<D, E, 1>(a, stream) : paged_start<D, E, 2>(a, stream);
}

hipError_t launch_paged_fwd(const PagedArgs& a, int D, int dtype, hipStream_t stream) {
  const bool bf = dtype == kBF16;
  switch (D) {
    case 32: return bf ? paged_start<32, BF16>(a, stream) : paged_start<32, F16>(a, stream);
    case 64: return bf ? paged_start<64, BF16>(a, stream) : paged_start<64, F16>(a, stream);
    case 128: return bf ? paged_start<128, BF16>(a, stream) : paged_start<128, F16>(a, stream);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace fa
