// fa_layer.hpp — argument blocks and launchers of the operators around the attention call
// (fa_rope.hip, fa_paged.hip), shared with their C ABI (fa_capi_layer.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fa_kernels.hpp"

namespace fa {

// ---- errors (defined in fa_capi.hip) ----------------------------------------------------
// Records the calling thread's message for fa_last_error() and returns `code`.
int capi_fail(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));
// FA_OK, or the hipError_t of a launch of the entry point `name` with its message.
int capi_launch_result(hipError_t e, const char* name);

// Blocks of 256 threads along a grid's first axis: HIP takes fewer than 2^32 threads there.
constexpr int64_t kMostBlocks = 0xffffffff / 256;

// ---- sums over a block's threads --------------------------------------------------------

// Inclusive sum over the lanes of a wave, up to this one, by DPP: no trip through the LDS unit.
__device__ __forceinline__ int wave_scan(int x) {
#define FA_SCAN_STEP(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xF, false)
  FA_SCAN_STEP(0x111, 0xF);  // row_shr 1, 2, 4, 8: within 16 lanes
  FA_SCAN_STEP(0x112, 0xF);
  FA_SCAN_STEP(0x114, 0xF);
  FA_SCAN_STEP(0x118, 0xF);
  FA_SCAN_STEP(0x142, 0xA);  // row_bcast 15 to rows 1 and 3, then 31 to rows 2 and 3
  FA_SCAN_STEP(0x143, 0xC);
#undef FA_SCAN_STEP
  return x;
}

// Sums over the threads before this one of a block of W waves (before[i] of x[i]) and the
// block's totals (all[i]), behind one barrier.
template <int W, int K>
__device__ __forceinline__ void block_scan(const int (&x)[K], int (*sums)[K], int (&before)[K],
                                           int (&all)[K]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int incl[K];
#pragma unroll
  for (int i = 0; i < K; ++i) incl[i] = wave_scan(x[i]);
  if (lane == 63)
#pragma unroll
    for (int i = 0; i < K; ++i) sums[wave][i] = incl[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < K; ++i) {
    before[i] = incl[i] - x[i];
    all[i] = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      if (w < wave) before[i] += sums[w][i];
      all[i] += sums[w][i];
    }
  }
}

// ---- norm and rotation of queries and keys ----------------------------------------------

// One of the two tensors, [B, H, N, D] with strides in elements (multiples of 8).
struct RopeSide {
  const half_t* x;   // the input rows (the backward of a plain rotation: null)
  const half_t* g;   // backward: gradient of the output
  half_t* out;       // the output, or the input's gradient: contiguous [B, H, N, D]
  const void* w;     // norm weight [D], 16-bit or fp32 (null without norms)
  float* part;       // backward: partial weight gradients [blocks, D], null to leave them out
  int64_t xs[3];     // batch, head and row stride of x
  int64_t gs[3];     // and of g
  int H;
  int chunks;        // head chunks of the launch (blockIdx.y), filled in by the launcher
};

struct RopeArgs {
  RopeSide side[2];      // queries, keys
  const float* cos;      // [P, R / 2], contiguous
  const float* sin;
  const void* pos;       // int32 or int64 positions, null for 0 .. N - 1
  int64_t pos_sb, pos_sn;
  int64_t T;             // B * N tokens
  int64_t P;             // rows of cos and sin
  int N, D, R;
  int heads;             // heads of a chunk, filled in by the launcher
  uint32_t first;        // forward: the launch's first token, filled in by the launcher
  int pos64, w32;        // positions are int64; weights are fp32
  float eps;
};

// Bytes of the backward's partial weight gradients (fp32, [blocks, D]).
int64_t rope_workspace_bytes(int64_t T, int D, int Hq, int Hkv);
hipError_t launch_rope(const RopeArgs& args, int dtype, bool norm, bool interleaved,
                       hipStream_t stream);
// dw: the two weight gradients, in the weights' type (null to leave one out); part: the
// workspace (unused without weight gradients).
hipError_t launch_rope_bwd(const RopeArgs& a, int dtype, bool norm, bool interleaved,
                           void* const dw[2], float* part, hipStream_t stream);

// ---- the paged key/value cache ----------------------------------------------------------

// Pages and slots of a step's new tokens (paged_plan_kernel).
struct PlanArgs {
  int* table;             // [B, M], rows table_stride apart; entries of new pages are written
  const int* lengths;     // [B] tokens held
  const int* new_tokens;  // [B]
  const int* free_pages;  // [F]
  const int* free_start;  // first free page's place in free_pages, null for 0
  int64_t* slots;         // [T]
  int* positions;         // [T]
  int* starts;            // [B + 1]
  int* lengths_out;       // [B]
  int* free_out;          // [1]
  int64_t table_stride;
  int64_t T;
  int B, M, F, S;
};
hipError_t launch_paged_plan(const PlanArgs& a, hipStream_t stream);

// A cache tensor [pages, H, S, D] (or the tokens' [T, H, D], S = 1), strides in elements.
struct StoreArgs {
  const half_t* src[2];  // keys, values
  half_t* dst[2];
  const int64_t* slots;
  int64_t ss[2][2];      // token and head stride of each source
  int64_t ds[3];         // page, head and row stride of the caches
  int64_t T, pages;
  int H, S, chunks;      // chunks: 16-byte pieces of a row
};
hipError_t launch_paged_store(const StoreArgs& a, hipStream_t stream);

// The attention of N new tokens a sequence over the paged cache (paged_fwd_kernel).
struct PagedArgs {
  const half_t* q;       // [B, Hq, N, d], strides qs
  const half_t* k;       // [pages, Hkv, S, d], strides ks; v the same
  const half_t* v;
  const int* table;      // [B, M], rows table_stride apart
  const int* lengths;    // [B]
  half_t* o;             // contiguous [B, Hq, N, d]
  float* part;           // partials of the pieces that share a row block (null: none do)
  int64_t qs[3];         // batch, head and row stride, elements
  int64_t ks[3];         // page, head and row stride
  int64_t table_stride;
  int64_t pages;
  float c;               // scale * log2(e)
  int B, Hkv, group, N, d, M, S;
  int rows;              // of a row block: 16 or 32 (paged_rows)
  int blocks;            // row blocks of a key/value head's group * N rows
  int grid;              // work-groups (paged_grid)
};
constexpr int kPagedUnit = 32;  // keys
// Rows of the blocks that `rows` rows are worked on in.
inline int paged_rows(int64_t rows) { return rows <= 16 ? 16 : 32; }
// Work-groups of a launch whose table rows hold `keys` keys; 0: one for each sequence,
// key/value head and row block.
int paged_grid(int64_t B, int64_t Hkv, int64_t blocks, int64_t keys);
hipError_t launch_paged_fwd(const PagedArgs& a, int D, int dtype, hipStream_t stream);

// ---- pages that sequences share -----------------------------------------------------------

// Row b of the page table becomes row parents[b] (fork_count_kernel).
struct ForkArgs {
  int* table;             // [B, M], rows table_stride apart
  const int* lengths;     // [B]
  const int* parents;     // [B]
  int* free_pages;        // [F]
  const int* free_start;  // null for 0
  int* shares;            // [pages], entries that hold a page beyond the first
  int* lengths_out;       // [B]; the copies that the rows need, -1 and 0 where they need none:
  int* sources;
  int* targets;
  int* tokens;
  int* free_out;          // [1]
  int64_t table_stride;
  int B, M, F, S, pages;
  // the workspace, and blocks a row, filled in by the launcher
  int* keeper;            // [B], the child that goes on in the row's begun page
  unsigned* bits;         // pages whose count fell below zero
  int* children;          // [B], and [B] that say which comes first (fork_children_kernel)
  int* rows;              // [B, M], the new rows
  int parts;
};
int64_t fork_workspace_bytes(int64_t B, int64_t M, int64_t pages);
hipError_t launch_fork(const ForkArgs& a, void* workspace, hipStream_t stream);

// Pages of the caches [pages, H, S, D] into others (page_copy_kernel), strides in elements.
struct CopyArgs {
  half_t* k;
  half_t* v;
  const int* sources;  // [n]
  const int* targets;
  const int* tokens;   // rows that are copied, null for all
  int64_t ks[3];       // page, head and row stride of both
  int64_t n, pages;
  int H, S, chunks;    // chunks: 16-byte pieces of a row
  // filled in by the launcher: blocks a pair, whether rows lie closer than heads, and without gaps
  unsigned blocks;
  int rows_inside, together;
};
hipError_t launch_page_copy(const CopyArgs& a, hipStream_t stream);

// Held pages move to the front of the cache (compact_rank_kernel).
struct CompactArgs {
  const int* table;       // [B, M], rows table_stride apart
  const int* free_pages;  // [F]
  const int* free_start;  // null for 0
  const int* shares;      // [pages]
  int* table_out;         // contiguous [B, M]
  int* free_pages_out;    // [F]
  int* shares_out;        // [pages]
  int* sources;           // [F], the moves, -1 behind the last
  int* targets;
  int* used;              // [1], held pages
  int64_t table_stride;
  int B, M, F, pages;
  // the workspace, filled in by the launcher
  int* counts;            // [1], moves
  unsigned* bits;         // free pages
  int* chunks;            // [pages / 1024 + 1], the free pages in front of each 1024, and all
  int* place;             // [pages], a moved page's place among the moves
};
int64_t compact_workspace_bytes(int64_t pages);
hipError_t launch_compact(const CompactArgs& a, void* workspace, hipStream_t stream);

// ---- attention where groups of sequences share a prefix (prefix_fwd_kernel) ----------------

struct PrefixArgs {
  const half_t* q;       // [B, Hq, N, d], strides qs
  const half_t* k;       // [pages, Hkv, S, d], strides ks; v the same
  const half_t* v;
  const int* table;      // [B, M], rows table_stride apart
  const int* lengths;    // [B]
  const int* starts;     // [G + 1], the groups' first sequences and the end of the last
  const int* prefix;     // [G], keys of the groups' prefixes
  half_t* o;             // contiguous [B, Hq, N, d]
  int* ws;               // four ints, then from int 16 on the join's PrefixSeq [B], PrefixGroup [G]
  float* part;           // partials: pslots slots of prows rows, then those of srows rows
  int64_t qs[3];         // batch, head and row stride, elements
  int64_t ks[3];         // page, head and row stride
  int64_t table_stride;
  int64_t pages;
  int64_t pslots;
  float c;               // scale * log2(e)
  int B, G, Hkv, group, N, d, M, S;
  int R;                 // rows of a sequence that read a key/value head: group * N
  int blocks;            // tiles of them
  int prows, srows;      // rows of a prefix's and of a sequence's own slot
  int grid;              // work-groups
  int most_pieces;       // of long prefixes
};
// Where a sequence's own units lie on the line of units, and its group and its place in it.
struct PrefixSeq {
  int own_base, own_units, group, member;
};
// Where a group's units lie on the line and which of the line's triples is its first, or which of the
// long prefixes' pieces, `cuts` a triple.
struct PrefixGroup {
  int base, units, first, tiles, cuts, pad[3];
};
constexpr int kPrefixTile = 128;   // query rows of a tile
constexpr int kPrefixLead = 6;     // empty units in front of a triple on the line
// Least units of a work-group. (4 beams over 512 shared keys, Hq32 Hkv8 D128: 16.4 us, with 2 16.9, with 8
// 17.6.)
constexpr int kPrefixStretch = 4;
// Groups (fewer) and sequences whose lengths and starts a work-group keeps in LDS.
constexpr int kPrefixKeptGroups = 1024, kPrefixKeptSeqs = 2048;
// Most rows of a sequence whose own keys are a wave's work, the rows of a tile there, and the empty units
// in front of a triple. (From 33 rows on the keys are read once a tile; the other way is a work-group for
// up to 128 rows. Which is faster goes by the keys, Hkv4 D128 bf16, this and the other: 100 sequences of
// 48 rows and up to 100 keys of their own 79 us and 85; 24 of 40 rows and 300 keys 44 and 43; 32 of 40 rows
// and 2000 keys 54 and 40; 24 of 72 rows and 300 keys 57 and 60, 32 of 72 and 2000 keys 75 and 48.)
constexpr int kOwnRows = 64, kOwnTile = 32, kOwnLead = 1;
inline __host__ __device__ int prefix_tiles(int64_t sequences, int64_t R) {
  return (int)((sequences * R + kPrefixTile - 1) / kPrefixTile);
}
// What a launch takes: its workspace, the slots of prefixes and the work-groups; `units` bounds
// the line.
struct PrefixSizes {
  int64_t bytes, head_bytes, pslots;
  double units;
  int blocks, prows, srows, grid, most_pieces;
};
PrefixSizes prefix_sizes(int64_t B, int64_t G, int64_t Hkv, int64_t R, int64_t D, int64_t keys);
hipError_t launch_prefix_fwd(const PrefixArgs& a, int dtype, hipStream_t stream);

}  // namespace fa
