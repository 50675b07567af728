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

}  // namespace fa
