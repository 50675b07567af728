// fa_capi_layer.hip — extern "C" entry points of the operators around the attention call
// (declared in include/fa_gfx950.h; kernels in fa_rope.hip, fa_paged.hip, fa_prefix.hip and
// fa_pages.hip). As in
// fa_capi.hip every argument is checked before any HIP call.
#include <float.h>
#include <math.h>
#include <string.h>

#include <initializer_list>

#include "../../include/fa_gfx950.h"
#include "fa_layer.hpp"

namespace {

using fa::capi_fail;

const fa::half_t* elems(const fa_half_t* p) { return reinterpret_cast<const fa::half_t*>(p); }
fa::half_t* elems(fa_half_t* p) { return reinterpret_cast<fa::half_t*>(p); }

int check_pointers(const char* name, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (!p) return capi_fail(FA_ERR_NULL_POINTER, "%s: null pointer", name);
  return FA_OK;
}

// Pointers the kernels read or write in pieces of `bytes` (null ones pass).
int check_aligned(const char* name, int bytes, std::initializer_list<const void*> ptrs) {
  for (const void* p : ptrs)
    if (reinterpret_cast<uintptr_t>(p) % bytes)
      return capi_fail(FA_ERR_MISALIGNED, "%s: tensor pointer %p is not %d-byte aligned", name, p,
                       bytes);
  return FA_OK;
}

int check_head_size(const char* name, int64_t D) {
  if (D < 8 || D % 8 || D > 128)
    return capi_fail(FA_ERR_HEAD_DIM,
                     "%s: the head size must be a multiple of 8 up to 128; got %lld", name,
                     (long long)D);
  return FA_OK;
}

// Strides in elements of 16-bit tensors whose rows are read in 16-byte pieces.
int check_strides(const char* name, const char* what, const int64_t* s, int n) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % 8 || s[i] >= (int64_t)1 << 40)
      return capi_fail(FA_ERR_BAD_STRIDE,
                       "%s: the strides of %s must be multiples of 8 elements, not negative and "
                       "below 2^40; got %lld", name, what, (long long)s[i]);
  return FA_OK;
}

// ---- norm and rotation ------------------------------------------------------------------

struct RopeSizes {
  int64_t B, Hq, Hkv, N, D, R, P;
  float eps;
  int flags;
};

int check_rope(const char* name, const RopeSizes& z, const void* q_weight, const void* k_weight) {
  if (z.B <= 0 || z.Hq <= 0 || z.Hkv <= 0 || z.N <= 0 || z.P <= 0)
    return capi_fail(FA_ERR_BAD_SHAPE, "%s: B, Hq, Hkv, N and P must be positive", name);
  if (const int rc = check_head_size(name, z.D)) return rc;
  if (z.R < 16 || z.R % 16 || z.R > z.D)
    return capi_fail(FA_ERR_HEAD_DIM,
                     "%s: the rotated values R must be a multiple of 16 up to the head size "
                     "%lld; got %lld", name, (long long)z.D, (long long)z.R);
  if (z.Hq >= 1 << 15 || z.Hkv >= 1 << 15 || z.B >= (int64_t)1 << 31 || z.N >= (int64_t)1 << 31 ||
      z.B * z.N >= (int64_t)1 << 31 || z.P >= (int64_t)1 << 40)
    return capi_fail(FA_ERR_TOO_LARGE, "%s: too many heads, tokens or positions", name);
  if (!q_weight != !k_weight)
    return capi_fail(FA_ERR_NULL_POINTER, "%s: one of the two norm weights is missing", name);
  if (!isfinite(z.eps) || z.eps < 0.f)
    return capi_fail(FA_ERR_BAD_SCALE, "%s: eps must be finite and not negative (got %g)", name,
                     (double)z.eps);
  if (z.flags & ~(FA_ROPE_INTERLEAVED | FA_ROPE_WEIGHT_F32 | FA_ROPE_POSITIONS_I64))
    return capi_fail(FA_ERR_BAD_SHAPE, "%s: unknown flags %d", name, z.flags);
  return FA_OK;
}

// The positions, the weights and (backward) their gradients, which are read and written value by
// value.
int check_rope_values(const char* name, int flags, const void* positions,
                      const int64_t* position_strides,
                      std::initializer_list<const void*> weights) {
  const int value = flags & FA_ROPE_WEIGHT_F32 ? 4 : 2;
  if (const int rc = check_aligned(name, value, weights)) return rc;
  if (!positions) return FA_OK;
  if (const int rc = check_aligned(name, flags & FA_ROPE_POSITIONS_I64 ? 8 : 4, {positions})) return rc;
  for (int i = 0; i < 2; ++i)
    if (position_strides[i] < 0)
      return capi_fail(FA_ERR_BAD_STRIDE, "%s: a negative stride of the positions: %lld", name,
                       (long long)position_strides[i]);
  return FA_OK;
}

fa::RopeArgs rope_args(const RopeSizes& z, const float* cos, const float* sin,
                       const void* positions, const int64_t* position_strides,
                       const void* q_weight, const void* k_weight) {
  fa::RopeArgs a;
  memset(&a, 0, sizeof(a));
  a.side[0].w = q_weight;
  a.side[1].w = k_weight;
  a.side[0].H = (int)z.Hq;
  a.side[1].H = (int)z.Hkv;
  a.cos = cos;
  a.sin = sin;
  a.pos = positions;
  if (positions) {
    a.pos_sb = position_strides[0];
    a.pos_sn = position_strides[1];
  }
  a.T = z.B * z.N;
  a.P = z.P;
  a.N = (int)z.N;
  a.D = (int)z.D;
  a.R = (int)z.R;
  a.pos64 = (z.flags & FA_ROPE_POSITIONS_I64) != 0;
  a.w32 = (z.flags & FA_ROPE_WEIGHT_F32) != 0;
  a.eps = z.eps;
  return a;
}

int run_rope(const char* name, int dtype, const fa_half_t* q, const fa_half_t* k, fa_half_t* q_out,
             fa_half_t* k_out, const float* cos, const float* sin, const void* positions,
             const void* q_weight, const void* k_weight, const int64_t* strides,
             const RopeSizes& z, void* stream) {
  if (const int rc = check_pointers(name, {q, k, q_out, k_out, cos, sin, strides})) return rc;
  if (const int rc = check_rope(name, z, q_weight, k_weight)) return rc;
  if (const int rc = check_aligned(name, 16, {q, k, q_out, k_out, cos, sin})) return rc;
  if (const int rc = check_strides(name, "the query", strides, 3)) return rc;
  if (const int rc = check_strides(name, "the key", strides + 3, 3)) return rc;
  if (const int rc = check_rope_values(name, z.flags, positions, strides + 6, {q_weight, k_weight}))
    return rc;
  fa::RopeArgs a = rope_args(z, cos, sin, positions, strides + 6, q_weight, k_weight);
  a.side[0].x = elems(q);
  a.side[1].x = elems(k);
  a.side[0].out = elems(q_out);
  a.side[1].out = elems(k_out);
  for (int i = 0; i < 3; ++i) {
    a.side[0].xs[i] = strides[i];
    a.side[1].xs[i] = strides[3 + i];
  }
  return fa::capi_launch_result(
      fa::launch_rope(a, dtype, q_weight != nullptr, (z.flags & FA_ROPE_INTERLEAVED) != 0,
                      static_cast<hipStream_t>(stream)), name);
}

int run_rope_bwd(const char* name, int dtype, const fa_half_t* gq, const fa_half_t* gk,
                 const fa_half_t* q, const fa_half_t* k, fa_half_t* dq, fa_half_t* dk,
                 void* dq_weight, void* dk_weight, const float* cos, const float* sin,
                 const void* positions, const void* q_weight, const void* k_weight,
                 const int64_t* strides, const RopeSizes& z, void* workspace,
                 int64_t workspace_bytes, void* stream) {
  if (const int rc = check_pointers(name, {gq, gk, dq, dk, cos, sin, strides})) return rc;
  if (const int rc = check_rope(name, z, q_weight, k_weight)) return rc;
  const bool norm = q_weight != nullptr;
  if (norm)
    if (const int rc = check_pointers(name, {q, k})) return rc;
  if (const int rc = check_aligned(name, 16, {gq, gk, q, k, dq, dk, cos, sin, workspace})) return rc;
  const char* what[4] = {"the query's gradient", "the key's gradient", "the query", "the key"};
  for (int i = 0; i < (norm ? 4 : 2); ++i)
    if (const int rc = check_strides(name, what[i], strides + 3 * i, 3)) return rc;
  if (const int rc = check_rope_values(name, z.flags, positions, strides + 12,
                                       {q_weight, k_weight, dq_weight, dk_weight}))
    return rc;
  if (norm && (dq_weight || dk_weight)) {
    const int64_t need = fa::rope_workspace_bytes(z.B * z.N, (int)z.D, (int)z.Hq, (int)z.Hkv);
    if (!workspace) return capi_fail(FA_ERR_NULL_POINTER, "%s: null pointer", name);
    if (workspace_bytes < need)
      return capi_fail(FA_ERR_BAD_SHAPE, "%s: workspace of %lld bytes is smaller than the %lld needed",
                       name, (long long)workspace_bytes, (long long)need);
  }
  fa::RopeArgs a = rope_args(z, cos, sin, positions, strides + 12, q_weight, k_weight);
  const fa_half_t *g[2] = {gq, gk}, *x[2] = {q, k};
  fa_half_t* out[2] = {dq, dk};
  for (int s = 0; s < 2; ++s) {
    a.side[s].g = elems(g[s]);
    a.side[s].x = elems(x[s]);
    a.side[s].out = elems(out[s]);
    for (int i = 0; i < 3; ++i) {
      a.side[s].gs[i] = strides[3 * s + i];
      a.side[s].xs[i] = strides[6 + 3 * s + i];
    }
  }
  void* const dw[2] = {dq_weight, dk_weight};
  return fa::capi_launch_result(
      fa::launch_rope_bwd(a, dtype, norm, (z.flags & FA_ROPE_INTERLEAVED) != 0, dw,
                          static_cast<float*>(workspace), static_cast<hipStream_t>(stream)), name);
}

// ---- paged cache ------------------------------------------------------------------------

constexpr int64_t kMaxTokens = ((int64_t)1 << 30) - 64;  // that a row of the page table holds

int check_pages(const char* name, int64_t S, int64_t M) {
  if (S <= 0 || S % 16)
    return capi_fail(FA_ERR_BAD_SHAPE, "%s: the page size must be a positive multiple of 16; got %lld",
                     name, (long long)S);
  if (M <= 0) return capi_fail(FA_ERR_BAD_SHAPE, "%s: the page table needs columns", name);
  if (S > kMaxTokens || M > kMaxTokens || S * M > kMaxTokens)
    return capi_fail(FA_ERR_TOO_LARGE, "%s: %lld pages of %lld tokens a sequence are too many", name,
                     (long long)M, (long long)S);
  return FA_OK;
}

// Strides of a cache [pages, H, S, D]: page, head, row.
int check_cache(const char* name, const int64_t* s, int64_t pages, int64_t D) {
  if (pages <= 0 || pages >= (int64_t)1 << 31)
    return capi_fail(FA_ERR_BAD_SHAPE, "%s: the cache needs between 1 and 2^31 - 1 pages", name);
  if (const int rc = check_strides(name, "the caches", s, 3)) return rc;
  if (s[2] < D || s[2] >= (int64_t)1 << 25)
    return capi_fail(FA_ERR_BAD_STRIDE,
                     "%s: the caches' row stride must be at least the head size %lld and below "
                     "2^25; got %lld", name, (long long)D, (long long)s[2]);
  return FA_OK;
}

int64_t row_blocks(int64_t rows) {
  const int64_t block = fa::paged_rows(rows);
  return (rows + block - 1) / block;
}

int check_attention(const char* name, int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t D,
                    int64_t M, int64_t S) {
  if (B <= 0 || Hq <= 0 || Hkv <= 0 || N <= 0 || Hq % Hkv)
    return capi_fail(FA_ERR_BAD_SHAPE,
                     "%s: B, Hq, Hkv and N must be positive and Hq divisible by Hkv (got %lld, "
                     "%lld, %lld, %lld)", name, (long long)B, (long long)Hq, (long long)Hkv,
                     (long long)N);
  if (const int rc = check_head_size(name, D)) return rc;
  if (const int rc = check_pages(name, S, M)) return rc;
  const int64_t most = (int64_t)1 << 30;
  if (B >= most || Hq >= 1 << 20 || N >= 1 << 20)
    return capi_fail(FA_ERR_TOO_LARGE, "%s: too many sequences, heads or queries", name);
  return FA_OK;
}

int check_paged(const char* name, int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t D,
                int64_t M, int64_t S) {
  if (const int rc = check_attention(name, B, Hq, Hkv, N, D, M, S)) return rc;
  const int64_t most = (int64_t)1 << 30;
  // Units of all sequences, heads and row blocks are counted in 32 bits, up to 24 more for each.
  const double units = (double)B * Hkv * row_blocks(Hq / Hkv * N) *
                       ((M * S + fa::kPagedUnit - 1) / fa::kPagedUnit + 24);
  if (units >= (double)most)
    return capi_fail(FA_ERR_TOO_LARGE,
                     "%s: %lld sequences of up to %lld keys are too many for one call", name,
                     (long long)B, (long long)(M * S));
  return FA_OK;
}

int check_scale(const char* name, float scale) {
  const float c = scale * fa::kLog2e;
  if (!isfinite(scale) || !isfinite(c) || !(c >= FLT_MIN))
    return capi_fail(FA_ERR_BAD_SCALE,
                     "%s: scale must be finite and > 0 with scale * log2(e) a normal float32 (got "
                     "%g)", name, (double)scale);
  return FA_OK;
}

// For each work-group 16 bytes, and two partials: a row block of O and its log-sum-exps.
int64_t paged_workspace(int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t D, int64_t M,
                        int64_t S) {
  const int64_t width = D <= 32 ? 32 : D <= 64 ? 64 : 128;
  const int64_t rows = Hq / Hkv * N;
  const int grid = fa::paged_grid(B, Hkv, row_blocks(rows), M * S);
  return grid == 0 ? 0 : (int64_t)grid * (16 + 2 * fa::paged_rows(rows) * (width + 1) * 4);
}

int run_paged(const char* name, int dtype, const fa_half_t* q, const fa_half_t* k_cache,
              const fa_half_t* v_cache, const int32_t* page_table, const int32_t* lengths,
              fa_half_t* o, const int64_t* strides, int64_t B, int64_t Hq, int64_t Hkv, int64_t N,
              int64_t D, int64_t pages, int64_t M, int64_t S, float scale, void* workspace,
              int64_t workspace_bytes, void* stream) {
  if (const int rc = check_pointers(name, {q, k_cache, v_cache, page_table, lengths, o, strides}))
    return rc;
  if (const int rc = check_paged(name, B, Hq, Hkv, N, D, M, S)) return rc;
  if (const int rc = check_aligned(name, 16, {q, k_cache, v_cache, o, workspace})) return rc;
  if (const int rc = check_aligned(name, 4, {page_table, lengths})) return rc;
  if (const int rc = check_strides(name, "the query", strides, 3)) return rc;
  if (const int rc = check_cache(name, strides + 3, pages, D)) return rc;
  if (strides[6] < 0) return capi_fail(FA_ERR_BAD_STRIDE, "%s: a negative page table stride", name);
  const float c = scale * fa::kLog2e;
  if (const int rc = check_scale(name, scale)) return rc;
  const int64_t need = paged_workspace(B, Hq, Hkv, N, D, M, S);
  if (need > 0 && !workspace) return capi_fail(FA_ERR_NULL_POINTER, "%s: null pointer", name);
  if (workspace_bytes < need)
    return capi_fail(FA_ERR_BAD_SHAPE, "%s: workspace of %lld bytes is smaller than the %lld needed",
                     name, (long long)workspace_bytes, (long long)need);
  fa::PagedArgs a;
  a.q = elems(q);
  a.k = elems(k_cache);
  a.v = elems(v_cache);
  a.table = page_table;
  a.lengths = lengths;
  a.o = elems(o);
  a.part = static_cast<float*>(workspace);
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = strides[i];
    a.ks[i] = strides[3 + i];
  }
  a.table_stride = strides[6];
  a.pages = pages;
  a.c = c;
  a.B = (int)B;
  a.Hkv = (int)Hkv;
  a.group = (int)(Hq / Hkv);
  a.N = (int)N;
  a.d = (int)D;
  a.M = (int)M;
  a.S = (int)S;
  a.rows = fa::paged_rows(Hq / Hkv * N);
  a.blocks = (int)row_blocks(Hq / Hkv * N);
  a.grid = fa::paged_grid(B, Hkv, a.blocks, M * S);
  return fa::capi_launch_result(
      fa::launch_paged_fwd(a, D <= 32 ? 32 : D <= 64 ? 64 : 128, dtype,
                           static_cast<hipStream_t>(stream)), name);
}

int check_workspace(const char* name, int64_t bytes, int64_t need) {
  if (bytes < need)
    return capi_fail(FA_ERR_BAD_SHAPE, "%s: workspace of %lld bytes is smaller than the %lld needed",
                     name, (long long)bytes, (long long)need);
  return FA_OK;
}

// A page table, a list of pages and the cache's pages, as the calls on pages number them.
int check_rows(const char* name, int64_t B, int64_t M, int64_t F, int64_t pages) {
  if (B < 0 || F < 0 || M <= 0 || pages <= 0)
    return capi_fail(FA_ERR_BAD_SHAPE,
                     "%s: M and pages must be positive, B and F must not be negative", name);
  const int64_t most = (int64_t)1 << 30;
  // (a launch has up to 16 blocks of 1024 threads for a row)
  if (B >= 1 << 17 || M >= most || F >= most || pages >= most || B * M >= (int64_t)1 << 40)
    return capi_fail(FA_ERR_TOO_LARGE, "%s: too many sequences or pages", name);
  return FA_OK;
}

int check_prefix(const char* name, int64_t B, int64_t G, int64_t Hq, int64_t Hkv, int64_t N,
                 int64_t D, int64_t M, int64_t S) {
  if (const int rc = check_attention(name, B, Hq, Hkv, N, D, M, S)) return rc;
  if (G < 0) return capi_fail(FA_ERR_BAD_SHAPE, "%s: G must not be negative", name);
  const int64_t R = Hq / Hkv * N;
  // Rows that read a head and units of the line are counted in 32 bits; two rows or more of the
  // output are a block of the join, whose grid's threads are too. Every work-group looks through all
  // groups, which takes 20 ms for 2^20 of them, however empty.
  if (G >= (int64_t)1 << 24 || R >= (int64_t)1 << 25 || B * Hkv * R > 2 * fa::kMostBlocks ||
      fa::prefix_sizes(B, G, Hkv, R, D, M * S).units >= (double)((int64_t)1 << 30))
    return capi_fail(FA_ERR_TOO_LARGE,
                     "%s: %lld sequences of up to %lld keys in %lld groups are too many for one call",
                     name, (long long)B, (long long)(M * S), (long long)G);
  return FA_OK;
}

int run_prefix(const char* name, int dtype, const fa_half_t* q, const fa_half_t* k_cache,
               const fa_half_t* v_cache, const int32_t* page_table, const int32_t* lengths,
               const int32_t* group_starts, const int32_t* prefix_lengths, fa_half_t* o,
               const int64_t* strides, int64_t B, int64_t G, int64_t Hq, int64_t Hkv, int64_t N,
               int64_t D, int64_t pages, int64_t M, int64_t S, float scale, void* workspace,
               int64_t workspace_bytes, void* stream) {
  if (const int rc = check_pointers(name, {q, k_cache, v_cache, page_table, lengths, group_starts, o,
                                           strides, workspace}))
    return rc;
  if (const int rc = check_prefix(name, B, G, Hq, Hkv, N, D, M, S)) return rc;
  if (G > 0)
    if (const int rc = check_pointers(name, {prefix_lengths})) return rc;
  if (const int rc = check_aligned(name, 16, {q, k_cache, v_cache, o, workspace})) return rc;
  if (const int rc = check_aligned(name, 4, {page_table, lengths, group_starts, prefix_lengths}))
    return rc;
  if (const int rc = check_strides(name, "the query", strides, 3)) return rc;
  if (const int rc = check_cache(name, strides + 3, pages, D)) return rc;
  if (strides[6] < 0) return capi_fail(FA_ERR_BAD_STRIDE, "%s: a negative page table stride", name);
  const float c = scale * fa::kLog2e;
  if (const int rc = check_scale(name, scale)) return rc;
  const int64_t R = Hq / Hkv * N;
  const fa::PrefixSizes z = fa::prefix_sizes(B, G, Hkv, R, D, M * S);
  if (const int rc = check_workspace(name, workspace_bytes, z.bytes)) return rc;
  fa::PrefixArgs a;
  a.q = elems(q);
  a.k = elems(k_cache);
  a.v = elems(v_cache);
  a.table = page_table;
  a.lengths = lengths;
  a.starts = group_starts;
  a.prefix = prefix_lengths;
  a.o = elems(o);
  a.ws = static_cast<int*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<char*>(workspace) + z.head_bytes);
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = strides[i];
    a.ks[i] = strides[3 + i];
  }
  a.table_stride = strides[6];
  a.pages = pages;
  a.pslots = z.pslots;
  a.c = c;
  a.B = (int)B;
  a.G = (int)G;
  a.Hkv = (int)Hkv;
  a.group = (int)(Hq / Hkv);
  a.N = (int)N;
  a.d = (int)D;
  a.M = (int)M;
  a.S = (int)S;
  a.R = (int)R;
  a.blocks = z.blocks;
  a.prows = z.prows;
  a.srows = z.srows;
  a.grid = z.grid;
  a.most_pieces = z.most_pieces;
  return fa::capi_launch_result(fa::launch_prefix_fwd(a, dtype, static_cast<hipStream_t>(stream)),
                                name);
}

}  // namespace

extern "C" {

#define FA_ROPE_PARAMS                                                                          \
  const fa_half_t *q, const fa_half_t *k, fa_half_t *q_out, fa_half_t *k_out, const float *cos, \
      const float *sin, const void *positions, const void *q_weight, const void *k_weight,      \
      const int64_t *strides, int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t D,         \
      int64_t R, int64_t P, float eps, int flags, void *stream
int fa_qk_norm_rope(FA_ROPE_PARAMS) {
  return run_rope("fa_qk_norm_rope", fa::kF16, q, k, q_out, k_out, cos, sin, positions, q_weight,
                  k_weight, strides, {B, Hq, Hkv, N, D, R, P, eps, flags}, stream);
}
int fa_qk_norm_rope_bf16(FA_ROPE_PARAMS) {
  return run_rope("fa_qk_norm_rope_bf16", fa::kBF16, q, k, q_out, k_out, cos, sin, positions,
                  q_weight, k_weight, strides, {B, Hq, Hkv, N, D, R, P, eps, flags}, stream);
}

int64_t fa_qk_norm_rope_bwd_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t N,
                                            int64_t D) {
  const char* name = "fa_qk_norm_rope_bwd_workspace_bytes";
  if (const int rc = check_head_size(name, D)) return rc;
  if (const int rc = check_rope(name, {B, Hq, Hkv, N, D < 16 ? 16 : D, 16, 1, 0.f, 0}, nullptr,
                                nullptr))
    return rc;
  return fa::rope_workspace_bytes(B * N, (int)D, (int)Hq, (int)Hkv);
}

#define FA_ROPE_BWD_PARAMS                                                                        \
  const fa_half_t *gq, const fa_half_t *gk, const fa_half_t *q, const fa_half_t *k, fa_half_t *dq, \
      fa_half_t *dk, void *dq_weight, void *dk_weight, const float *cos, const float *sin,         \
      const void *positions, const void *q_weight, const void *k_weight, const int64_t *strides,   \
      int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t D, int64_t R, int64_t P, float eps,   \
      int flags, void *workspace, int64_t workspace_bytes, void *stream
int fa_qk_norm_rope_bwd(FA_ROPE_BWD_PARAMS) {
  return run_rope_bwd("fa_qk_norm_rope_bwd", fa::kF16, gq, gk, q, k, dq, dk, dq_weight, dk_weight,
                      cos, sin, positions, q_weight, k_weight, strides,
                      {B, Hq, Hkv, N, D, R, P, eps, flags}, workspace, workspace_bytes, stream);
}
int fa_qk_norm_rope_bwd_bf16(FA_ROPE_BWD_PARAMS) {
  return run_rope_bwd("fa_qk_norm_rope_bwd_bf16", fa::kBF16, gq, gk, q, k, dq, dk, dq_weight,
                      dk_weight, cos, sin, positions, q_weight, k_weight, strides,
                      {B, Hq, Hkv, N, D, R, P, eps, flags}, workspace, workspace_bytes, stream);
}

int fa_paged_plan(int32_t* page_table, int64_t table_stride, const int32_t* lengths,
                  const int32_t* new_tokens, const int32_t* free_pages, const int32_t* free_start,
                  int64_t* slots, int32_t* positions, int32_t* starts, int32_t* lengths_out,
                  int32_t* free_start_out, int64_t B, int64_t M, int64_t S, int64_t F, int64_t T,
                  void* stream) {
  const char* name = "fa_paged_plan";
  if (const int rc = check_pages(name, S, M)) return rc;
  if (B < 0 || F < 0 || T < 0)
    return capi_fail(FA_ERR_BAD_SHAPE, "%s: B, F and T must not be negative", name);
  if (B >= (int64_t)1 << 30 || F >= (int64_t)1 << 31 || T >= (int64_t)1 << 30)
    return capi_fail(FA_ERR_TOO_LARGE, "%s: too many sequences, free pages or tokens", name);
  if (const int rc = check_pointers(name, {starts, free_start_out})) return rc;
  if (B > 0)
    if (const int rc = check_pointers(name, {page_table, lengths, new_tokens, lengths_out}))
      return rc;
  if (F > 0)
    if (const int rc = check_pointers(name, {free_pages})) return rc;
  if (T > 0)
    if (const int rc = check_pointers(name, {slots, positions})) return rc;
  if (const int rc = check_aligned(name, 4, {page_table, lengths, new_tokens, free_pages, free_start,
                                             positions, starts, lengths_out, free_start_out}))
    return rc;
  if (const int rc = check_aligned(name, 8, {slots})) return rc;
  if (table_stride < 0 || (B > 1 && table_stride < M))
    return capi_fail(FA_ERR_BAD_STRIDE, "%s: rows of the page table must not overlap", name);
  fa::PlanArgs a;
  a.table = page_table;
  a.lengths = lengths;
  a.new_tokens = new_tokens;
  a.free_pages = free_pages;
  a.free_start = free_start;
  a.slots = slots;
  a.positions = positions;
  a.starts = starts;
  a.lengths_out = lengths_out;
  a.free_out = free_start_out;
  a.table_stride = table_stride;
  a.T = T;
  a.B = (int)B;
  a.M = (int)M;
  a.F = (int)F;
  a.S = (int)S;
  return fa::capi_launch_result(fa::launch_paged_plan(a, static_cast<hipStream_t>(stream)), name);
}

int fa_paged_store(const fa_half_t* key, const fa_half_t* value, fa_half_t* k_cache,
                   fa_half_t* v_cache, const int64_t* slots, const int64_t* strides, int64_t T,
                   int64_t H, int64_t D, int64_t pages, int64_t S, void* stream) {
  const char* name = "fa_paged_store";
  if (T == 0) return FA_OK;
  if (const int rc = check_pointers(name, {key, value, k_cache, v_cache, slots, strides})) return rc;
  if (T < 0 || H <= 0) return capi_fail(FA_ERR_BAD_SHAPE, "%s: T and H must be positive", name);
  if (T >= (int64_t)1 << 31 || H >= 1 << 20)
    return capi_fail(FA_ERR_TOO_LARGE, "%s: too many tokens or heads", name);
  if (const int rc = check_head_size(name, D)) return rc;
  if (const int rc = check_pages(name, S, 1)) return rc;
  if (const int rc = check_aligned(name, 16, {key, value, k_cache, v_cache})) return rc;
  if (const int rc = check_aligned(name, 8, {slots})) return rc;
  if (const int rc = check_strides(name, "the keys", strides, 2)) return rc;
  if (const int rc = check_strides(name, "the values", strides + 2, 2)) return rc;
  if (const int rc = check_cache(name, strides + 4, pages, D)) return rc;
  fa::StoreArgs a;
  a.src[0] = elems(key);
  a.src[1] = elems(value);
  a.dst[0] = elems(k_cache);
  a.dst[1] = elems(v_cache);
  a.slots = slots;
  for (int i = 0; i < 2; ++i) {
    a.ss[0][i] = strides[i];
    a.ss[1][i] = strides[2 + i];
  }
  for (int i = 0; i < 3; ++i) a.ds[i] = strides[4 + i];
  a.T = T;
  a.pages = pages;
  a.H = (int)H;
  a.S = (int)S;
  a.chunks = (int)(D / 8);
  return fa::capi_launch_result(fa::launch_paged_store(a, static_cast<hipStream_t>(stream)), name);
}

int64_t fa_paged_fwd_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t D,
                                     int64_t M, int64_t S) {
  if (const int rc = check_paged("fa_paged_fwd_workspace_bytes", B, Hq, Hkv, N, D, M, S)) return rc;
  return paged_workspace(B, Hq, Hkv, N, D, M, S);
}

#define FA_PAGED_PARAMS                                                                       \
  const fa_half_t *q, const fa_half_t *k_cache, const fa_half_t *v_cache,                     \
      const int32_t *page_table, const int32_t *lengths, fa_half_t *o, const int64_t *strides, \
      int64_t B, int64_t Hq, int64_t Hkv, int64_t N, int64_t D, int64_t pages, int64_t M,      \
      int64_t S, float scale, void *workspace, int64_t workspace_bytes, void *stream
int fa_paged_fwd(FA_PAGED_PARAMS) {
  return run_paged("fa_paged_fwd", fa::kF16, q, k_cache, v_cache, page_table, lengths, o, strides,
                   B, Hq, Hkv, N, D, pages, M, S, scale, workspace, workspace_bytes, stream);
}
int fa_paged_fwd_bf16(FA_PAGED_PARAMS) {
  return run_paged("fa_paged_fwd_bf16", fa::kBF16, q, k_cache, v_cache, page_table, lengths, o,
                   strides, B, Hq, Hkv, N, D, pages, M, S, scale, workspace, workspace_bytes,
                   stream);
}

int64_t fa_paged_fork_workspace_bytes(int64_t B, int64_t M, int64_t pages) {
  if (const int rc = check_rows("fa_paged_fork_workspace_bytes", B, M, 0, pages)) return rc;
  return fa::fork_workspace_bytes(B, M, pages);
}

int fa_paged_fork(int32_t* page_table, int64_t table_stride, const int32_t* lengths,
                  const int32_t* parents, int32_t* free_pages, const int32_t* free_start,
                  int32_t* page_shares, int32_t* lengths_out, int32_t* sources, int32_t* targets,
                  int32_t* tokens, int32_t* free_start_out, int64_t B, int64_t M, int64_t S,
                  int64_t F, int64_t pages, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "fa_paged_fork";
  if (const int rc = check_pages(name, S, M)) return rc;
  if (const int rc = check_rows(name, B, M, F, pages)) return rc;
  if (const int rc = check_pointers(name, {page_shares, free_start_out, workspace})) return rc;
  if (B > 0)
    if (const int rc = check_pointers(name, {page_table, lengths, parents, lengths_out, sources,
                                             targets, tokens}))
      return rc;
  if (F > 0)
    if (const int rc = check_pointers(name, {free_pages})) return rc;
  if (const int rc = check_aligned(name, 4, {page_table, lengths, parents, free_pages, free_start,
                                             page_shares, lengths_out, sources, targets, tokens,
                                             free_start_out, workspace}))
    return rc;
  if (table_stride < 0 || (B > 1 && table_stride < M))
    return capi_fail(FA_ERR_BAD_STRIDE, "%s: rows of the page table must not overlap", name);
  if (const int rc = check_workspace(name, workspace_bytes, fa::fork_workspace_bytes(B, M, pages)))
    return rc;
  fa::ForkArgs a;
  memset(&a, 0, sizeof(a));
  a.table = page_table;
  a.lengths = lengths;
  a.parents = parents;
  a.free_pages = free_pages;
  a.free_start = free_start;
  a.shares = page_shares;
  a.lengths_out = lengths_out;
  a.sources = sources;
  a.targets = targets;
  a.tokens = tokens;
  a.free_out = free_start_out;
  a.table_stride = table_stride;
  a.B = (int)B;
  a.M = (int)M;
  a.F = (int)F;
  a.S = (int)S;
  a.pages = (int)pages;
  return fa::capi_launch_result(fa::launch_fork(a, workspace, static_cast<hipStream_t>(stream)), name);
}

int fa_paged_copy(fa_half_t* k_cache, fa_half_t* v_cache, const int32_t* sources,
                  const int32_t* targets, const int32_t* tokens, const int64_t* strides, int64_t n,
                  int64_t H, int64_t D, int64_t pages, int64_t S, void* stream) {
  const char* name = "fa_paged_copy";
  if (n == 0) return FA_OK;
  if (const int rc = check_pointers(name, {k_cache, v_cache, sources, targets, strides})) return rc;
  if (n < 0 || H <= 0) return capi_fail(FA_ERR_BAD_SHAPE, "%s: n and H must be positive", name);
  if (n >= (int64_t)1 << 31 || H >= 1 << 20)
    return capi_fail(FA_ERR_TOO_LARGE, "%s: too many pages or heads", name);
  if (const int rc = check_head_size(name, D)) return rc;
  if (const int rc = check_pages(name, S, 1)) return rc;
  if (H * S * (D / 8) >= (int64_t)1 << 30)
    return capi_fail(FA_ERR_TOO_LARGE, "%s: pages of %lld tokens and %lld heads are too large", name,
                     (long long)S, (long long)H);
  if (const int rc = check_aligned(name, 16, {k_cache, v_cache})) return rc;
  if (const int rc = check_aligned(name, 4, {sources, targets, tokens})) return rc;
  if (const int rc = check_cache(name, strides, pages, D)) return rc;
  fa::CopyArgs a;
  memset(&a, 0, sizeof(a));
  a.k = elems(k_cache);
  a.v = elems(v_cache);
  a.sources = sources;
  a.targets = targets;
  a.tokens = tokens;
  for (int i = 0; i < 3; ++i) a.ks[i] = strides[i];
  a.n = n;
  a.pages = pages;
  a.H = (int)H;
  a.S = (int)S;
  a.chunks = (int)(D / 8);
  return fa::capi_launch_result(fa::launch_page_copy(a, static_cast<hipStream_t>(stream)), name);
}

int64_t fa_paged_compact_workspace_bytes(int64_t pages) {
  if (const int rc = check_rows("fa_paged_compact_workspace_bytes", 0, 1, 0, pages)) return rc;
  return fa::compact_workspace_bytes(pages);
}

int fa_paged_compact(const int32_t* page_table, int64_t table_stride, const int32_t* free_pages,
                     const int32_t* free_start, const int32_t* page_shares, int32_t* table_out,
                     int32_t* free_pages_out, int32_t* shares_out, int32_t* sources,
                     int32_t* targets, int32_t* used_out, int64_t B, int64_t M, int64_t F,
                     int64_t pages, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* name = "fa_paged_compact";
  if (const int rc = check_rows(name, B, M, F, pages)) return rc;
  if (const int rc = check_pointers(name, {page_shares, shares_out, used_out, workspace})) return rc;
  if (B > 0)
    if (const int rc = check_pointers(name, {page_table, table_out})) return rc;
  if (F > 0)
    if (const int rc = check_pointers(name, {free_pages, free_pages_out, sources, targets})) return rc;
  if (const int rc = check_aligned(name, 4, {page_table, free_pages, free_start, page_shares,
                                             table_out, free_pages_out, shares_out, sources, targets,
                                             used_out}))
    return rc;
  if (const int rc = check_aligned(name, 16, {workspace})) return rc;
  if (table_stride < 0)
    return capi_fail(FA_ERR_BAD_STRIDE, "%s: a negative page table stride", name);
  if (const int rc = check_workspace(name, workspace_bytes, fa::compact_workspace_bytes(pages)))
    return rc;
  fa::CompactArgs a;
  memset(&a, 0, sizeof(a));
  a.table = page_table;
  a.free_pages = free_pages;
  a.free_start = free_start;
  a.shares = page_shares;
  a.table_out = table_out;
  a.free_pages_out = free_pages_out;
  a.shares_out = shares_out;
  a.sources = sources;
  a.targets = targets;
  a.used = used_out;
  a.table_stride = table_stride;
  a.B = (int)B;
  a.M = (int)M;
  a.F = (int)F;
  a.pages = (int)pages;
  return fa::capi_launch_result(fa::launch_compact(a, workspace, static_cast<hipStream_t>(stream)),
                                name);
}

int64_t fa_paged_prefix_fwd_workspace_bytes(int64_t B, int64_t G, int64_t Hq, int64_t Hkv, int64_t N,
                                            int64_t D, int64_t M, int64_t S) {
  if (const int rc = check_prefix("fa_paged_prefix_fwd_workspace_bytes", B, G, Hq, Hkv, N, D, M, S))
    return rc;
  return fa::prefix_sizes(B, G, Hkv, Hq / Hkv * N, D, M * S).bytes;
}

#define FA_PREFIX_PARAMS                                                                           \
  const fa_half_t *q, const fa_half_t *k_cache, const fa_half_t *v_cache,                          \
      const int32_t *page_table, const int32_t *lengths, const int32_t *group_starts,              \
      const int32_t *prefix_lengths, fa_half_t *o, const int64_t *strides, int64_t B, int64_t G,    \
      int64_t Hq, int64_t Hkv, int64_t N, int64_t D, int64_t pages, int64_t M, int64_t S,           \
      float scale, void *workspace, int64_t workspace_bytes, void *stream
int fa_paged_prefix_fwd(FA_PREFIX_PARAMS) {
  return run_prefix("fa_paged_prefix_fwd", fa::kF16, q, k_cache, v_cache, page_table, lengths,
                    group_starts, prefix_lengths, o, strides, B, G, Hq, Hkv, N, D, pages, M, S,
                    scale, workspace, workspace_bytes, stream);
}
int fa_paged_prefix_fwd_bf16(FA_PREFIX_PARAMS) {
  return run_prefix("fa_paged_prefix_fwd_bf16", fa::kBF16, q, k_cache, v_cache, page_table, lengths,
                    group_starts, prefix_lengths, o, strides, B, G, Hq, Hkv, N, D, pages, M, S,
                    scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
