// fa_rope.hip — RMS norm of each head's queries and keys and their rotation by position, in
// one pass over both tensors, and its backward (gfx950).
//
// A row x of D values (one head of one token), its norm weight w and its token's angles:
//   r = 1 / sqrt(mean(x^2) + eps),  y = x r w        (without norms y = x)
//   z = y rotated: values i and i + R/2 (or 2 i and 2 i + 1) as a pair by angle i, i < R/2;
//   the values from R on stay.
// Backward, g the gradient of z and u = g rotated by the opposite angles:
//   dw = sum over rows of u x r,  t = u w,  dx = r (t - x r mean(t x r)).
//
// Some 20 operations a value: memory bound. So each value is read once and written once in
// 16-byte chunks; a lane holds the two chunks whose values pair up, so that the rotation
// stays in its registers and only the sum over a row crosses lanes (DPP, within the 2, 4 or 8
// lanes of a row); a token's cosines and sines, which take twice the bytes of one row, are
// loaded once and kept while the lane walks over heads, four rows (two in the backward) asked
// for at a time. B2 Hq32 Hkv8 N2048 D128 bf16: forward 17-21 us for 84 MB, backward 25-27 for
// 126 MB, 4.0-5.0 TB/s, a copy's rate on the same cards. Writing the outputs past the caches
// took 2 us off the forward and cost the attention call that reads them 6.
#include <algorithm>

#include "fa_common.hpp"
#include "fa_layer.hpp"

namespace fa {

namespace {

constexpr int kRopeWaves = 4;

// Sum over the LPR (2, 4 or 8) neighbouring lanes of a row.
template <int LPR>
__device__ __forceinline__ float row_sum(float x) {
  auto add = [&](int moved) __attribute__((always_inline)) {
    x += __builtin_bit_cast(float, moved);
  };
  const auto bits = [&]() __attribute__((always_inline)) { return __builtin_bit_cast(int, x); };
  add(__builtin_amdgcn_mov_dpp(bits(), 0xB1, 0xF, 0xF, true));  // quad_perm [1, 0, 3, 2]
  if constexpr (LPR >= 4) add(__builtin_amdgcn_mov_dpp(bits(), 0x4E, 0xF, 0xF, true));  // [2, 3, 0, 1]
  if constexpr (LPR >= 8) add(__builtin_amdgcn_mov_dpp(bits(), 0x141, 0xF, 0xF, true));  // row_half_mirror
  return x;
}

template <class E>
__device__ __forceinline__ void unpack8(u32x4 v, float* f) {
  const half8 h = __builtin_bit_cast(half8, v);
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = elem_to_f32<E>(h[e]);
}
template <class E>
__device__ __forceinline__ u32x4 pack8(const float* f) {
  half8 h;
#pragma unroll
  for (int e = 0; e < 8; ++e) h[e] = to_elem<E>(f[e]);
  return __builtin_bit_cast(u32x4, h);
}

// The two 8-value chunks of a row that lane p of its LPR lanes holds, and its token's angles.
struct RopeLane {
  int c0, c1;        // first value of each chunk
  bool has0, has1;   // it exists
  bool turns, turns1;  // the pair, or with pairs inside a chunk each chunk, is rotated
  int a0, a1;        // first of each four angles
  float cos[8], sin[8];
  float poison;      // 0, or NaN for a token whose position is outside the tables
};

template <int LPR, bool INTER>
__device__ __forceinline__ RopeLane rope_lane(const RopeArgs& a, int p) {
  RopeLane l;
  const int turned = a.R / 16;  // pairs of chunks that are rotated
  int c0, c1;
  if constexpr (INTER) {  // pairs within a chunk: any two chunks
    c0 = p;
    c1 = p + LPR;
  } else if (p >= turned) {
    c0 = 2 * p;
    c1 = c0 + 1;
  } else {
    c0 = p;
    c1 = p + turned;
  }
  l.c0 = 8 * c0;
  l.c1 = 8 * c1;
  l.has0 = l.c0 < a.D;
  l.has1 = l.c1 < a.D;
  l.turns = INTER ? l.c0 < a.R : p < turned;
  l.turns1 = INTER ? l.c1 < a.R : l.turns;
  // the first of the two chunks' angles
  l.a0 = INTER ? 4 * c0 : 8 * p;
  l.a1 = INTER ? 4 * c1 : 8 * p + 4;
  return l;
}

// The angles of token (b, n). A position outside the tables reads nothing and makes the
// token's rows NaN.
__device__ __forceinline__ void rope_angles(const RopeArgs& a, int64_t b, int n, RopeLane& l) {
  int64_t pos = n;
  if (a.pos) {
    const int64_t i = b * a.pos_sb + n * a.pos_sn;
    pos = a.pos64 ? static_cast<const int64_t*>(a.pos)[i]
                  : (int64_t) static_cast<const int*>(a.pos)[i];
  }
  const bool ok = pos >= 0 && pos < a.P;
  l.poison = ok ? 0.f : __builtin_nanf("");
  const int64_t at = ok ? pos * (a.R / 2) : 0;
  float4v c0 = {1.f, 1.f, 1.f, 1.f}, c1 = c0, s0 = {0.f, 0.f, 0.f, 0.f}, s1 = s0;
  if (ok && l.turns) {
    c0 = *reinterpret_cast<const float4v*>(a.cos + at + l.a0);
    s0 = *reinterpret_cast<const float4v*>(a.sin + at + l.a0);
  }
  if (ok && l.turns1) {
    c1 = *reinterpret_cast<const float4v*>(a.cos + at + l.a1);
    s1 = *reinterpret_cast<const float4v*>(a.sin + at + l.a1);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    l.cos[e] = c0[e];
    l.cos[4 + e] = c1[e];
    l.sin[e] = s0[e];
    l.sin[4 + e] = s1[e];
  }
}

// Rotates the pairs in place; DIR = 1 by the angles, -1 by the opposite ones. A lane whose
// pairs are not rotated keeps them as they are (a product with sin = 0 would spread an
// infinity to its partner).
template <bool INTER, int DIR>
__device__ __forceinline__ void rope_turn(const RopeLane& l, float* v0, float* v1) {
  auto turn = [&](float& x, float& y, float c, float s) __attribute__((always_inline)) {
    const float t = DIR * s;
    const float nx = x * c - y * t;
    y = y * c + x * t;
    x = nx;
  };
  if constexpr (!INTER) {
    if (!l.turns) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) turn(v0[e], v1[e], l.cos[e], l.sin[e]);
  } else {
    if (l.turns)
#pragma unroll
      for (int e = 0; e < 4; ++e) turn(v0[2 * e], v0[2 * e + 1], l.cos[e], l.sin[e]);
    if (l.turns1)
#pragma unroll
      for (int e = 0; e < 4; ++e) turn(v1[2 * e], v1[2 * e + 1], l.cos[4 + e], l.sin[4 + e]);
  }
}

// A lane's 16 weights (0 for values that do not exist).
template <class E>
__device__ __forceinline__ void rope_weights(const RopeArgs& a, const void* w, const RopeLane& l,
                                             float* w0, float* w1) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    if (a.w32) {
      const float* f = static_cast<const float*>(w);
      w0[e] = l.has0 ? f[l.c0 + e] : 0.f;
      w1[e] = l.has1 ? f[l.c1 + e] : 0.f;
    } else {
      const half_t* h = static_cast<const half_t*>(w);
      w0[e] = l.has0 ? elem_to_f32<E>(h[l.c0 + e]) : 0.f;
      w1[e] = l.has1 ? elem_to_f32<E>(h[l.c1 + e]) : 0.f;
    }
  }
}

__device__ __forceinline__ u32x4 load_chunk(const half_t* row, int c, bool has) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if (has) v = *reinterpret_cast<const u32x4*>(row + c);
  return v;
}

// The chunk of heads a block of the grid's second axis works on: of the queries first.
struct RopeHeads {
  int side, first, last;
};
__device__ __forceinline__ RopeHeads rope_heads(const RopeArgs& a, int y) {
  RopeHeads h;
  h.side = y >= a.side[0].chunks;
  if (h.side) y -= a.side[0].chunks;
  h.first = y * a.heads;
  h.last = min(a.side[h.side].H, h.first + a.heads);
  return h;
}

}  // namespace

// A row as it comes, two 16-byte chunks a lane.
struct RopeRow {
  u32x4 c0, c1;
};
__device__ __forceinline__ RopeRow load_row(const half_t* row, const RopeLane& l) {
  return {load_chunk(row, l.c0, l.has0), load_chunk(row, l.c1, l.has1)};
}
template <class E>
__device__ __forceinline__ void store_row(half_t* row, const RopeLane& l, const float* v0,
                                          const float* v1) {
  if (l.has0) *reinterpret_cast<u32x4*>(row + l.c0) = pack8<E>(v0);
  if (l.has1) *reinterpret_cast<u32x4*>(row + l.c1) = pack8<E>(v1);
}

// f(h, row[0]) for the heads [first, last), rows asked for U at a time.
template <int U, class Load, class Use>
__device__ __forceinline__ void rope_walk(int first, int last, Load load, Use use) {
  int h = first;
  for (; h + U <= last; h += U) {
    decltype(load(0)) r[U];
#pragma unroll
    for (int u = 0; u < U; ++u) r[u] = load(h + u);
#pragma unroll
    for (int u = 0; u < U; ++u) use(h + u, r[u]);
  }
  for (; h < last; ++h) use(h, load(h));
}

template <int LPR, class E, bool NORM, bool INTER>
__global__ __launch_bounds__(64 * kRopeWaves) void rope_kernel(RopeArgs a) {
  constexpr int TPW = 64 / LPR;  // tokens of a wave
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p = lane % LPR;
  const uint32_t t = a.first + (blockIdx.x * kRopeWaves + wave) * TPW + lane / LPR;
  if (t >= (uint32_t)a.T) return;  // all lanes of a row at once: the sums stay within a row
  const RopeHeads hs = rope_heads(a, blockIdx.y);
  const RopeSide& s = a.side[hs.side];
  const int64_t b = t / (uint32_t)a.N;
  const int n = (int)(t - (uint32_t)b * (uint32_t)a.N);
  RopeLane l = rope_lane<LPR, INTER>(a, p);
  rope_angles(a, b, n, l);
  float w0[8], w1[8];
  if constexpr (NORM) rope_weights<E>(a, s.w, l, w0, w1);
  const half_t* const x = s.x + b * s.xs[0] + n * s.xs[2];
  half_t* const out = s.out + (b * s.H * a.N + n) * a.D;
  rope_walk<4>(
      hs.first, hs.last, [&](int h) __attribute__((always_inline)) { return load_row(x + h * s.xs[1], l); },
      [&](int h, const RopeRow& row) __attribute__((always_inline)) {
        float v0[8], v1[8];
        unpack8<E>(row.c0, v0);
        unpack8<E>(row.c1, v1);
        if constexpr (NORM) {
          float ss = 0.f;
#pragma unroll
          for (int e = 0; e < 8; ++e) ss += v0[e] * v0[e] + v1[e] * v1[e];
          const float r = rsqrtf(row_sum<LPR>(ss) / (float)a.D + a.eps);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            v0[e] *= r * w0[e];
            v1[e] *= r * w1[e];
          }
        }
        rope_turn<INTER, 1>(l, v0, v1);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v0[e] += l.poison;
          v1[e] += l.poison;
        }
        store_row<E>(out + (int64_t)h * a.N * a.D, l, v0, v1);
      });
}

// Backward. A block takes every gridDim.x-th group of tokens, so that the number of
// partial weight gradients stays small however many tokens there are.
template <int LPR, class E, bool NORM, bool INTER>
__global__ __launch_bounds__(64 * kRopeWaves) void rope_bwd_kernel(RopeArgs a) {
  constexpr int TPW = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int p = lane % LPR;
  const RopeHeads hs = rope_heads(a, blockIdx.y);
  const RopeSide& s = a.side[hs.side];
  RopeLane l = rope_lane<LPR, INTER>(a, p);
  float w0[8], w1[8], d0[8], d1[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) d0[e] = d1[e] = 0.f;
  if constexpr (NORM) rope_weights<E>(a, s.w, l, w0, w1);
  const uint32_t step = gridDim.x * kRopeWaves * TPW;
  for (uint32_t t = (blockIdx.x * kRopeWaves + wave) * TPW + lane / LPR; t < (uint32_t)a.T;
       t += step) {
    const int64_t b = t / (uint32_t)a.N;
    const int n = (int)(t - (uint32_t)b * (uint32_t)a.N);
    rope_angles(a, b, n, l);
    const half_t* const g = s.g + b * s.gs[0] + n * s.gs[2];
    const half_t* const x = NORM ? s.x + b * s.xs[0] + n * s.xs[2] : nullptr;
    half_t* const out = s.out + (b * s.H * a.N + n) * a.D;
    struct Rows {
      RopeRow g, x;
    };
    rope_walk<2>(
        hs.first, hs.last,
        [&](int h) __attribute__((always_inline)) {
          Rows r;
          r.g = load_row(g + h * s.gs[1], l);
          if constexpr (NORM) r.x = load_row(x + h * s.xs[1], l);
          return r;
        },
        [&](int h, const Rows& row) __attribute__((always_inline)) {
          float u0[8], u1[8];
          unpack8<E>(row.g.c0, u0);
          unpack8<E>(row.g.c1, u1);
          rope_turn<INTER, -1>(l, u0, u1);
          if constexpr (NORM) {
            float x0[8], x1[8];
            unpack8<E>(row.x.c0, x0);
            unpack8<E>(row.x.c1, x1);
            float ss = 0.f, tx = 0.f;  // sums of x^2 and of t x
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              ss += x0[e] * x0[e] + x1[e] * x1[e];
              tx += u0[e] * w0[e] * x0[e] + u1[e] * w1[e] * x1[e];
            }
            const float inv_d = 1.f / (float)a.D;
            const float r = rsqrtf(row_sum<LPR>(ss) * inv_d + a.eps) + l.poison;
            const float m = row_sum<LPR>(tx) * r * inv_d;  // mean of t x r
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              const float n0 = x0[e] * r, n1 = x1[e] * r;
              d0[e] += u0[e] * n0;
              d1[e] += u1[e] * n1;
              u0[e] = r * (u0[e] * w0[e] - n0 * m);
              u1[e] = r * (u1[e] * w1[e] - n1 * m);
            }
          } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              u0[e] += l.poison;
              u1[e] += l.poison;
            }
          }
          store_row<E>(out + (int64_t)h * a.N * a.D, l, u0, u1);
        });
  }
  if constexpr (NORM) {
    if (s.part == nullptr) return;
    // The block's sum over its tokens and heads, in a fixed order.
    __shared__ float sums[kRopeWaves][LPR][16];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
#pragma unroll
      for (int m = LPR; m < 64; m <<= 1) {
        d0[e] += __shfl_xor(d0[e], m, 64);
        d1[e] += __shfl_xor(d1[e], m, 64);
      }
    }
    if (lane < LPR) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sums[wave][p][e] = d0[e];
        sums[wave][p][8 + e] = d1[e];
      }
    }
    __syncthreads();
    if (wave == 0 && lane < LPR) {
      const int y = blockIdx.y - (hs.side ? a.side[0].chunks : 0);
      float* row = s.part + ((int64_t)y * gridDim.x + blockIdx.x) * a.D;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float v0 = 0.f, v1 = 0.f;
#pragma unroll
        for (int w = 0; w < kRopeWaves; ++w) {
          v0 += sums[w][p][e];
          v1 += sums[w][p][8 + e];
        }
        if (l.has0) row[l.c0 + e] = v0;
        if (l.has1) row[l.c1 + e] = v1;
      }
    }
  }
}

struct RopeReduceArgs {
  const float* part[2];
  void* dw[2];
  int rows[2];
  int D;
  int w32;
};

// dw = the sum of the blocks' partial sums: 16 columns of one tensor a block, 64 threads a
// column that each add every 64th row.
constexpr int kReduceGroups = 64;

template <class E>
__global__ __launch_bounds__(16 * kReduceGroups) void rope_reduce_kernel(RopeReduceArgs a) {
  __shared__ float sums[kReduceGroups][17];
  const int side = blockIdx.y, c = threadIdx.x & 15, g = threadIdx.x >> 4;
  const int col = blockIdx.x * 16 + c;
  if (a.dw[side] == nullptr) return;
  float v = 0.f;
  if (col < a.D) {
#pragma unroll 8
    for (int r = g; r < a.rows[side]; r += kReduceGroups) v += a.part[side][(int64_t)r * a.D + col];
  }
  sums[g][c] = v;
  __syncthreads();
  if (g != 0 || col >= a.D) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < kReduceGroups; ++i) v += sums[i][c];
  if (a.w32) static_cast<float*>(a.dw[side])[col] = v;
  else static_cast<half_t*>(a.dw[side])[col] = to_elem<E>(v);
}

namespace {

int rope_lanes(int D) { return D > 64 ? 8 : D > 32 ? 4 : 2; }
int rope_tokens(int D) { return kRopeWaves * 64 / rope_lanes(D); }  // of a block

// Blocks that fill the chip. With more each loads its tokens' angles for fewer heads (forward
// of the case above: 384 to 512 blocks 17.2 us, 1024 19.3, 2048 21.1; its backward, which walks
// over tokens too, 25.8 with 512 blocks, 28.9 with 2048).
constexpr int64_t kRopeBlocks = 384;
constexpr int64_t kRopeBwdBlocks = 512;

// A launch: `heads` heads of one tensor a chunk, chunks[0] of the queries and chunks[1] of the
// keys along the grid's second axis, `grid` blocks along its first.
struct RopePlan {
  int heads;
  int64_t chunks[2], grid;
  // Rows of partial weight gradients the backward writes.
  int64_t parts() const { return (chunks[0] + chunks[1]) * grid; }
};

RopePlan rope_plan(int64_t T, int D, int Hq, int Hkv, bool bwd) {
  const int64_t tokens = rope_tokens(D);
  const int64_t tiles = (T + tokens - 1) / tokens;
  RopePlan p;
  // As few heads a chunk as fill the chip (about kRopeBlocks blocks).
  p.heads = (int)std::clamp<int64_t>(tiles * (Hq + Hkv) / kRopeBlocks, 1, 16);
  p.chunks[0] = (Hq + p.heads - 1) / p.heads;
  p.chunks[1] = (Hkv + p.heads - 1) / p.heads;
  p.grid = tiles;
  if (bwd) p.grid = std::min(tiles, std::max<int64_t>(1, kRopeBwdBlocks / (p.chunks[0] + p.chunks[1])));
  return p;
}

template <int LPR, class E, bool NORM, bool INTER>
hipError_t rope_start(const RopeArgs& a, const RopePlan& p, bool bwd, hipStream_t stream) {
  const dim3 grid((unsigned)p.grid, (unsigned)(p.chunks[0] + p.chunks[1])), block(64 * kRopeWaves);
  if (bwd) hipLaunchKernelGGL((rope_bwd_kernel<LPR, E, NORM, INTER>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((rope_kernel<LPR, E, NORM, INTER>), grid, block, 0, stream, a);
  return hipGetLastError();
}

template <int LPR, class E>
hipError_t rope_start(const RopeArgs& a, const RopePlan& p, bool bwd, bool norm, bool inter,
                      hipStream_t stream) {
  if (norm) return inter ? rope_start<LPR, E, true, true>(a, p, bwd, stream)
                         : rope_start<LPR, E, true, false>(a, p, bwd, stream);
  return inter ? rope_start<LPR, E, false, true>(a, p, bwd, stream)
               : rope_start<LPR, E, false, false>(a, p, bwd, stream);
}

hipError_t rope_start(RopeArgs a, const RopePlan& p, bool bwd, int dtype, bool norm, bool inter,
                      hipStream_t stream) {
  if (p.grid <= 0 || p.grid > kMostBlocks || p.chunks[0] + p.chunks[1] > 65535)
    return hipErrorInvalidConfiguration;
  a.heads = p.heads;
  for (int i = 0; i < 2; ++i) a.side[i].chunks = (int)p.chunks[i];
  const bool bf = dtype == kBF16;
  switch (rope_lanes(a.D)) {
    case 2: return bf ? rope_start<2, BF16>(a, p, bwd, norm, inter, stream)
                      : rope_start<2, F16>(a, p, bwd, norm, inter, stream);
    case 4: return bf ? rope_start<4, BF16>(a, p, bwd, norm, inter, stream)
                      : rope_start<4, F16>(a, p, bwd, norm, inter, stream);
    default: return bf ? rope_start<8, BF16>(a, p, bwd, norm, inter, stream)
                       : rope_start<8, F16>(a, p, bwd, norm, inter, stream);
  }
}

}  // namespace

int64_t rope_workspace_bytes(int64_t T, int D, int Hq, int Hkv) {
  return rope_plan(T, D, Hq, Hkv, true).parts() * D * 4;
}

hipError_t launch_rope(const RopeArgs& args, int dtype, bool norm, bool interleaved,
                       hipStream_t stream) {
  RopeArgs a = args;
  const RopePlan all = rope_plan(a.T, a.D, a.side[0].H, a.side[1].H, false);
  for (int64_t b = 0; b < all.grid; b += kMostBlocks) {  // past one grid's blocks: another launch
    RopePlan p = all;
    p.grid = std::min(kMostBlocks, all.grid - b);
    a.first = (uint32_t)(b * rope_tokens(a.D));
    const hipError_t e = rope_start(a, p, false, dtype, norm, interleaved, stream);
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

hipError_t launch_rope_bwd(const RopeArgs& args, int dtype, bool norm, bool interleaved,
                           void* const dw[2], float* part, hipStream_t stream) {
  RopeArgs a = args;
  const RopePlan p = rope_plan(a.T, a.D, a.side[0].H, a.side[1].H, true);
  const bool sums = norm && (dw[0] || dw[1]);
  a.side[0].part = norm && dw[0] ? part : nullptr;
  a.side[1].part = norm && dw[1] ? part + p.chunks[0] * p.grid * a.D : nullptr;
  const hipError_t e = rope_start(a, p, true, dtype, norm, interleaved, stream);
  if (e != hipSuccess || !sums) return e;
  RopeReduceArgs r;
  for (int i = 0; i < 2; ++i) {
    r.part[i] = a.side[i].part;
    r.dw[i] = dw[i];
    r.rows[i] = (int)(p.chunks[i] * p.grid);
  }
  r.D = a.D;
  r.w32 = a.w32;
  const dim3 grid((unsigned)((a.D + 15) / 16), 2);
  if (dtype == kBF16) hipLaunchKernelGGL((rope_reduce_kernel<BF16>), grid, dim3(16 * kReduceGroups), 0, stream, r);
  else hipLaunchKernelGGL((rope_reduce_kernel<F16>), grid, dim3(16 * kReduceGroups), 0, stream, r);
  return hipGetLastError();
}

}  // namespace fa
