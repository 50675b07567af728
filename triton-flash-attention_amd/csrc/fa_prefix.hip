// fa_prefix.hip — attention of the newest tokens over the paged cache where groups of sequences
// share a prefix (gfx950): prefix_fwd_kernel works on the prefixes, each once for all rows of its
// group, and on what follows them; prefix_join_kernel joins the two for every row.
//
//   o = softmax(scale q K^T) V, query n of a sequence of len keys seeing keys j <= len - N + n
//
// Group g holds the sequences starts[g] .. starts[g + 1] - 1. Its prefix is the first P keys of
// its first sequence, P = prefix_lengths[g] or that sequence's length where this is less (no keys
// in a group of one, whose sequence reads them as its own): keys j < P of all its sequences lie in
// the pages of the first one, keys j >= P in each one's own.
#include <algorithm>
#include <type_traits>

#include "fa_common.hpp"
#include "fa_layer.hpp"

namespace fa {

// The work is a list of triples: (group, key/value head, tile of 128 query rows) over the keys of
// the group's prefix, then (sequence, key/value head, tile) over a sequence's own keys. A tile's
// rows are those that read the key/value head: the group's heads and the N tokens of one sequence
// after the other. Units of 32 keys of all triples lie on one line, each triple's behind `lead`
// empty ones that stand for opening and closing a piece; every work-group takes an equal stretch of
// it, found from the lengths on the GPU. It writes what it has of a triple as one piece, normalised
// partial O and base-2 log-sum-exp of each row, into a slot of its own: stretch s + triple t, which
// no two pieces share since from one piece to the next on the line either s or t grows by one.
constexpr int kPrefixWaves = 4;
constexpr int kPrefixStarts = 2048;       // of the groups' starts that are kept in LDS

template <int D>
struct PrefixRing {
  static constexpr int KT = 32;             // keys of a unit
  static constexpr int TILE = KT * D;       // halves of its K (or V) rows
  static constexpr int STAGE = 2 * TILE;
  static constexpr int NS = D == 128 ? 5 : 6;
  static constexpr int WGS = D == 128 ? 2 : 3;  // work-groups a CU
  static constexpr int AHEAD = NS - 2;          // units asked for before the first step
  static constexpr int IN_FLIGHT = AHEAD - 2;   // of them not awaited at a barrier
  static constexpr int INSTR = TILE * 2 / 1024;
  static constexpr int PER_WAVE = INSTR >= kPrefixWaves ? INSTR / kPrefixWaves : 1;
  static constexpr int HALVES = NS * STAGE;
  static_assert(WGS * HALVES * 2 <= 160 * 1024, "LDS of a CU");
};

// As in fa_paged.hip: the reference of a row's probabilities is 2^7 below the max for fp16 and 2^16
// above it, or above the sum, for bf16, whose probabilities so far are held to 1/4 a lane, 1/2 a row.
template <class E>
constexpr bool kPrefixWide = std::is_same_v<E, BF16>;
template <class E>
constexpr float kPrefixShift = kPrefixWide<E> ? -16.f : 7.f;
template <class E>
constexpr float kPrefixSumLimit = kPrefixWide<E> ? 0.25f : 32768.f;

namespace {

// ---- the line ---------------------------------------------------------------------------

__device__ __forceinline__ int fitting(const PrefixArgs& a, int len) {
  return len > 0 && len <= a.M * a.S ? len : 0;
}
// Prefix keys of a group that begins at sequence b and ends before e.
__device__ __forceinline__ int prefix_keys(const PrefixArgs& a, int g, int b, int e) {
  return e - b < 2 ? 0 : min(max(a.prefix[g], 0), fitting(a, a.lengths[b]));
}
// Units that n keys from `first` on take: a unit's halves of 16 keys lie in one page each.
__device__ __forceinline__ int key_units(int first, int end) {
  return end > first ? (end - (first & ~15) + 31) / 32 : 0;
}
__device__ __forceinline__ int on_line(int units) { return units > 0 ? units + kPrefixLead : 0; }

// Where the search for sequence b among the groups ends: the last g with starts[g] <= b, or -1.
__device__ __forceinline__ int group_of(const int* starts, int G, int b) {
  int g = -1;
  for (int step = 1 << (31 - __builtin_clz(G + 1)); step > 0; step >>= 1)
    if (g + step <= G && starts[g + step] <= b) g += step;
  return g;
}

// A place on the line: unit `unit` (lead included) of triple `sub` (head-major) of group `at` or,
// behind the prefixes, of sequence `at`; `first` is the index of that group's first triple.
struct PrefixPlace {
  int own;  // 0: a prefix, 1: a sequence's own keys
  int at, sub, unit, first;
};
struct PrefixLine {
  int total, stretch;
  bool bad;  // the groups' starts do not ascend within [0, B]
};

// What the kernels know of sequence b's rows: written by work-group 0 for the join.
__device__ __forceinline__ PrefixSeq* prefix_seqs(const PrefixArgs& a) {
  return reinterpret_cast<PrefixSeq*>(a.ws + 16);
}

// The line, and its place at stretch `s`, defined where the line reaches it. `lds`: the
// work-group's memory, free before and after.
__device__ __forceinline__ PrefixLine prefix_find(const PrefixArgs& a, int s, int* lds,
                                                  PrefixPlace* place) {
  constexpr int W = kPrefixWaves, T = 64 * W;
  int* const found = lds;                                  // [8]
  int(*const sums)[3] = reinterpret_cast<int(*)[3]>(lds + 8);  // [W]
  int* const kept = lds + 32;                              // the starts
  const int tid = threadIdx.x;
  bool wrong = false;
  for (int g = tid; g <= a.G; g += T) {
    const int x = a.starts[g];
    wrong |= x < 0 || x > a.B || (g > 0 && a.starts[g - 1] > x);
    if (g < kPrefixStarts) kept[g] = x;
  }
  // (the flags of the waves, beside found[]: __syncthreads_or would take LDS of its own)
  if ((tid & 63) == 0) lds[24 + (tid >> 6)] = 0;
  if (wrong) lds[24 + (tid >> 6)] = 1;
  __syncthreads();
  PrefixLine line;
  line.bad = (lds[24] | lds[25] | lds[26] | lds[27]) != 0;
  const int G = line.bad ? 0 : a.G;
  const int* const starts = a.G < kPrefixStarts ? kept : a.starts;

  // The thread's groups and sequences: their parts of the line, and the groups' triples.
  const int per_g = (G + T - 1) / T, g0 = tid * per_g, g1 = min(G, g0 + per_g);
  const int per_b = (a.B + T - 1) / T, b0 = tid * per_b, b1 = min(a.B, b0 + per_b);
  auto group_triples = [&](int g) __attribute__((always_inline)) {
    return prefix_tiles(starts[g + 1] - starts[g], a.R) * a.Hkv;
  };
  auto group_units = [&](int g) __attribute__((always_inline)) {
    return key_units(0, prefix_keys(a, g, starts[g], starts[g + 1]));
  };
  auto group_at = [&](int b) __attribute__((always_inline)) {
    const int g = G > 0 ? group_of(starts, G, b) : -1;
    return g < G ? g : -1;  // behind the last group there is none
  };
  auto front_of = [&](int g) __attribute__((always_inline)) {
    return g < 0 ? 0 : prefix_keys(a, g, starts[g], starts[g + 1]);
  };
  auto own_units = [&](int b, int front) __attribute__((always_inline)) {
    return key_units(front, fitting(a, a.lengths[b]));
  };
  int own[3] = {0, 0, 0}, first[3], all[3];
  for (int g = g0; g < g1; ++g) {
    const int u = group_units(g), t = u > 0 ? group_triples(g) : 0;
    own[0] += on_line(u) * t;
    own[1] += t;
  }
  const int HB = a.Hkv * a.blocks;
  for (int b = b0; b < b1; ++b) own[2] += on_line(own_units(b, front_of(group_at(b)))) * HB;
  block_scan<W>(own, sums, first, all);
  line.total = all[0] + all[2];
  line.stretch = max((line.total + a.grid - 1) / a.grid, kPrefixStretch);
  first[2] += all[0];

  const int64_t at = (int64_t)s * line.stretch;
  if (at >= first[0] && at < (int64_t)first[0] + own[0]) {
    int rest = (int)(at - first[0]), t = first[1];
    for (int g = g0; g < g1; ++g) {
      const int u = group_units(g), n = u > 0 ? group_triples(g) : 0;
      const int len = on_line(u);
      if (rest < len * n) {
        found[0] = 0;
        found[1] = g;
        found[2] = rest / len;
        found[3] = rest % len;
        found[4] = t;
        break;
      }
      rest -= len * n;
      t += n;
    }
  }
  if (at >= first[2] && at < (int64_t)first[2] + own[2]) {
    int rest = (int)(at - first[2]);
    for (int b = b0; b < b1; ++b) {
      const int len = on_line(own_units(b, front_of(group_at(b))));
      if (rest < len * HB) {
        found[0] = 1;
        found[1] = b;
        found[2] = rest / len;
        found[3] = rest % len;
        found[4] = 0;
        break;
      }
      rest -= len * HB;
    }
  }
  if (s == 0) {
    // The join's part: where each sequence's and each group's units lie.
    if (tid == 0) {
      a.ws[0] = line.stretch;
      a.ws[1] = line.bad;
    }
    int base = first[2];
    for (int b = b0; b < b1; ++b) {
      const int g = group_at(b), front = front_of(g), u = own_units(b, front);
      PrefixSeq* const q = prefix_seqs(a) + b;
      q->own_base = base;
      q->own_units = u;
      q->group = g;
      q->member = g < 0 ? 0 : b - starts[g];
      base += on_line(u) * HB;
    }
    PrefixGroup* const gs = reinterpret_cast<PrefixGroup*>(prefix_seqs(a) + a.B);
    int pre = first[0], t = first[1];
    for (int g = g0; g < g1; ++g) {
      const int u = group_units(g), n = u > 0 ? group_triples(g) : 0;
      gs[g] = {pre, u, t, group_triples(g) / a.Hkv};
      pre += on_line(u) * n;
      t += n;
    }
  }
  __syncthreads();
  place->own = uniform(found[0]);
  place->at = uniform(found[1]);
  place->sub = uniform(found[2]);
  place->unit = uniform(found[3]);
  place->first = uniform(found[4]);
  __syncthreads();
  return line;
}

// Slots of pieces: a prefix's hold a.prows rows, a sequence's own keys' a.srows.
__device__ __forceinline__ float* prefix_slot(const PrefixArgs& a, int D, int64_t i) {
  return a.part + i * ((int64_t)a.prows * (D + 4));
}
__device__ __forceinline__ float* own_slot(const PrefixArgs& a, int D, int64_t i) {
  return a.part + a.pslots * ((int64_t)a.prows * (D + 4)) + i * ((int64_t)a.srows * (D + 4));
}

// A piece of work: the rows row0 .. of the sequences from b0 on, `rows` in all, over keys
// [k_lo, k_hi), the first of them k_first (k_lo is that rounded down to 16), in the pages of
// `table`.
struct PrefixJob {
  const int* table;
  int b0, row0, rows, kvh;
  int k_lo, k_first, k_hi;
  float* slot;
  int slot_rows;
};

// What issue_kv_unit asks of a wave's share of a unit.
template <int P>
struct PrefixDma {
  static constexpr int PER_WAVE = P;
  uint32_t voff[P];  // byte offsets in the page's half of the unit
  uint32_t row_bytes;
};

template <int I, int N, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    each<I + 1, N>(f);
  }
}

}  // namespace

// Four waves of 32 query rows over 32-key units, the body of the dense forward's 32x32x16 pipeline
// (fa_fwd.hip): S^T = K Q^T of unit u + 1 and O^T += V^T P^T of unit u - 1 run beside the vector
// work of unit u. Each wave moves its share of a unit's K and V rows to the LDS ring by DMA; a
// share lies within half a unit, so in one page, and is read through a descriptor of that page,
// whose range ends with the keys: rows past them, and in front of the first one, read zeros.
// Waves without rows move their share and wait.
template <int D, class E>
__device__ __forceinline__ void prefix_piece(const PrefixArgs& a, const PrefixJob& job,
                                             half_t* lds) {
  using T = PrefixRing<D>;
  constexpr int NS = T::NS;
  constexpr int IPU = 2 * T::PER_WAVE;
  constexpr int NQ = D / 16;
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int ql = lane & 31;
  const int g = lane >> 5;

  // The lane's row, the keys that it sees, and its query.
  const int r = job.row0 + 32 * wave + ql;
  const bool real = r < job.rows;
  const bool active = uniform(job.row0 + 32 * wave < job.rows) != 0;
  const int member = r / a.R, rr = r - member * a.R;
  const int h = rr / a.N, n = rr - h * a.N;
  const int b = job.b0 + member;
  int see = INT32_MAX, len = 0;
  half8 qf[NQ];
  {
    const half_t* q = a.q + b * a.qs[0] + (int64_t)(job.kvh * a.group + h) * a.qs[1] + n * a.qs[2];
#pragma unroll
    for (int kk = 0; kk < NQ; ++kk) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (real && 16 * kk + 8 * g < a.d) v = *reinterpret_cast<const u32x4*>(q + 16 * kk + 8 * g);
      qf[kk] = __builtin_bit_cast(half8, v);
    }
    if (real) {
      len = a.lengths[b];
      see = min(fitting(a, len) - a.N + n + 1, job.k_hi);
    }
  }
  // Units that end below this need no mask.
  int all_see = see;
#pragma unroll
  for (int i = 32; i > 0; i >>= 1) all_see = min(all_see, __shfl_xor(all_see, i, 64));
  all_see = uniform(min(all_see, job.k_hi));

  const int row_bytes = (int)a.ks[2] * 2;
  const half_t* const k_head = a.k + job.kvh * a.ks[1];
  const half_t* const v_head = a.v + job.kvh * a.ks[1];
  const int units = (job.k_hi - job.k_lo + T::KT - 1) / T::KT;

  // The wave's share of a unit: its 1 KiB pieces, all in half `e` of the unit.
  PrefixDma<T::PER_WAVE> dma;
  const int piece0 = T::INSTR >= kPrefixWaves ? wave * T::PER_WAVE : wave % T::INSTR;
  const int e = piece0 * 1024 / (D * 2) / 16;
  dma.row_bytes = (uint32_t)row_bytes;
#pragma unroll
  for (int i = 0; i < T::PER_WAVE; ++i) {
    const int byte = (piece0 + i) * 1024 + lane * 16;
    const int row = byte / (D * 2);
    const int c = swz_chunk<D>(row, (byte % (D * 2)) / 16);
    dma.voff[i] = 8 * c < a.d ? (uint32_t)((row & 15) * row_bytes + 16 * c) : kOutOfRange;
  }

  // Pages of the half units from unit i & ~31 on, one a lane, and the next 32 units'.
  int bad_key = INT32_MAX;  // first key of the first page that does not exist
  auto half_key = [&](int i) __attribute__((always_inline)) { return job.k_lo + 32 * i + 16 * lane; };
  auto fetch = [&](int i) __attribute__((always_inline)) {
    const int key = half_key(i);
    return key < job.k_hi ? job.table[key / a.S] : 0;
  };
  auto known = [&](int page, int i) __attribute__((always_inline)) {
    const bool ok = page >= 0 && page < a.pages;
    if (!ok) bad_key = min(bad_key, half_key(i));
    return ok ? page : -1;
  };
  int next_page = fetch(0);
  int page = 0, in_page = 0;
  int iu = 0;  // next unit to ask for
  const uint32_t lds0 = lds_addr(lds);
  auto issue = [&](int slot) __attribute__((always_inline)) {
    if ((iu & 31) == 0) {
      page = known(next_page, iu);
      in_page = half_key(iu) % a.S;
      next_page = fetch(iu + 32);
    }
    const int key = job.k_lo + T::KT * iu + 16 * e;
    const int at = 2 * (iu & 31) + e;
    const int pg = __builtin_amdgcn_readlane(page, at);
    const int skip = max(job.k_first - key, 0);  // rows in front of the first key
    const int there = min(job.k_hi - key, 16) - skip;
    const int64_t off = pg * a.ks[0] + (__builtin_amdgcn_readlane(in_page, at) + skip) * a.ks[2];
    const uint32_t bytes = there > 0 && pg >= 0 ? (uint32_t)((there - 1) * row_bytes + a.d * 2) : 0u;
    issue_kv_unit<T::TILE * 2>(dma, make_rsrc_words(k_head + off, bytes),
                               make_rsrc_words(v_head + off, bytes), -skip,
                               lds0 + (uint32_t)slot * (T::STAGE * 2u) + (uint32_t)piece0 * 1024u);
    ++iu;
  };

  // The units end in the ring's last slot: the first turn starts at slot p0.
  const int npad = (units + NS - 1) / NS * NS;
  const int p0 = uniform(npad - units);
#pragma unroll
  for (int u = 0; u < T::AHEAD - T::IN_FLIGHT; ++u) issue(p0 + u < NS ? p0 + u : p0 + u - NS);
  wait_all_vm();
#pragma unroll
  for (int u = T::AHEAD - T::IN_FLIGHT; u < T::AHEAD; ++u)
    issue(p0 + u < NS ? p0 + u : p0 + u - NS);
  // The V tile read as "unit -1" holds zeros (its P is zero too).
  {
    half_t* zs = lds + (p0 > 0 ? p0 - 1 : NS - 1) * T::STAGE + T::TILE;
    unsigned zr;  // from an asm move, so that no loop keeps it in a register
    asm volatile("v_mov_b32 %0, 0" : "=v"(zr));
    const u32x4 z = {zr, zr, zr, zr};
    for (int i = tid; i < T::TILE / 8; i += 64 * kPrefixWaves) *reinterpret_cast<u32x4*>(zs + 8 * i) = z;
  }
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(T::IN_FLIGHT * IPU) : "memory");

  int k_off[NQ];  // row reads of K: row row_perm(ql), chunk 2 kk + g
#pragma unroll
  for (int kk = 0; kk < NQ; ++kk) k_off[kk] = swz_offset<D>(row_perm(ql), 2 * kk + g);
  int v_off[D / 32][2];  // transposed reads of V (see read_tr)
  {
    const int grp = lane >> 4, i = lane & 15, r4 = i >> 2, qq = i & 3;
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
      const int col = 32 * db + 16 * (grp & 1) + 4 * qq;
#pragma unroll
      for (int h2 = 0; h2 < 2; ++h2) {
        const int row = 8 * g + r4 + 4 * h2;
        v_off[db][h2] = row * D + 8 * swz_chunk<D>(row, col >> 3) + (col & 7);
      }
    }
  }
  auto tr8 = [&](const half_t* base, int db) __attribute__((always_inline)) {
    const half4 lo = __builtin_bit_cast(
        half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(base + v_off[db][0])));
    const half4 hi = __builtin_bit_cast(
        half4, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(base + v_off[db][1])));
    half8 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = lo[i];
      v[4 + i] = hi[i];
    }
    return v;
  };

  float16v o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int j = 0; j < 16; ++j) o[db][j] = 0.f;
  float m = -INFINITY;  // the row's reference
  float l = 0.f;        // the lane's sum of the row's probabilities
  const float c = a.c;

  float16v s_cur;  // S^T of the current unit
#pragma unroll
  for (int j = 0; j < 16; ++j) s_cur[j] = 0.f;
  half8 pa_prev[2];  // P^T of the one before
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) pa_prev[i][j] = (half_t)0.f;
  if (active)
#pragma unroll
    for (int kk = 0; kk < NQ; ++kk)
      s_cur = mma<E>(*reinterpret_cast<const half8*>(lds + p0 * T::STAGE + k_off[kk]), qf[kk], s_cur);

  int ka = job.k_lo;  // first key of the unit the body works on
  auto body = [&](auto slot_c) __attribute__((always_inline)) {
    constexpr int SLOT = decltype(slot_c)::value;
    const half_t* nxt = lds + ((SLOT + 1) % NS) * T::STAGE;
    const half_t* prv = lds + ((SLOT + NS - 1) % NS) * T::STAGE;
    if (ka + T::KT > all_see || ka < job.k_first) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int key = ka + result_row(j, g);
        if (key >= see || key < job.k_first) s_cur[j] = -INFINITY;
      }
    }

    // D / 16 S tasks (unit u + 1) and D / 16 O tasks (unit u - 1), alternating; group i issues
    // the LDS reads of task i + LEAD, runs task i and a part of unit u's vector work; fences keep
    // the order.
    constexpr int NTASK = 2 * NQ, LEAD = 3;
    auto load_op = [&](auto t_c) __attribute__((always_inline)) -> half8 {
      constexpr int t = decltype(t_c)::value, q = t / 2;
      if constexpr (t % 2 == 0) return *reinterpret_cast<const half8*>(nxt + k_off[q]);
      else return tr8(prv + T::TILE + 16 * (q / (D / 32)) * D, q % (D / 32));
    };
    float16v s_nx;
#pragma unroll
    for (int j = 0; j < 16; ++j) s_nx[j] = 0.f;
    auto run_task = [&](auto t_c, const half8& op) __attribute__((always_inline)) {
      constexpr int t = decltype(t_c)::value, q = t / 2;
      if constexpr (t % 2 == 0) s_nx = mma<E>(op, qf[q], s_nx);
      else o[q % (D / 32)] = mma<E>(op, pa_prev[q / (D / 32)], o[q % (D / 32)]);
    };
    // Vector work of a pair of values in three stages, each in a group of its own: the exponent's
    // argument, p, and sums and rounding.
    half8 pa[2];
    float targ[16], pexp[16], lsum[2];
    float ref = m;
    auto stage_f = [&](int pr) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 2; ++i) targ[2 * pr + i] = fmaf(s_cur[2 * pr + i], c, -ref);
      asm volatile("" : "+v"(targ[2 * pr]), "+v"(targ[2 * pr + 1]));
    };
    auto stage_a = [&](int pr) __attribute__((always_inline)) {
      float p2[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) p2[i] = exp2_fast(targ[2 * pr + i]);
      asm volatile("" : "+v"(p2[0]), "+v"(p2[1]));
      pexp[2 * pr] = p2[0];
      pexp[2 * pr + 1] = p2[1];
    };
    auto stage_b = [&](int pr) __attribute__((always_inline)) {
      half2v pp;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        lsum[i] = pr == 0 ? pexp[i] : lsum[i] + pexp[2 * pr + i];
        pp[i] = to_elem<E>(pexp[2 * pr + i]);
      }
      asm volatile("" : "+v"(pp));
      const int j = 2 * pr;
      pa[j >> 3][j & 7] = pp[0];
      pa[j >> 3][(j & 7) + 1] = pp[1];
    };
    half8 op[NTASK];
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" : "+v"(ref));
    each<0, (LEAD < NTASK ? LEAD : NTASK)>(
        [&](auto t_c) __attribute__((always_inline)) { op[decltype(t_c)::value] = load_op(t_c); });
#pragma unroll
    for (int pr = 0; pr < 8; ++pr)
      if ((2 * pr * NTASK) / 16 == 0) stage_f(pr);
    __builtin_amdgcn_sched_barrier(0);
    each<0, NTASK>([&](auto i_c) __attribute__((always_inline)) {
      constexpr int i = decltype(i_c)::value;
      if constexpr (i + LEAD < NTASK) op[i + LEAD] = load_op(std::integral_constant<int, i + LEAD>{});
      run_task(i_c, op[i]);
#pragma unroll
      for (int pr = 0; pr < 8; ++pr) {
        const int ga = (2 * pr * NTASK) / 16;
        const int gb = ga + 1 < NTASK ? ga + 1 : NTASK - 1;
        if (ga == i) stage_a(pr);
        if (gb == i) stage_b(pr);
      }
#pragma unroll
      for (int pr = 0; pr < 8; ++pr)
        if ((2 * pr * NTASK) / 16 == i + 1) stage_f(pr);
      __builtin_amdgcn_sched_barrier(0);
    });

    // The row's sum of unit u; rarely, the reference moves.
    float l_u = lsum[0] + lsum[1];
    const float held = kPrefixWide<E> ? l + l_u : l_u;
    if (__builtin_amdgcn_ballot_w64(!(held <= kPrefixSumLimit<E>)) != 0) {
      float mt = s_cur[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) mt = __builtin_fmaxf(mt, s_cur[j]);
      float m_new = __builtin_fmaxf(m, halves_max(mt) * c - kPrefixShift<E>);
      if constexpr (kPrefixWide<E>)
        m_new = __builtin_fmaxf(m_new, m + log2_fast(halves_max(l)) - kPrefixShift<E>);
      const float to = exp_reference(m_new);
      const float alpha = exp2_fast(m - to);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] *= alpha;
      m = m_new;
      l_u = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float p = exp2_fast(fmaf(s_cur[j], c, -to));
        l_u += p;
        pa[j >> 3][j & 7] = to_elem<E>(p);
      }
    }
    l += l_u;
    s_cur = s_nx;
#pragma unroll
    for (int i = 0; i < 2; ++i) pa_prev[i] = pa[i];
  };
  auto step = [&](auto p_c) __attribute__((always_inline)) {
    constexpr int P = decltype(p_c)::value;
    issue((P + T::AHEAD) % NS);
    if (active) body(p_c);
    ka += T::KT;
    wait_vm_and_barrier<T::IN_FLIGHT * IPU>();
  };
  each<0, NS>([&](auto p_c) __attribute__((always_inline)) {
    if (decltype(p_c)::value >= p0) step(p_c);
  });
  for (int u = NS; u < npad; u += NS) each<0, NS>([&](auto p_c) __attribute__((always_inline)) { step(p_c); });
  // O of the last unit, which lies in the ring's last slot.
  if (active) {
    const half_t* prv = lds + (NS - 1) * T::STAGE + T::TILE;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int db = 0; db < D / 32; ++db) o[db] = mma<E>(tr8(prv + 16 * i * D, db), pa_prev[i], o[db]);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");

  // The piece: lane (row ql, half g) holds d = 32 db + 8 (j / 4) + 4 g + j % 4 of O.
#pragma unroll
  for (int i = 32; i > 0; i >>= 1) bad_key = min(bad_key, __shfl_xor(bad_key, i, 64));
  float lt = halves_sum(l);
  if (len > bad_key) lt = __builtin_nanf("");  // the row's sequence needs a page that does not exist
  if (real) {
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
    const int row = 32 * wave + ql;
    float* const out = job.slot + (int64_t)row * D;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int jq = 0; jq < 4; ++jq) {
        float4v v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = o[db][4 * jq + i] * inv;
        *reinterpret_cast<float4v*>(out + 32 * db + 8 * jq + 4 * g) = v;
      }
    if (g == 0)
      job.slot[(int64_t)job.slot_rows * D + row] = lt == 0.f ? -INFINITY : m + log2_fast(lt);
  }
  __syncthreads();
}

template <int D, class E>
__global__ __launch_bounds__(64 * kPrefixWaves, PrefixRing<D>::WGS) void prefix_fwd_kernel(PrefixArgs a) {
  __shared__ __attribute__((aligned(1024))) half_t lds[PrefixRing<D>::HALVES];
  static_assert(sizeof(lds) >= (32 + kPrefixStarts) * 4, "the line is found in the ring's memory");
  const int s = blockIdx.x;
  PrefixPlace at;
  const PrefixLine line = prefix_find(a, s, reinterpret_cast<int*>(lds), &at);
  const int64_t from = (int64_t)s * line.stretch;
  if (from >= line.total) return;
  int left = min(line.stretch, (int)(line.total - from));
  const int G = line.bad ? 0 : a.G;
  const int HB = a.Hkv * a.blocks;
  PrefixJob job;
  int units = 0, subs = 0, tiles = 1, k0 = 0, k_first = 0, k_end = 0;
  bool turned = true;  // to another group or sequence
  while (true) {
    if (turned) {
      if (at.own == 0 && at.at >= G) at = {1, 0, 0, 0, 0};
      if (at.own == 0) {
        job.b0 = uniform(a.starts[at.at]);
        const int end = uniform(a.starts[at.at + 1]);
        k_first = 0;
        k_end = uniform(prefix_keys(a, at.at, job.b0, end));
        tiles = prefix_tiles(end - job.b0, a.R);
        job.rows = (end - job.b0) * a.R;
        job.slot_rows = a.prows;
      } else {
        job.b0 = at.at;
        const int g = G > 0 ? uniform(group_of(a.starts, G, at.at)) : -1;
        k_first = g < 0 || g >= G ? 0 : uniform(prefix_keys(a, g, a.starts[g], a.starts[g + 1]));
        k_end = uniform(fitting(a, a.lengths[at.at]));
        tiles = a.blocks;
        job.rows = a.R;
        job.slot_rows = a.srows;
      }
      job.table = a.table + job.b0 * a.table_stride;
      units = key_units(k_first, k_end);
      subs = units > 0 ? tiles * a.Hkv : 0;
      k0 = k_first & ~15;
      turned = false;
    }
    if (at.sub >= subs) {
      at.first += subs;
      ++at.at;
      at.sub = 0;
      turned = true;
      continue;
    }
    // The part of the triple's units that is the work-group's.
    const int len = units + kPrefixLead;
    const int u0 = max(at.unit - kPrefixLead, 0);
    const int u1 = left < len - at.unit ? max(at.unit + left - kPrefixLead, 0) : units;
    if (u1 > u0) {
      job.kvh = at.sub / tiles;
      job.row0 = (at.sub - job.kvh * tiles) * kPrefixTile;
      job.k_lo = k0 + 32 * u0;
      job.k_first = max(k_first, job.k_lo);
      job.k_hi = min(k_end, k0 + 32 * u1);
      job.slot = at.own == 0 ? prefix_slot(a, D, (int64_t)s + at.first + at.sub)
                             : own_slot(a, D, (int64_t)s + (int64_t)at.at * HB + at.sub);
      prefix_piece<D, E>(a, job, lds);
    }
    left -= len - at.unit;
    if (left <= 0) return;
    at.unit = 0;
    ++at.sub;
  }
}

// Joins the pieces of each row: those of its group's prefix, then those of its own keys. A lane
// holds four columns of a row, a wave 64 / (D / 4) rows, one after the other in the output; a
// block's four waves take every fourth piece of the same rows and merge through LDS, in a fixed
// order. A piece weighs exp2 of its log-sum-exp against the others'.
template <int D, class E>
__global__ __launch_bounds__(64 * kPrefixWaves) void prefix_join_kernel(PrefixArgs a) {
  constexpr int W = kPrefixWaves;
  constexpr int COLS = D / 4, RPP = 64 / COLS;
  constexpr int AHEAD = 4;
  // The weight of the largest piece: those of 1024 pieces sum to 1/2, so that sums of values near
  // 2^128 stay in float32.
  constexpr float kWeight = 0x1p-11f;
  __shared__ __attribute__((aligned(16))) float acc_s[W][64][4];
  __shared__ float m_s[W][64], l_s[W][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * RPP + lane / COLS;  // of the output [B, Hq, N]
  const int col = 4 * (lane % COLS);
  const int64_t seq_rows = (int64_t)a.Hkv * a.R;
  const bool real = row < a.B * seq_rows;
  const int64_t rr = real ? row : 0;
  const int b = (int)(rr / seq_rows), in_seq = (int)(rr - b * seq_rows);
  const int kvh = in_seq / a.R, r = in_seq - kvh * a.R;
  const int stretch = a.ws[0];
  const bool bad = a.ws[1] != 0;
  const int len = a.lengths[b];
  const PrefixSeq q = prefix_seqs(a)[b];
  PrefixGroup grp = {0, 0, 0, 0};
  if (q.group >= 0) grp = reinterpret_cast<const PrefixGroup*>(prefix_seqs(a) + a.B)[q.group];

  // The stretches s0 .. s1 that hold the units of triple `sub`, whose line begins at `base`.
  auto range = [&](int base, int units, int sub, int* s0, int* s1) __attribute__((always_inline)) {
    const int64_t at = base + (int64_t)sub * on_line(units) + kPrefixLead;
    *s0 = (int)(at / stretch);
    *s1 = units > 0 ? (int)((at + units - 1) / stretch) : *s0 - 1;
  };
  int p0, p1, q0, q1;
  const int64_t gr = (int64_t)q.member * a.R + r;
  const int psub = kvh * grp.tiles + (int)(gr / kPrefixTile);
  range(grp.base, grp.units, psub, &p0, &p1);
  const int osub = kvh * a.blocks + r / kPrefixTile;
  range(q.own_base, q.own_units, osub, &q0, &q1);
  const int np = p1 - p0 + 1, count = real ? np + (q1 - q0 + 1) : 0;
  struct Piece {
    float lse;
    float4v o;
  };
  auto load = [&](int i) __attribute__((always_inline)) {
    Piece p = {-INFINITY, {0.f, 0.f, 0.f, 0.f}};
    if (i < count) {
      const bool pre = i < np;
      const float* slot = pre ? prefix_slot(a, D, (int64_t)p0 + i + grp.first + psub)
                              : own_slot(a, D, (int64_t)q0 + (i - np) + (int64_t)b * a.Hkv * a.blocks + osub);
      const int at = pre ? (int)(gr % kPrefixTile) : r % kPrefixTile;
      p.lse = slot[(int64_t)(pre ? a.prows : a.srows) * D + at];
      p.o = *reinterpret_cast<const float4v*>(slot + (int64_t)at * D + col);
    }
    return p;
  };
  float m = -INFINITY, l = 0.f;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = wave; i0 < count; i0 += W * AHEAD) {
    Piece p[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) p[i] = load(i0 + W * i);
    float mx = m;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) mx = __builtin_fmaxf(mx, p[i].lse);
    const float ref = exp_reference(mx);
    const float keep = m == -INFINITY ? 0.f : exp2_fast(m - ref);
    l *= keep;
    acc *= keep;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float f = p[i].lse == -INFINITY ? 0.f : exp2_fast(p[i].lse - ref) * kWeight;
      l += f;
      acc += p[i].o * f;
    }
    m = mx;
  }
  *reinterpret_cast<float4v*>(acc_s[wave][lane]) = acc;
  m_s[wave][lane] = m;
  l_s[wave][lane] = l;
  __syncthreads();
  if (wave != 0 || !real || col >= a.d) return;
  float mx = -INFINITY;
#pragma unroll
  for (int i = 0; i < W; ++i) mx = __builtin_fmaxf(mx, m_s[i][lane]);
  float lt = 0.f;
  float4v v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float f = m_s[i][lane] == -INFINITY ? 0.f : exp2_fast(m_s[i][lane] - mx);
    lt += f * l_s[i][lane];
    v += *reinterpret_cast<const float4v*>(acc_s[i][lane]) * f;
  }
  v *= lt == 0.f ? 0.f : 1.0f / lt;  // a row that saw no key is 0
  if (bad || len < 0 || len > a.M * a.S) {
    const float nan = __builtin_nanf("");
    v = {nan, nan, nan, nan};
  }
  *reinterpret_cast<u32x2*>(a.o + row * a.d + col) = pack4<E>(v[0], v[1], v[2], v[3]);
}

static int prefix_width(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

PrefixSizes prefix_sizes(int64_t B, int64_t G, int64_t Hkv, int64_t R, int64_t D, int64_t keys) {
  PrefixSizes z;
  z.blocks = prefix_tiles(R, 1);
  z.prows = std::min<int64_t>(kPrefixTile, B * R);
  z.srows = std::min<int64_t>(kPrefixTile, R);
  // Groups of two sequences or more have prefixes, in at most so many tiles.
  const int64_t groups = std::min(G, B / 2), own = B * Hkv * z.blocks;
  const int64_t triples = groups > 0 ? Hkv * (B * R / kPrefixTile + groups) : 0;
  const double each = (double)((keys + 31) / 32 + 1 + kPrefixLead);
  z.units = each * ((double)triples + (double)own);
  const int64_t most = 256 * (prefix_width(D) == 128 ? 2 : 3);
  z.grid = (int)std::max(1.0, std::min((double)most, z.units / kPrefixStretch));
  z.pslots = triples > 0 ? z.grid + triples : 0;
  z.head_bytes = (64 + B * (int64_t)sizeof(PrefixSeq) + G * (int64_t)sizeof(PrefixGroup) + 63) / 64 * 64;
  const int64_t rows = z.pslots * z.prows + (z.grid + own) * z.srows;
  z.bytes = z.head_bytes + rows * (prefix_width(D) + 4) * 4;
  return z;
}

template <int D, class E>
hipError_t prefix_start(const PrefixArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL((prefix_fwd_kernel<D, E>), dim3((unsigned)a.grid), dim3(64 * kPrefixWaves), 0,
                     stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  constexpr int RPP = 64 / (D / 4);
  const int64_t rows = (int64_t)a.B * a.Hkv * a.R;
  hipLaunchKernelGGL((prefix_join_kernel<D, E>), dim3((unsigned)((rows + RPP - 1) / RPP)),
                     dim3(64 * kPrefixWaves), 0, stream, a);
  return hipGetLastError();
}

hipError_t launch_prefix_fwd(const PrefixArgs& a, int dtype, hipStream_t stream) {
  const bool bf = dtype == kBF16;
  switch (prefix_width(a.d)) {
    case 32: return bf ? prefix_start<32, BF16>(a, stream) : prefix_start<32, F16>(a, stream);
    case 64: return bf ? prefix_start<64, BF16>(a, stream) : prefix_start<64, F16>(a, stream);
    default: return bf ? prefix_start<128, BF16>(a, stream) : prefix_start<128, F16>(a, stream);
  }
}

}  // namespace fa
