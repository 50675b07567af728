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
#include <cmath>
#include <type_traits>

#include "fa_common.hpp"
#include "fa_layer.hpp"

namespace fa {

// The work is a list of triples: (group, key/value head, tile of 128 query rows) over the keys of
// the group's prefix, and (sequence, key/value head, tile) over a sequence's own keys. A tile's
// rows are those that read the key/value head: the group's heads and the N tokens of one sequence
// after the other. A work-group writes what it has of a triple as one piece, normalised partial O
// and base-2 log-sum-exp of each row, into a slot of its own.
//
// Prefixes meet many rows: a work-group's four waves share each unit of 32 keys (prefix_piece). A
// sequence's own keys meet few, rarely more than 32 in decoding, and come in many short triples: there
// each wave works on a triple of its own, with tiles of 32 rows, so that eight are open on a CU
// (own_piece); with many rows a head they go the prefixes' way (WAVES false).
//
// Units of all triples lie on a line, each triple's behind `lead` empty ones that stand for opening
// and closing a piece; the line is cut into equal stretches, one a work-group or a wave, found from
// the lengths on the GPU, as in fa_paged.hip. Stretch s has its piece of the line's triple t in
// slot s + t, which no two pieces share since from one piece to the next either s or t grows by one.
//
// A prefix that is long against a stretch is not on the line: each of its triples is cut into k
// equal pieces, so that no work-group opens two, and the tiles of one range of keys go to
// neighbouring work-groups of one XCD, whose L2 then reads the keys once for all of them.
//
// Measured (Hq32 Hkv8 D128): 64 sequences over 4096 shared keys and up to 1024 of their own, bf16, 154 MB:
// 37 us and 7 for the join; 128 sequences over 32768 shared keys, fp16, 70 GFLOP: 114-160 and 12. About 6 us
// go into finding the work and 5 until the first keys arrive.
constexpr int kPrefixWaves = 4;

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

// Work-groups that the chip holds, and pieces of one row: one a work-group of its group's prefix, and
// one a wave of its own keys.
constexpr int kPrefixMostGrid = 256 * PrefixRing<64>::WGS;
constexpr int kPrefixMostPieces = kPrefixMostGrid * (1 + kPrefixWaves);

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
__device__ __forceinline__ int on_line(int units, int lead) { return units > 0 ? units + lead : 0; }

// A place: unit `unit` (lead included) of triple `sub` (head-major) of group or sequence `at`, and
// what its keys are.
struct PrefixPlace {
  int kind;    // 0: a group's prefix on the line, 1: a sequence's own keys, 2: a piece of a long prefix
  int at, sub, unit;
  int first;   // kind 0: the line's triple index of the group's first triple
  int b0, n;   // first sequence and number of sequences of the rows
  int k_first, k_end;
  int g, g_end;  // kind 1: the sequence's group, and the first sequence behind it
};
struct PrefixLine {
  int stretch, left;  // a work-group's; left: 0 where it has nothing to do
  int s;              // its stretch, or its place among the pieces of long prefixes
  int pieces;         // of long prefixes
  bool own;           // it, or its waves, take sequences' own keys
  bool bad;           // the groups' starts do not ascend within [0, B]
};

// What the join needs, written by block 0: the stretch, a wave's stretch, whether the starts are bad,
// and the long prefixes' pieces; then every sequence's and every
// group's places.
__device__ __forceinline__ PrefixSeq* prefix_seqs(const PrefixArgs& a) {
  return reinterpret_cast<PrefixSeq*>(a.ws + 16);
}
__device__ __forceinline__ PrefixGroup* prefix_groups(const PrefixArgs& a) {
  return reinterpret_cast<PrefixGroup*>(prefix_seqs(a) + a.B);
}

// Whether a prefix of `units` units is cut into pieces instead of lying on the line whose stretches
// are of L.
__device__ __forceinline__ bool prefix_long(int units, int L) {
  return L >= 2 * kPrefixLead && units >= 2 * (L - kPrefixLead);
}

// A wave's stretch of the sequences' own keys, where a work-group's is L: four waves take five units
// of them in the time that it takes for four of a prefix. (Hq32 Hkv8 D128 bf16; 64 sequences over 4096
// shared keys, 8 groups of 8 with up to 2000 keys of their own: 43.7 and 100 us; 4 for 4 43.7 and 98; 6 for
// 4 45.5 and 101. Of 5 tokens and 8192 shared keys: 44.4, 44.5 and 43.7.)
__device__ __forceinline__ int own_stretch(int L) { return max((5 * L + 15) / 16, 2); }

// The work-group's place, or the wave's. `lds`: the work-group's memory, free before and after.
template <bool WAVES>
__device__ __forceinline__ PrefixLine prefix_find(const PrefixArgs& a, int* lds, PrefixPlace* place) {
  constexpr int W = kPrefixWaves, T = 64 * W;
  int(*const found)[12] = reinterpret_cast<int(*)[12]>(lds);    // [W]
  int* const wrongs = lds + 48;                                // [W]
  int(*const sums)[1] = reinterpret_cast<int(*)[1]>(lds + 52);  // [W]
  int* const kept_starts = lds + 96;
  int* const kept_prefix = kept_starts + kPrefixKeptGroups;
  int* const kept_lengths = kept_prefix + kPrefixKeptGroups;
  const int tid = threadIdx.x;
  bool wrong = false;
  for (int g = tid; g <= a.G; g += T) {
    const int x = a.starts[g];
    wrong |= x < 0 || x > a.B || (g > 0 && a.starts[g - 1] > x);
    if (a.G < kPrefixKeptGroups) {
      kept_starts[g] = x;
      if (g < a.G) kept_prefix[g] = a.prefix[g];
    }
  }
  if (a.B <= kPrefixKeptSeqs)
    for (int b = tid; b < a.B; b += T) kept_lengths[b] = a.lengths[b];
  if ((tid & 63) == 0) wrongs[tid >> 6] = 0;
  if (wrong) wrongs[tid >> 6] = 1;
  __syncthreads();
  PrefixLine line;
  line.bad = uniform(wrongs[0] | wrongs[1] | wrongs[2] | wrongs[3]) != 0;
  const int G = line.bad ? 0 : a.G;
  auto start = [&](int g) __attribute__((always_inline)) {
    return a.G < kPrefixKeptGroups ? kept_starts[g] : a.starts[g];
  };
  auto length = [&](int b) __attribute__((always_inline)) {
    return fitting(a, a.B <= kPrefixKeptSeqs ? kept_lengths[b] : a.lengths[b]);
  };
  // Prefix keys of group g, and its triples.
  auto front_of = [&](int g) __attribute__((always_inline)) {
    const int b = start(g), e = start(g + 1);
    if (e - b < 2) return 0;
    const int keys = a.G < kPrefixKeptGroups ? kept_prefix[g] : a.prefix[g];
    return min(max(keys, 0), length(b));
  };
  auto triples_of = [&](int g) __attribute__((always_inline)) {
    return prefix_tiles(start(g + 1) - start(g), a.R) * a.Hkv;
  };
  // The last group that begins at sequence b or before, -1 or G for a sequence outside all.
  auto group_at = [&](int b) __attribute__((always_inline)) {
    int g = -1;
    for (int step = 1 << (31 - __builtin_clz(G + 1)); step > 0; step >>= 1)
      if (g + step <= G && start(g + step) <= b) g += step;
    return g;
  };
  auto front_at = [&](int g) __attribute__((always_inline)) { return g >= 0 && g < G ? front_of(g) : 0; };

  // A lane's groups, alike in every wave, and a thread's sequences. (One of each is the rule: what is
  // known of the first is kept.)
  const int lane = tid & 63;
  const int per_g = (G + 63) / 64, g0 = min(G, lane * per_g), g1 = min(G, g0 + per_g);
  const int per_b = (a.B + T - 1) / T, b0 = min(a.B, tid * per_b), b1 = min(a.B, b0 + per_b);
  const int HB = a.Hkv * a.blocks, lead = WAVES ? kOwnLead : kPrefixLead;
  const int g0_keys = g0 < g1 ? front_of(g0) : 0, g0_triples = g0 < g1 ? triples_of(g0) : 0;
  auto keys_in = [&](int g) __attribute__((always_inline)) { return g == g0 ? g0_keys : front_of(g); };
  auto triples_in = [&](int g) __attribute__((always_inline)) { return g == g0 ? g0_triples : triples_of(g); };
  const int b0_group = G > 0 && b0 < b1 ? group_at(b0) : -1;
  const int b0_front = front_at(b0_group), b0_end = b0 < b1 ? length(b0) : 0;
  auto group_in = [&](int b) __attribute__((always_inline)) {
    return b == b0 ? b0_group : G > 0 ? group_at(b) : -1;
  };
  auto front_in = [&](int b, int g) __attribute__((always_inline)) { return b == b0 ? b0_front : front_at(g); };
  auto end_in = [&](int b) __attribute__((always_inline)) { return b == b0 ? b0_end : length(b); };
  // Units of sequences' own keys and of the prefixes, on the line.
  int own[1] = {0}, own_before[1], own_all[1];
  for (int b = b0; b < b1; ++b)
    own[0] += on_line(key_units(front_in(b, group_in(b)), end_in(b)), lead) * HB;
  block_scan<W>(own, sums, own_before, own_all);
  own_all[0] = uniform(own_all[0]);
  // Of the lane's groups: pieces of the long prefixes; units and triples of the others on the line;
  // units of the long ones. And the sums of the lanes before, and all.
  int x[4], before[4], all[4];
  auto sum = [&](int i) __attribute__((always_inline)) {
    const int incl = wave_scan(x[i]);
    before[i] = incl - x[i];
    all[i] = __builtin_amdgcn_readlane(incl, 63);
  };
  x[1] = 0;
  for (int g = g0; g < g1; ++g) x[1] += on_line(key_units(0, keys_in(g)), kPrefixLead) * triples_in(g);
  sum(1);
  // (The line's two parts end with a stretch of their own each.)
  const int room = a.grid - 2;
  const int own_cost = WAVES ? own_all[0] - own_all[0] / 5 : own_all[0];
  const int L = max((all[1] + own_cost + room - 1) / room, kPrefixStretch);
  // Long prefixes are cut by the work-groups that the line leaves: of all[3] units in all, a triple
  // of u into the whole part of u / all[3] of those, but of 16 units at least. (32 sequences, Hq32 Hkv8 D128,
  // four groups over 2048 keys each, or 40 over 8192: 35.5 and 32 us; of 8 at least 36 and 34, of 32 41 and
  // 36.) Where the grid would not hold the pieces, they stay on the line.
  const bool any = all[1] > 0;
  bool cut = any;
  int budget = 0;
  auto cuts_of = [&](int u) __attribute__((always_inline)) {
    return cut && prefix_long(u, L) ? max(1, min((int)((double)u * budget / all[3]), u / 16)) : 0;
  };
  x[0] = x[2] = x[3] = 0;
  sum(0);
  sum(2);
  while (any) {
    x[0] = x[1] = x[2] = x[3] = 0;
    before[0] = all[0] = 0;
    for (int g = g0; g < g1; ++g) {
      const int u = key_units(0, keys_in(g)), t = u > 0 ? triples_in(g) : 0;
      if (cut && prefix_long(u, L)) {
        x[3] += u * t;
      } else {
        x[1] += on_line(u, kPrefixLead) * t;
        x[2] += t;
      }
    }
    sum(1);
    sum(2);
    sum(3);
    if (all[3] == 0) break;
    const int each = WAVES ? W * own_stretch(L) : L;
    const int rest = WAVES ? (all[1] + L - 1) / L + (own_all[0] + each - 1) / each
                           : (all[1] + own_all[0] + L - 1) / L;
    budget = min(a.grid - rest, a.most_pieces) & ~7;
    for (int g = g0; g < g1; ++g) x[0] += cuts_of(key_units(0, keys_in(g))) * triples_in(g);
    sum(0);
    if ((all[0] + 7) / 8 * 8 <= a.grid - rest) break;
    cut = false;
  }
  line.stretch = L;
  line.pieces = all[0];

  // Block i takes pieces of long prefixes first, an XCD consecutive ones, then a stretch of the
  // others, then sequences' own keys.
  const int xcd = blockIdx.x % 8, i = blockIdx.x / 8, each = (all[0] + 7) / 8;
  const bool piece = i < each;
  line.s = piece ? xcd * each + i : (i - each) * 8 + xcd;
  const int stretches = WAVES ? (all[1] + L - 1) / L : 0;
  line.own = !piece && WAVES && line.s >= stretches;
  int mine = L, end = WAVES ? all[1] : all[1] + own_all[0];  // of the line
  if (line.own) {
    line.s = (line.s - stretches) * W + (tid >> 6);
    mine = own_stretch(L);
    end = own_all[0];
  }
  int64_t from = (int64_t)line.s * mine;
  line.left = piece ? (line.s < all[0] ? 1 : 0) : from < end ? (int)min((int64_t)mine, end - from) : 0;
  if (piece) {
    if (tid < 64 && line.s >= before[0] && line.s < before[0] + x[0]) {
      int at = line.s - before[0];
      for (int g = g0; g < g1; ++g) {
        const int keys = keys_in(g), u = key_units(0, keys), k = cuts_of(u);
        const int n = triples_in(g) * k;
        if (at >= n) {
          at -= n;
          continue;
        }
        // piece p of head kvh, tile t: place (kvh k + p) tiles + t
        const int tiles = triples_in(g) / a.Hkv, t = at % tiles, p = at / tiles % k;
        int* const f = found[0];
        f[0] = 2;
        f[1] = g;
        f[2] = at / tiles / k * tiles + t;
        f[3] = 0;
        f[4] = 0;
        f[5] = start(g);
        f[6] = start(g + 1) - start(g);
        f[7] = 32 * (int)((int64_t)u * p / k);
        f[8] = min(keys, 32 * (int)((int64_t)u * (p + 1) / k));
        break;
      }
    }
  } else {
    if (!line.own && tid < 64 && from >= before[1] && from < (int64_t)before[1] + x[1]) {
      int at = (int)(from - before[1]), t = before[2];
      for (int g = g0; g < g1; ++g) {
        const int keys = keys_in(g), u = key_units(0, keys);
        const int n = u > 0 && !(cut && prefix_long(u, L)) ? triples_in(g) : 0;
        const int len = on_line(u, kPrefixLead);
        if (at < len * n) {
          int* const f = found[0];
          f[0] = 0;
          f[1] = g;
          f[2] = at / len;
          f[3] = at % len;
          f[4] = t;
          f[5] = start(g);
          f[6] = start(g + 1) - start(g);
          f[7] = 0;
          f[8] = keys;
          break;
        }
        at -= len * n;
        t += n;
      }
    }
    // The waves' places, or the work-group's.
    if (line.own || !WAVES)
      for (int w = 0; w < (WAVES ? W : 1); ++w) {
        if (WAVES) from = (int64_t)((line.s & ~(W - 1)) + w) * mine;
        else from = (int64_t)line.s * mine - all[1];
        if (from < own_before[0] || from >= (int64_t)own_before[0] + own[0]) continue;
        int at = (int)(from - own_before[0]);
        for (int b = b0; b < b1; ++b) {
          const int g = group_in(b), keys = front_in(b, g), stop = end_in(b);
          const int len = on_line(key_units(keys, stop), lead);
          if (at < len * HB) {
            int* const f = found[w];
            f[0] = 1;
            f[1] = b;
            f[2] = at / len;
            f[3] = at % len;
            f[4] = 0;
            f[5] = b;
            f[6] = 1;
            f[7] = keys;
            f[8] = stop;
            f[9] = g;
            f[10] = g < 0 ? (G > 0 ? start(0) : a.B) : g < G ? start(g + 1) : a.B;
            break;
          }
          at -= len * HB;
        }
      }
  }
  if (blockIdx.x == 0) {
    if (tid == 0) {
      a.ws[0] = L;
      a.ws[1] = WAVES ? own_stretch(L) : L;
      a.ws[2] = line.bad;
      a.ws[3] = all[0];
    }
    int base = (WAVES ? 0 : all[1]) + own_before[0];
    for (int b = b0; b < b1; ++b) {
      const int g = group_in(b), u = key_units(front_in(b, g), end_in(b));
      const bool in = g >= 0 && g < G;
      PrefixSeq* const q = prefix_seqs(a) + b;
      q->own_base = base;
      q->own_units = u;
      q->group = in ? g : -1;
      q->member = in ? b - start(g) : 0;
      base += on_line(u, lead) * HB;
    }
    int pieces = before[0], t = before[2];
    base = before[1];
    for (int g = tid < 64 ? g0 : g1; g < g1; ++g) {
      const int u = key_units(0, keys_in(g)), n = triples_in(g), k = cuts_of(u);
      prefix_groups(a)[g] = {k > 0 ? pieces : base, u, t, n / a.Hkv, k, 0, 0, 0};
      if (k > 0) {
        pieces += n * k;
      } else if (u > 0) {
        base += on_line(u, kPrefixLead) * n;
        t += n;
      }
    }
  }
  __syncthreads();
  const int* const f = found[line.own ? tid >> 6 : 0];
  place->kind = uniform(f[0]);
  place->at = uniform(f[1]);
  place->sub = uniform(f[2]);
  place->unit = uniform(f[3]);
  place->first = uniform(f[4]);
  place->b0 = uniform(f[5]);
  place->n = uniform(f[6]);
  place->k_first = uniform(f[7]);
  place->k_end = uniform(f[8]);
  place->g = uniform(f[9]);
  place->g_end = uniform(f[10]);
  line.s = uniform(line.s);
  line.left = uniform(line.left);
  __syncthreads();
  return line;
}

// Turns to the next sequence that has keys of its own; false behind the last.
__device__ __forceinline__ bool next_sequence(const PrefixArgs& a, PrefixPlace& at) {
  do {
    ++at.at;
    while (at.at >= at.g_end && at.at < a.B) {  // in the next group, or behind the last
      const int begin = at.g_end;
      ++at.g;
      at.g_end = at.g < a.G ? uniform(a.starts[at.g + 1]) : a.B;
      at.k_first = at.g < a.G ? uniform(prefix_keys(a, at.g, begin, at.g_end)) : 0;
    }
    if (at.at >= a.B) return false;
    at.k_end = uniform(fitting(a, a.lengths[at.at]));
  } while (key_units(at.k_first, at.k_end) == 0);
  at.b0 = at.at;
  return true;
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

// A wave's share of a unit: one or two of the 1 KiB pieces of its K rows and of its V rows.
template <int P>
struct PrefixDma {
  static_assert(P == 1 || P == 2, "one or two pieces");
  uint32_t voff[P];  // byte offsets in the page's half of the unit
};
// Moves the share to the LDS tiles at `base` (K) and base + TILE_BYTES (V); `back` bytes are taken
// off the offsets. The descriptors' words come from v_readlane, and a load may read such a register
// five wait states later at the earliest, and M0 one behind its write: the compiler does not look into
// the block for either, so the block waits.
template <int TILE_BYTES, int P>
__device__ __forceinline__ void issue_unit(const PrefixDma<P>& dma, int4v r_k, int4v r_v, uint32_t back,
                                           uint32_t base) {
  const uint32_t v0 = dma.voff[0] - back;
  uint32_t saved;
  if constexpr (P == 1) {
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %4\n\t"
        "s_nop 2\n\t"
        "buffer_load_dwordx4 %1, %2, 0 offen lds\n\t"
        "s_mov_b32 m0, %5\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(v0), "s"(r_k), "s"(r_v), "s"(base), "s"(base + TILE_BYTES)
        : "memory");
  } else {
    const uint32_t v1 = dma.voff[1] - back;
    asm volatile(
        "s_mov_b32 %0, m0\n\t"
        "s_mov_b32 m0, %5\n\t"
        "s_nop 2\n\t"
        "buffer_load_dwordx4 %1, %3, 0 offen lds\n\t"
        "s_mov_b32 m0, %6\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %2, %3, 0 offen lds\n\t"
        "s_mov_b32 m0, %7\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %1, %4, 0 offen lds\n\t"
        "s_mov_b32 m0, %8\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %2, %4, 0 offen lds\n\t"
        "s_mov_b32 m0, %0"
        : "=&s"(saved)
        : "v"(v0), "v"(v1), "s"(r_k), "s"(r_v), "s"(base), "s"(base + 1024u), "s"(base + TILE_BYTES),
          "s"(base + TILE_BYTES + 1024u)
        : "memory");
  }
}

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
  // (from an asm statement, so that what follows from it is not kept from one piece to the next)
  int tid = threadIdx.x;
  asm volatile("" : "+v"(tid));
  const int lane = tid & 63;
  const int wave = uniform(tid >> 6);
  const int ql = lane & 31;
  const int g = lane >> 5;

  // Pages of half units, one a lane, clamped to the last key's, so that the load needs no branch.
  auto half_key = [&](int i) __attribute__((always_inline)) { return job.k_lo + 32 * i + 16 * lane; };
  auto fetch = [&](int i) __attribute__((always_inline)) {
    return job.table[min(half_key(i), job.k_hi - 1) / a.S];
  };
  int next_page = fetch(0);

  // The lane's row, the keys that it sees, and its query.
  const int r = job.row0 + 32 * wave + ql;
  const bool real = r < job.rows;
  const bool active = uniform(job.row0 + 32 * wave < job.rows) != 0;
  const int member = r / a.R, rr = r - member * a.R;
  const int h = rr / a.N, n = rr - h * a.N;
  const int b = job.b0 + member;
  int see = INT32_MAX;
  half8 qf[NQ];
  {
    const half_t* q = a.q + b * a.qs[0] + (int64_t)(job.kvh * a.group + h) * a.qs[1] + n * a.qs[2];
#pragma unroll
    for (int kk = 0; kk < NQ; ++kk) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (real && 16 * kk + 8 * g < a.d) v = *reinterpret_cast<const u32x4*>(q + 16 * kk + 8 * g);
      qf[kk] = __builtin_bit_cast(half8, v);
    }
    if (real) see = min(fitting(a, a.lengths[b]) - a.N + n + 1, job.k_hi);
  }
  // Units that end below this need no mask.
  int all_see = see;
#pragma unroll
  for (int i = 32; i > 0; i >>= 1) all_see = min(all_see, __shfl_xor(all_see, i, 64));
  all_see = uniform(min(all_see, job.k_hi));

  const int row_bytes = (int)a.ks[2] * 2;
  const char* const k_head = reinterpret_cast<const char*>(a.k + job.kvh * a.ks[1]);
  const char* const v_head = reinterpret_cast<const char*>(a.v + job.kvh * a.ks[1]);
  const int units = (job.k_hi - job.k_lo + T::KT - 1) / T::KT;

  // The wave's share of a unit: its 1 KiB pieces, all in half `e` of the unit.
  PrefixDma<T::PER_WAVE> dma;
  const int piece0 = T::INSTR >= kPrefixWaves ? wave * T::PER_WAVE : wave % T::INSTR;
  const int e = piece0 * 1024 / (D * 2) / 16;
#pragma unroll
  for (int i = 0; i < T::PER_WAVE; ++i) {
    const int byte = (piece0 + i) * 1024 + lane * 16;
    const int row = byte / (D * 2);
    const int c = swz_chunk<D>(row, (byte % (D * 2)) / 16);
    dma.voff[i] = 8 * c < a.d ? (uint32_t)((row & 15) * row_bytes + 16 * c) : kOutOfRange;
  }

  // Where the half units from unit iu & ~31 on lie, one a lane: the byte offset of the first of
  // their rows that exist, and the bytes from it to the end of the last.
  int bad_key = INT32_MAX;  // first key of the first page that does not exist
  int64_t off = 0;
  uint32_t rows_bytes = 0;
  int iu = 0;  // next unit to ask for
  const uint32_t lds0 = lds_addr(lds);
  auto issue = [&](int slot) __attribute__((always_inline)) {
    if ((iu & 31) == 0) {
      const int key = half_key(iu), skip = max(job.k_first - key, 0);
      const int there = min(job.k_hi - key, 16) - skip;
      const bool ok = next_page >= 0 && next_page < a.pages;
      if (there > 0 && !ok) bad_key = min(bad_key, key);
      off = 2 * (next_page * a.ks[0] + (key % a.S + skip) * a.ks[2]);
      rows_bytes = ok && there > 0 ? (uint32_t)((there - 1) * row_bytes + a.d * 2) : 0u;
      next_page = fetch(iu + 32);
    }
    const int at = 2 * (iu & 31) + e;
    const int skip = iu == 0 ? max(job.k_first - job.k_lo - 16 * e, 0) : 0;
    const uint64_t o = (uint32_t)__builtin_amdgcn_readlane((int)off, at) |
                       (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), at) << 32;
    const uint32_t n = __builtin_amdgcn_readlane(rows_bytes, at);
    issue_unit<T::TILE * 2>(dma, make_rsrc_words(k_head + o, n), make_rsrc_words(v_head + o, n),
                            (uint32_t)(skip * row_bytes),
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
  // A row whose sequence needs a page that does not exist.
  if (bad_key != INT32_MAX && real && a.lengths[b] > bad_key) lt = __builtin_nanf("");
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

// A wave's piece of a sequence's own keys [k_lo, k_hi), of which k_first is the first (k_lo is that
// rounded down to 16), against the 32 rows from row0 on that read head kvh, as in paged_fwd_kernel: K
// rows come in the layout of the MFMA operand, V rows go through a tile in LDS (`vt`) for the
// transposing reads, both asked for a unit ahead.
template <int D, class E>
__device__ __forceinline__ void own_piece(const PrefixArgs& a, int b, int kvh, int row0, int k_lo, int k_first,
                                          int k_hi, int len, float* slot, half_t* vt) {
  constexpr int KD = D / 32, DD = D / 16, RB = 2;
  constexpr int VI = 32 * D * 2 / 1024, VROWS = 512 / D;  // 1 KiB loads of a unit's V, rows of one
  const int lane = threadIdx.x & 63, c16 = lane & 15, G = lane >> 4;
  const int row_bytes = (int)a.ks[2] * 2;
  uint32_t k_off[KD], v_off[VI];
  int v_at[VI], t_off[DD];
#pragma unroll
  for (int kd = 0; kd < KD; ++kd) {
    const int col = 32 * kd + 8 * G;
    k_off[kd] = col < a.d ? (uint32_t)(c16 * row_bytes + col * 2) : kOutOfRange;
  }
#pragma unroll
  for (int i = 0; i < VI; ++i) {
    const int row = i * VROWS + lane / (D / 8), chunk = lane % (D / 8);
    v_off[i] = 8 * chunk < a.d ? (uint32_t)((row & 15) * row_bytes + chunk * 16) : kOutOfRange;
    v_at[i] = swz_offset<D>(row, chunk);
  }
#pragma unroll
  for (int dd = 0; dd < DD; ++dd) {
    const int row = 4 * G + (c16 >> 2), col = 16 * dd + 4 * (c16 & 3);
    t_off[dd] = row * D + 8 * swz_chunk<D>(row, col >> 3) + (col & 7);
  }

  const int units = (k_hi - k_lo + 31) / 32;
  const int* const table = a.table + b * a.table_stride;
  auto half_key = [&](int i) __attribute__((always_inline)) { return k_lo + 32 * i + 16 * lane; };
  auto fetch = [&](int i) __attribute__((always_inline)) {
    return table[min(half_key(i), k_hi - 1) / a.S];
  };
  int next_page = fetch(0);

  // The lane's rows. Each sees the keys below see[]; rows that do not exist score 0 everywhere.
  const int all_see = len - a.N + 1;
  int see[RB];
  half8 qf[RB][KD];
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = row0 + 16 * rb + c16, h = r / a.N, n = r - h * a.N;
    see[rb] = r < a.R ? min(all_see + n, k_hi) : INT32_MAX;
    const half_t* q = a.q + b * a.qs[0] + (int64_t)(kvh * a.group + h) * a.qs[1] + n * a.qs[2];
#pragma unroll
    for (int kd = 0; kd < KD; ++kd) {
      u32x4 v = {0u, 0u, 0u, 0u};
      const int col = 32 * kd + 8 * G;
      if (r < a.R && col < a.d) v = *reinterpret_cast<const u32x4*>(q + col);
      qf[rb][kd] = __builtin_bit_cast(half8, v);
    }
  }

  const char* const k_head = reinterpret_cast<const char*>(a.k + kvh * a.ks[1]);
  const char* const v_head = reinterpret_cast<const char*>(a.v + kvh * a.ks[1]);
  bool bad = false;
  int64_t off = 0;  // where the half units from i & ~31 on lie, one a lane, as in prefix_piece
  uint32_t bytes = 0;
  u32x4 kx[2][KD], vx[VI];
  uint64_t at[2];
  uint32_t n[2], back[2];
  auto turn_to = [&](int i) __attribute__((always_inline)) {
    if ((i & 31) == 0) {
      const int key = half_key(i), skip = max(k_first - key, 0);
      const int there = min(k_hi - key, 16) - skip;
      const bool ok = next_page >= 0 && next_page < a.pages;
      bad |= there > 0 && !ok;
      off = 2 * (next_page * a.ks[0] + (key % a.S + skip) * a.ks[2]);
      bytes = ok && there > 0 ? (uint32_t)((there - 1) * row_bytes + a.d * 2) : 0u;
      next_page = fetch(i + 32);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int l = 2 * (i & 31) + e;
      at[e] = (uint32_t)__builtin_amdgcn_readlane((int)off, l) |
              (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(off >> 32), l) << 32;
      n[e] = __builtin_amdgcn_readlane(bytes, l);
      back[e] = i == 0 ? (uint32_t)(max(k_first - k_lo - 16 * e, 0) * row_bytes) : 0u;
    }
  };
  auto load_k = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const rsrc_t r = make_rsrc(k_head + at[e], n[e]);
#pragma unroll
      for (int kd = 0; kd < KD; ++kd) kx[e][kd] = buf_load_b128(r, k_off[kd] - back[e]);
    }
  };
  auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < VI; ++j) {
      const int e = j * VROWS / 16;
      vx[j] = buf_load_b128(make_rsrc(v_head + at[e], n[e]), v_off[j] - back[e]);
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
  for (int i = 0; i < units; ++i) {
    const int ka = k_lo + 32 * i;
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
    for (int j = 0; j < VI; ++j) *reinterpret_cast<u32x4*>(vt + v_at[j]) = vx[j];
    load_v();
    half8 pa[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      if (ka + 32 > min(all_see, k_hi) || ka < k_first) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int key = ka + 16 * kb + 4 * G + j;
            if (key >= see[rb] || key < k_first) s[rb][kb][j] = -INFINITY;
          }
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
      float l_u = probs(m[rb]);
      const float held = kPrefixWide<E> ? l[rb] + l_u : l_u;
      if (__builtin_amdgcn_ballot_w64(!(held <= 0.5f * kPrefixSumLimit<E>)) != 0) {
        float mt = s[rb][0][0];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int j = 0; j < 4; ++j) mt = __builtin_fmaxf(mt, s[rb][kb][j]);
        float m_new = __builtin_fmaxf(m[rb], quarters_max(mt) * c - kPrefixShift<E>);
        if constexpr (kPrefixWide<E>)
          m_new = __builtin_fmaxf(m_new, m[rb] + log2_fast(quarters_max(l[rb])) - kPrefixShift<E>);
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

  bad = __builtin_amdgcn_ballot_w64(bad) != 0;
#pragma unroll
  for (int rb = 0; rb < RB; ++rb) {
    const int r = 16 * rb + c16;
    float lt = quarters_sum(l[rb]);
    if (bad) lt = __builtin_nanf("");
    if (row0 + r >= a.R) continue;
    const float inv = lt == 0.f ? 0.f : 1.0f / lt;
#pragma unroll
    for (int dd = 0; dd < DD; ++dd)
      *reinterpret_cast<float4v*>(slot + (int64_t)r * D + 16 * dd + 4 * G) = o[rb][dd] * inv;
    if (G == 0) slot[(int64_t)a.srows * D + r] = lt == 0.f ? -INFINITY : m[rb] + log2_fast(lt);
  }
}

template <int D, class E, bool WAVES>
__global__ __launch_bounds__(64 * kPrefixWaves, PrefixRing<D>::WGS) void prefix_fwd_kernel(PrefixArgs a) {
  __shared__ __attribute__((aligned(1024))) half_t lds[PrefixRing<D>::HALVES];
  static_assert(sizeof(lds) >= (96 + 2 * kPrefixKeptGroups + kPrefixKeptSeqs) * 4,
                "places are found in the ring's memory");
  PrefixPlace at;
  const PrefixLine line = prefix_find<WAVES>(a, reinterpret_cast<int*>(lds), &at);
  int left = line.left;
  if (left <= 0) return;
  const int HB = a.Hkv * a.blocks;
  if (WAVES && line.own) {
    half_t* const vt = lds + uniform(threadIdx.x >> 6) * (32 * D);
    while (true) {
      const int k0 = at.k_first & ~15, units = key_units(at.k_first, at.k_end);
      const int len = units + kOwnLead;
      const int u0 = max(at.unit - kOwnLead, 0);
      const int u1 = left < len - at.unit ? max(at.unit + left - kOwnLead, 0) : units;
      const int kvh = at.sub / a.blocks;
      if (u1 > u0)
        own_piece<D, E>(a, at.at, kvh, (at.sub - kvh * a.blocks) * kOwnTile, k0 + 32 * u0, max(at.k_first, k0 + 32 * u0),
                        min(at.k_end, k0 + 32 * u1), at.k_end,
                        own_slot(a, D, (int64_t)line.s + (int64_t)at.at * HB + at.sub), vt);
      left -= len - at.unit;
      if (left <= 0) return;
      at.unit = 0;
      if (++at.sub < HB) continue;
      at.sub = 0;
      if (!next_sequence(a, at)) return;
    }
  }
  while (true) {
    // The triple's part that is the work-group's.
    PrefixJob job;
    const int tiles = at.kind == 1 ? a.blocks : prefix_tiles(at.n, a.R);
    job.kvh = at.sub / tiles;
    job.row0 = (at.sub - job.kvh * tiles) * kPrefixTile;
    job.b0 = at.b0;
    job.rows = at.n * a.R;
    job.table = a.table + at.b0 * a.table_stride;
    job.slot_rows = at.kind == 1 ? a.srows : a.prows;
    const bool piece = at.kind == 2;
    const int k0 = at.k_first & ~15, units = key_units(at.k_first, at.k_end);
    const int len = units + kPrefixLead;
    const int u0 = piece ? 0 : max(at.unit - kPrefixLead, 0);
    const int u1 = piece || left >= len - at.unit ? units : max(at.unit + left - kPrefixLead, 0);
    if (u1 > u0) {
      job.k_lo = k0 + 32 * u0;
      job.k_first = max(at.k_first, job.k_lo);
      job.k_hi = min(at.k_end, k0 + 32 * u1);
      job.slot = piece          ? prefix_slot(a, D, line.s)
                 : at.kind == 0 ? prefix_slot(a, D, (int64_t)line.pieces + line.s + at.first + at.sub)
                                : own_slot(a, D, (int64_t)line.s + (int64_t)at.at * HB + at.sub);
      prefix_piece<D, E>(a, job, lds);
    }
    if (piece) return;
    left -= len - at.unit;
    if (left <= 0) return;
    // The next triple on the line, of this group or sequence or the next that has any there.
    at.unit = 0;
    if (++at.sub < tiles * a.Hkv) continue;
    at.sub = 0;
    if (at.kind == 0) {
      at.first += tiles * a.Hkv;
      int units = 0;
      while (units == 0 && ++at.at < a.G) {
        at.b0 = uniform(a.starts[at.at]);
        const int end = uniform(a.starts[at.at + 1]);
        at.n = end - at.b0;
        at.k_end = uniform(prefix_keys(a, at.at, at.b0, end));
        units = key_units(0, at.k_end);
        if (line.pieces > 0 && prefix_long(units, line.stretch)) units = 0;
      }
      if (units > 0) continue;
      if (WAVES) return;
      at.kind = at.n = 1;  // the line goes on with the sequences' own keys
      at.at = at.g = -1;
      at.g_end = line.bad || a.G == 0 ? a.B : uniform(a.starts[0]);
      at.k_first = 0;
    }
    if (!next_sequence(a, at)) return;
  }
}

// Joins the pieces of each row: those of its group's prefix, then those of its own keys. A lane
// holds four columns of a row, a wave 64 / (D / 4) rows, one after the other in the output; SPLIT of a
// block's waves take every SPLIT-th piece of the same rows and merge through LDS, in a fixed order.
// A piece weighs exp2 of its log-sum-exp against the others'.
template <int D, class E, int SPLIT>
__global__ __launch_bounds__(64 * (SPLIT < 4 ? 4 : SPLIT)) void prefix_join_kernel(PrefixArgs a) {
  constexpr int W = SPLIT < 4 ? 4 : SPLIT;  // waves
  constexpr int COLS = D / 4, RPP = 64 / COLS;
  constexpr int AHEAD = 4;
  __shared__ __attribute__((aligned(16))) float acc_s[SPLIT > 1 ? W : 1][64][4];
  __shared__ float m_s[W][64], l_s[W][64];
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int part = wave % SPLIT;
  const unsigned row = (blockIdx.x * (W / SPLIT) + wave / SPLIT) * RPP + lane / COLS;  // of [B, Hq, N]
  const int col = 4 * (lane % COLS);
  const unsigned seq_rows = a.Hkv * a.R;
  const bool real = row < a.B * seq_rows;
  const unsigned rr = real ? row : 0;
  const int b = rr / seq_rows, in_seq = rr - b * seq_rows;
  const int kvh = in_seq / a.R, r = in_seq - kvh * a.R;
  const int stretch = a.ws[0], own_stretch = a.ws[1], cut = a.ws[3];
  const bool bad = a.ws[2] != 0;
  const int len = a.lengths[b];
  const PrefixSeq q = prefix_seqs(a)[b];
  // (most batches have one group: it is asked for beside the sequence)
  PrefixGroup grp = {0, 0, 0, 1, 0, 0, 0, 0};
  if (a.G > 0) grp = prefix_groups(a)[0];
  if (q.group > 0) grp = prefix_groups(a)[q.group];
  if (q.group < 0) grp = {0, 0, 0, 1, 0, 0, 0, 0};

  // Pieces of a triple on the line whose part of it begins at `base`: the first one's stretch, and
  // how many there are.
  auto range = [](int64_t base, int units, int lead, int stretch, int* n) __attribute__((always_inline)) {
    const int64_t at = base + lead;
    const int s0 = (int)(at / stretch);
    *n = units > 0 ? (int)((at + units - 1) / stretch) - s0 + 1 : 0;
    return s0;
  };
  const int64_t gr = (int64_t)q.member * a.R + r;
  const int tile = (int)(gr / kPrefixTile), psub = kvh * grp.tiles + tile;
  int np, no, step = 1;
  int64_t pslot;
  if (grp.cuts > 0) {
    np = grp.cuts;
    step = grp.tiles;
    pslot = (int64_t)grp.base + (int64_t)kvh * grp.cuts * grp.tiles + tile;
  } else {
    pslot = range(grp.base + (int64_t)psub * on_line(grp.units, kPrefixLead), grp.units, kPrefixLead,
                  stretch, &np);
    pslot += (int64_t)cut + grp.first + psub;
  }
  const bool waves = a.R <= kOwnRows;
  const int own_tile = waves ? kOwnTile : kPrefixTile, lead = waves ? kOwnLead : kPrefixLead;
  const int osub = kvh * a.blocks + r / own_tile;
  int64_t oslot = range(q.own_base + (int64_t)osub * on_line(q.own_units, lead), q.own_units, lead,
                        own_stretch, &no);
  oslot += (int64_t)b * a.Hkv * a.blocks + osub;
  const int count = real ? np + no : 0;
  // The weight of the largest piece: those of a row sum to 1/2 at most, so that sums of values near
  // 2^128 stay in float32. (Up to 1024 pieces the weight is larger, which leaves small values more bits.)
  static_assert(kPrefixMostPieces <= 4096, "weights of 2^-13");
  const float weight = count <= 1024 ? 0x1p-11f : 0x1p-13f;
  struct Piece {
    float lse;
    float4v o;
  };
  auto load = [&](int i) __attribute__((always_inline)) {
    Piece p = {-INFINITY, {0.f, 0.f, 0.f, 0.f}};
    if (i < count) {
      const bool pre = i < np;
      const float* slot = pre ? prefix_slot(a, D, pslot + (int64_t)i * step)
                              : own_slot(a, D, oslot + (i - np));
      const int at = pre ? (int)(gr % kPrefixTile) : r % own_tile;
      p.lse = slot[(int64_t)(pre ? a.prows : a.srows) * D + at];
      p.o = *reinterpret_cast<const float4v*>(slot + (int64_t)at * D + col);
    }
    return p;
  };
  float m = -INFINITY, l = 0.f;
  float4v acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = part; i0 < count; i0 += SPLIT * AHEAD) {
    Piece p[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) p[i] = load(i0 + SPLIT * i);
    float mx = m;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) mx = __builtin_fmaxf(mx, p[i].lse);
    const float ref = exp_reference(mx);
    const float keep = m == -INFINITY ? 0.f : exp2_fast(m - ref);
    l *= keep;
    acc *= keep;
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const float f = p[i].lse == -INFINITY ? 0.f : exp2_fast(p[i].lse - ref) * weight;
      l += f;
      acc += p[i].o * f;
    }
    m = mx;
  }
  float lt = l;
  float4v v = acc;
  if constexpr (SPLIT > 1) {
    *reinterpret_cast<float4v*>(acc_s[wave][lane]) = acc;
    m_s[wave][lane] = m;
    l_s[wave][lane] = l;
    __syncthreads();
    if (part != 0) return;
    float mx = -INFINITY;
#pragma unroll
    for (int i = 0; i < SPLIT; ++i) mx = __builtin_fmaxf(mx, m_s[wave + i][lane]);
    lt = 0.f;
    v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < SPLIT; ++i) {
      const float f = m_s[wave + i][lane] == -INFINITY ? 0.f : exp2_fast(m_s[wave + i][lane] - mx);
      lt += f * l_s[wave + i][lane];
      v += *reinterpret_cast<const float4v*>(acc_s[wave + i][lane]) * f;
    }
  }
  if (!real || col >= a.d) return;
  v *= lt == 0.f ? 0.f : 1.0f / lt;  // a row that saw no key is 0
  if (bad || len < 0 || len > a.M * a.S) {
    const float nan = __builtin_nanf("");
    v = {nan, nan, nan, nan};
  }
  *reinterpret_cast<u32x2*>(a.o + (int64_t)row * a.d + col) = pack4<E>(v[0], v[1], v[2], v[3]);
}

static int prefix_width(int64_t D) { return D <= 32 ? 32 : D <= 64 ? 64 : 128; }

PrefixSizes prefix_sizes(int64_t B, int64_t G, int64_t Hkv, int64_t R, int64_t D, int64_t keys) {
  PrefixSizes z;
  const int64_t own_tile = R <= kOwnRows ? kOwnTile : kPrefixTile;
  z.blocks = (int)((R + own_tile - 1) / own_tile);
  z.prows = (int)std::min<int64_t>(kPrefixTile, B * R);
  z.srows = (int)std::min(own_tile, R);
  // Groups of two sequences or more have prefixes, in at most so many tiles.
  const int64_t groups = std::min(G, B / 2), own = B * Hkv * z.blocks;
  const int64_t triples = groups > 0 ? Hkv * (B * R / kPrefixTile + groups) : 0;
  const double each = (double)((keys + 31) / 32 + 1 + kPrefixLead);
  z.units = each * ((double)triples + (double)own);
  const int64_t most = prefix_width(D) == 128 ? PrefixRing<128>::WGS * 256 : kPrefixMostGrid;
  // Work-groups that the chip holds at once, at most one for each four units that the tables could
  // hold; as many on each XCD.
  z.grid = (int)std::min((double)most, std::ceil(z.units / kPrefixStretch));
  z.grid = std::max((z.grid + 7) / 8 * 8, 16);
  // Where all rows fit one tile memory bounds a prefix, and 256 pieces keep it busy. (4 sequences over
  // 65536 and 262144 keys, Hq32 Hkv8 D128: 58 and 197 us; 128 pieces 77 and 263; 512, with twice the
  // partials, 56 and 198.)
  z.most_pieces = B * R <= kPrefixTile ? std::min(z.grid, 256) : z.grid;
  z.pslots = triples > 0 ? z.grid + triples : 0;
  z.head_bytes = (64 + B * (int64_t)sizeof(PrefixSeq) + G * (int64_t)sizeof(PrefixGroup) + 63) / 64 * 64;
  const int64_t rows = z.pslots * z.prows + (kPrefixWaves * z.grid + own) * z.srows;
  z.bytes = z.head_bytes + rows * (prefix_width(D) + 4) * 4;
  return z;
}

// Few rows have many pieces and are joined by more waves each; with many rows the waves are enough.
// (Whole calls over 4096 shared keys, Hq32 Hkv8 D128: 128 waves of rows 20.0 us with sixteen for each and
// 21.7 with four; 256 23.1 and 24.6; 384 27.9 and 26.5.)
template <int D, class E, int SPLIT>
hipError_t prefix_join_start(const PrefixArgs& a, hipStream_t stream) {
  constexpr int W = SPLIT < 4 ? 4 : SPLIT;
  constexpr int RPB = 64 / (D / 4) * (W / SPLIT);
  const int64_t rows = (int64_t)a.B * a.Hkv * a.R;
  hipLaunchKernelGGL((prefix_join_kernel<D, E, SPLIT>), dim3((unsigned)((rows + RPB - 1) / RPB)),
                     dim3(64 * W), 0, stream, a);
  return hipGetLastError();
}

template <int D, class E>
hipError_t prefix_start(const PrefixArgs& a, hipStream_t stream) {
  const dim3 grid((unsigned)a.grid), block(64 * kPrefixWaves);
  if (a.R <= kOwnRows) hipLaunchKernelGGL((prefix_fwd_kernel<D, E, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((prefix_fwd_kernel<D, E, false>), grid, block, 0, stream, a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t waves = (int64_t)a.B * a.Hkv * a.R / (64 / (D / 4));
  return waves >= 256 ? prefix_join_start<D, E, 4>(a, stream)
                      : prefix_join_start<D, E, 16>(a, stream);
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
