// Attention of one new token of every sequence over a paged cache, for one dimension (PITCH_DIM = 64 or 128) and one width of
// the key codes (PITCH_KB = 2, 3, 4; 0 for the widths 5 to 8).
//
//   out = softmax(z) V,  z_t = cap tanh(scale q . k_t / cap) + slope (t - (L - 1)),  t in [L - window, L)
//
// No token is decoded: k_t = s H c(code_t) n_t / sqrt(d), so a query is rotated once (H s q), scores are its products with the
// table values of the codes times the token's scale, and the weighted table values are rotated back once.
//
// Work split. The sequences' tiles of 64 tokens, sequence by sequence and KV head by KV head, form one line that is cut into
// equal runs, one per workgroup (one per compute unit), and each run into equal runs of its waves: a batch of any lengths loads
// every wave alike, and only the host-known number of workgroups is launched. What is cut equally is tiles and one more per pair of
// sequence and KV head, whose queries and output cost about a tile (200 sequences of 1 to 500 tokens, 12 heads, with a join: 34 us
// then, 31 now, by tiles alone 41). A wave goes through its run by itself (scores, online softmax, weighted values; no barrier), pair by pair. A pair that
// lies in one wave is written by it; the parts of one that several waves of a workgroup share are merged at the end through LDS,
// and paged_join merges what crosses workgroups through the workspace, in an order fixed by the lengths alone. Where no pair can
// have more than a tile per wave, workgroups take whole pairs and there is no join.
//
// What bounds it: HBM in between, and latencies at either end, which are half of the time even of the longest calls. 32 sequences of
// up to 8,000 tokens, d = 128 bf16, 4 queries per KV head (138 MB, 45 us with the join), by stamps of the waves: lengths known after
// 0.7 us, page looked up 1.7, tables written 2.6, first loads asked for 4.8, queries rotated 6.2, first tile done 9.6; then 120 MB
// until the median wave ends at 30 us (5.8 TB/s), the first at 25 and the last at 36; merged at 39; the join 5.2. 131,072 tokens of
// one sequence (126 MB) 47 us, 777 tokens 14.7 us. Heads of 64: eight bits and float16 (two parts, a window of 1,000 tokens, 64
// sequences) 31 us and the short sequences above 28, bound by the arithmetic of the lookups. Writing the tables takes 0.3 to 1 us of
// a wave; without it calls were 0 to 2.3 us shorter. Two tiles in registers, 12 or 16 waves (spills), priorities for the waves
// behind, non-temporal reads and a touch of the second tile's lines at the start were no faster.
//
// Contractions on the 16-bit matrix cores (v_mfma_f32_16x16x32_f16), 16 rows of one operand for a KV head's query heads. A code
// pair is looked up in LDS as two float16 values, which are operand words as they are: for the scores two neighbouring
// coordinates of a token on the contraction axis; for the values a pair's two coordinates of one token side by side on it, with
// the weight at the one or the other: rows 0 - 7 weigh the first coordinate, rows 8 - 15 the second. What rows remain hold the
// operands' rest after rounding to float16: up to four heads, queries and weights both in two parts (22 bits); five to eight
// heads, the queries in two and the weights in one (11 bits), or with float16 queries, whose outputs resolve that, in two by a
// second instruction. TurboQuant's table values are stored times a factor at which they
// nearly are float16 values (gen_tables.py: 4e-5 of a codebook's size for four bits, instead of 2e-4). With float16 queries the
// keys' and the values' table values have two parts as well, whose products are added by a second instruction: a rounding of 2e-4
// in the keys moves a score of size 5 by 1e-3, several times what float16 outputs resolve (bfloat16: a quarter), and one in
// the values is as large as the output's own. Errors of outputs relative to their norm, 4 sequences of up to 900 tokens: float16
// 2.0e-4, the rounding of the exact result (values in one part: up to 1.25 times that for eight bits, 1.6 for PolarQuant); bfloat16,
// one part each, 1.6e-3, at most 6 % above the rounding (PolarQuant of 6 and 8 bits, whose pairs are a product of two rounded values, else 0.8 %).
// The log-sum-exps are off by 3e-6 with float16 queries, with bfloat16 by up to 4e-4 (TurboQuant) and 2e-3 (PolarQuant).
// The second parts of the values cost 5 % (64 sequences, window of 1,000, 8 heads of 64 of eight bits: 31.1 us, 29.6 without).
//
// The table's entry of a pair (four codes for two bits) is 256 bytes long, copies for the keys in its first half and for the
// values in its second (float16 queries: a table each): lanes read copies in different banks, and where the index is a byte of
// the row, one v_perm makes the address.
#include <atomic>

#include "pitch_attn_shared.h"
#include "pitch_paged.h"

#ifndef PITCH_DIM
#error "compile with -DPITCH_DIM=<dim>"
#endif
#ifndef PITCH_KB
#error "compile with -DPITCH_KB=<key bits>"
#endif

namespace pitch {
namespace {

constexpr int D = PITCH_DIM;
constexpr int NC = D / 32;       // groups of 16 pairs: accumulators of a wave
constexpr int KS = D / 32;       // score instructions per 16 tokens
constexpr int kPRow = 68;        // dwords of a row of staged weights
constexpr float kLoScale = 2048.f;
constexpr float kTop = 32768.f;  // largest weight in an operand

typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint64_t u64_any __attribute__((aligned(1)));
// (an address made of integers is a flat one, which counts as an LDS access too: the table reads would wait for it)
typedef __attribute__((address_space(1))) uint8_t global_u8;
template <typename V>
using global = __attribute__((address_space(1))) V;
typedef __attribute__((address_space(3))) const uint32_t lds_cu32;
typedef __attribute__((address_space(3))) const u2 lds_cu2;
typedef __attribute__((address_space(3))) const w4 lds_cw4;

constexpr int W = 8;   // waves of a workgroup: two per SIMD (256 registers each)
static_assert(W <= (int)kPagedAttnWaves, "waves of a workgroup");

__device__ __forceinline__ uint32_t f16_pair(float a, float b) { return narrow2<1>(a, b); }

// ---------------------------------------------------------------------------------------------------- tables
// Bytes of LDS of a table: 256 bytes per entry.
constexpr uint32_t table_bytes(int b) { return b == 3 ? 64u * 256u : 65536u; }
// With two parts the keys' and the values' tables follow each other, else they share their entries. A table of 64 KB begins at a multiple
// of its size: its lane bytes hold the base in their third byte, which v_perm passes on.
constexpr uint32_t key_base(int kb, int vb, bool two) { return two && kb == 3 && vb != 3 ? 65536u : 0u; }
constexpr uint32_t value_base(int kb, int vb, bool two) { return !two ? 128u : kb != 3 ? 65536u : vb != 3 ? 0u : 16384u; }
constexpr uint32_t tables_bytes(int kb, int vb, bool two) {
  return two ? table_bytes(kb) + table_bytes(vb) : table_bytes(kb) > table_bytes(vb) ? table_bytes(kb) : table_bytes(vb);
}

// What float16 rounding leaves of a pair of values: (the values as float16, the rests as float16).
__device__ __forceinline__ u2 split_pair(float x, float y) {
  const uint32_t hi = f16_pair(x, y);
  float a, b;
  widen2<1>(hi, a, b);
  return u2{hi, f16_pair(x - a, y - b)};
}

// A table for codes of B bits (0: p.bits), of values in one part or in two (TWO), in two steps: a thread's
// source values are loaded when the kernel begins, and written to LDS when other loads are on their way.
//   B = 3, 4, two codes: 32 copies of the pair, or of its two parts
//   B = 2, four codes: 16 copies of two pairs, or of their two parts
//   B = 0, one code: 16 copies of (value at an even coordinate, 1), then of (1, value at an odd one), PolarQuant (radius, radius)
//     and (cosine, sine): a pair's values are the products. TWO: 32 copies of the value's two parts; PolarQuant 16 copies of the
//     radius, then of (cosine, sine), as float32.
template <int B, bool TWO>
struct Table {
  static constexpr int kEntries = B == 2 || B == 0 ? 256 : 1 << (2 * B);
  static constexpr int R = (kEntries * 4 + 64 * W - 1) / (64 * W);   // quarters of entries per thread
  uint32_t x[R][B == 0 ? 3 : B == 2 ? 4 : 2];

  __device__ __forceinline__ void load(const PagedPool& p, int tid) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t e = min((uint32_t)(tid + r * 64 * W) >> 2, (uint32_t)kEntries - 1u);
      if constexpr (B == 0) {
        const uint32_t c = min(e, (1u << p.bits) - 1u);
        if (p.polar) {
          const int off = pitch_polar_offset(p.bits) + c;
          x[r][0] = __float_as_uint(pitch_polar_radius_tab[off]);
          x[r][1] = __float_as_uint(pitch_polar_cos_tab[off]);
          x[r][2] = __float_as_uint(pitch_polar_sin_tab[off]);
        } else {
          x[r][0] = __float_as_uint(pitch_codebook_tab[pitch_codebook_offset(ilog2(D), p.bits) + c]);
          x[r][1] = x[r][2] = 0u;
        }
      } else {
        const u2* const tab = (const u2*)pitch_pair16_tab + pitch_pair16_offset(ilog2(D), p.polar != 0, B);
        const u2 v = tab[B == 2 ? e & 15u : e];
        x[r][0] = v.x;
        x[r][1] = v.y;
        if constexpr (B == 2) {
          const u2 w = tab[e >> 4];
          x[r][2] = w.x;
          x[r][3] = w.y;
        }
      }
    }
  }
  __device__ __forceinline__ void write(uint32_t* tab, const PagedPool& p, float factor, int tid) const {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = tid + r * 64 * W;
      if (i >= kEntries * 4) break;
      const uint32_t e = (uint32_t)i >> 2;
      w4* const at = (w4*)(tab + 64 * e) + (TWO ? 4 : 2) * (i & 3);
      w4* const one = (w4*)(tab + 64 * e) + (i & 3);
      if constexpr (B == 2) {
        const w4 w = TWO ? w4{x[r][0], x[r][2], x[r][1], x[r][3]} : w4{x[r][0], x[r][2], x[r][0], x[r][2]};
#pragma unroll
        for (int k = 0; k < (TWO ? 4 : 2); ++k) at[k] = w;
      } else if constexpr (B != 0) {
        const w4 w = TWO ? w4{x[r][0], x[r][1], x[r][0], x[r][1]} : w4{x[r][0], x[r][0], x[r][0], x[r][0]};
#pragma unroll
        for (int k = 0; k < (TWO ? 4 : 2); ++k) at[k] = w;
      } else {
        const float v = __uint_as_float(x[r][0]) * factor, c = __uint_as_float(x[r][1]), n = __uint_as_float(x[r][2]);
        if constexpr (TWO) {
          if (p.polar) {
            const uint32_t u = __float_as_uint(v);
            one[0] = w4{u, u, u, u};
            one[4] = one[8] = w4{x[r][1], x[r][2], x[r][1], x[r][2]};
          } else {
            const u2 s = split_pair(v, 0.f);
            const uint32_t u = (s.x & 0xFFFFu) | s.y << 16;
            one[0] = one[4] = w4{u, u, u, u};
          }
        } else {
          const uint32_t even = f16_pair(v, p.polar ? v : 1.f), odd = p.polar ? f16_pair(c, n) : f16_pair(1.f, v);
          one[0] = w4{even, even, even, even};
          one[4] = w4{odd, odd, odd, odd};
        }
      }
    }
  }
};

// A lane's byte of an entry.
template <int B, bool TWO>
__device__ __forceinline__ uint32_t lane_byte(int lane) {
  if constexpr (B == 2) return (uint32_t)(lane & 15) * (TWO ? 16u : 8u);
  if constexpr (B == 0) return TWO ? (uint32_t)(lane & 31) * 4u : (uint32_t)(lane & 15) * 4u;
  return (uint32_t)(lane & 31) * (TWO ? 8u : 4u);
}

__device__ __forceinline__ uint32_t product(uint32_t a, uint32_t b) {
  return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, a) * __builtin_bit_cast(f16x2, b));
}

// Four codes of 5 to 7 bits as bytes.
__device__ __forceinline__ uint32_t spread(uint32_t x, uint32_t bits) {
  const uint32_t two = (1u << 2 * bits) - 1u, one = ((1u << bits) - 1u) * 0x10001u;
  const uint32_t t = (x & two) | (x >> 2 * bits & two) << 16;
  return (t & one) | (t & one << bits) << (8u - bits);
}

// The COUNT pairs of 2 COUNT codes: the N words w hold the codes from bit `at` on (constants); the widths above four bits have a
// byte per code. hi: the pairs' float16 values, lo (TWO): their rests.
template <int B, bool TWO, int COUNT, int N>
__device__ __forceinline__ void look_pairs(const uint32_t (&w)[N], int at, uint32_t lb, bool polar, uint32_t (&hi)[COUNT],
                                           uint32_t (&lo)[COUNT]) {
  constexpr uint32_t kSel = 0x0C060004u;   // bytes: the lane's, a byte of the codes, the table's base above 64 KB, 0
  if constexpr (B == 2) {
#pragma unroll
    for (int i = 0; i < COUNT / 2; ++i) {
      const int p = at + 8 * i;
      const uint32_t a = __builtin_amdgcn_perm(lb, w[p >> 5], kSel | (uint32_t)((p & 31) >> 3) << 8);
      if constexpr (TWO) {
        const w4 v = *(lds_cw4*)(uintptr_t)a;
        hi[2 * i] = v.x; hi[2 * i + 1] = v.y; lo[2 * i] = v.z; lo[2 * i + 1] = v.w;
      } else {
        const u2 v = *(lds_cu2*)(uintptr_t)a;
        hi[2 * i] = v.x; hi[2 * i + 1] = v.y;
      }
    }
  } else if constexpr (B != 0) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const int p = at + 2 * B * i;
      uint32_t a;
      if constexpr (B == 4) a = __builtin_amdgcn_perm(lb, w[p >> 5], kSel | (uint32_t)((p & 31) >> 3) << 8);
      else a = and_or(bits_at(w, p, 6, 8), 0x3F00u, lb);
      if constexpr (TWO) {
        const u2 v = *(lds_cu2*)(uintptr_t)a;
        hi[i] = v.x; lo[i] = v.y;
      } else {
        hi[i] = *(lds_cu32*)(uintptr_t)a;
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < COUNT; ++i) {
      const int p = at + 16 * i;
      const uint32_t a0 = __builtin_amdgcn_perm(lb, w[p >> 5], kSel | (uint32_t)((p & 31) >> 3) << 8);
      const uint32_t a1 = __builtin_amdgcn_perm(lb, w[p >> 5], kSel | (uint32_t)((p & 31) / 8 + 1) << 8);
      if constexpr (!TWO) {
        hi[i] = product(*(lds_cu32*)(uintptr_t)a0, *(lds_cu32*)(uintptr_t)(a1 + 64u));
      } else if (polar) {   // the copies' bytes: 16 of four, then 16 of eight
        const uint32_t c = lb & 63u;
        const float r = __uint_as_float(*(lds_cu32*)(uintptr_t)((a0 & ~127u) | c));
        const u2 v = *(lds_cu2*)(uintptr_t)((a1 & ~127u) + 64u + 2u * c);
        const u2 t = split_pair(r * __uint_as_float(v.x), r * __uint_as_float(v.y));
        hi[i] = t.x; lo[i] = t.y;
      } else {
        const uint32_t u = *(lds_cu32*)(uintptr_t)a0, v = *(lds_cu32*)(uintptr_t)a1;
        hi[i] = __builtin_amdgcn_perm(v, u, 0x05040100u);
        lo[i] = __builtin_amdgcn_perm(v, u, 0x07060302u);
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------- the line of tiles
struct Span {            // what a sequence's new token sees
  uint32_t begin, end;   // tokens
  uint32_t base, tiles;  // the tiles' first token (a multiple of 16), tiles of 64 tokens
};
// len: cached tokens, cut to the table.
__device__ __forceinline__ Span span_of(const PagedAttnArgs& a, uint32_t len) {
  Span s;
  s.end = len;
  s.begin = a.window && s.end > a.window ? s.end - a.window : 0u;
  s.base = s.begin & ~15u;
  s.tiles = s.end > s.base ? (s.end - s.base + 63u) >> 6 : 0u;
  return s;
}
__device__ __forceinline__ uint32_t cut_length(const PagedAttnArgs& a, int32_t len) { return len < 0 ? 0u : min((uint32_t)len, a.most_tokens); }
__device__ __forceinline__ uint32_t length_of(const PagedAttnArgs& a, uint32_t b) { return cut_length(a, a.lengths[b]); }

// Sums over the lanes up to and with this one.
__device__ __forceinline__ uint32_t wave_scan(uint32_t x) {
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x111, 0xF, 0xF, false);   // row_shr 1, 2, 4, 8
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x112, 0xF, 0xF, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x114, 0xF, 0xF, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x118, 0xF, 0xF, false);
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x142, 0xA, 0xF, false);   // row_bcast 15, 31
  x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x143, 0xC, 0xF, false);
  return x;
}

// The sequences along the line, in the lanes of a wave (no barrier: every wave looks the lengths up by itself). Up to 64 sequences
// have a lane each; of more, a lane sums `per` sequences, and the group that a place lies in is looked up one by one. Places on the
// line are counted twice: in tiles, and in units, of which a pair has one more than tiles, in front of them: its queries, its
// output. Runs are cut in units. The line's units, times KV heads, are below 2^31 (checked by the caller).
struct Place {
  uint32_t lane, kv, unit, tile, x;   // of the window; KV head; unit and tile of the pair; tiles of the line before it
};
struct Line {
  uint32_t per, tsums, usums, tiles, units;   // sequences of a lane; tiles and units (of one KV head) before this lane's, and of all
  uint32_t first, count, len, own, tbefore, ubefore;   // the window: lane i has sequence first + i's length, tiles, and those before it
  uint32_t begin, end;                        // its units

  // raw: lengths[lane], of the last sequence for lanes behind it.
  __device__ __forceinline__ void load(const PagedAttnArgs& a, int32_t raw, int lane) {
    const uint32_t n = a.sequences;
    per = (n + 63u) >> 6;
    uint32_t t = 0, u = 0;
    first = begin = end = 0;
    count = n;
    if (per == 1) {
      len = (uint32_t)lane < n ? cut_length(a, raw) : 0u;
      own = t = span_of(a, len).tiles;
      u = t + (t != 0);
    } else {
      const uint32_t at = lane * per;
#pragma unroll 4
      for (uint32_t i = 0; i < per; ++i) {
        const uint32_t l = length_of(a, min(at + i, n - 1)), x = at + i < n ? span_of(a, l).tiles : 0u;
        t += x;
        u += x + (x != 0);
      }
    }
    const uint32_t ti = wave_scan(t), ui = wave_scan(u);
    tbefore = tsums = ti - t;
    ubefore = usums = ui - u;
    tiles = __builtin_amdgcn_readlane(ti, 63);
    units = __builtin_amdgcn_readlane(ui, 63);
    if (per == 1) end = units;
  }
  // The group of sequences of lane `at` as the window.
  __device__ __forceinline__ void window(const PagedAttnArgs& a, uint32_t at, int lane) {
    first = at * per;
    count = min(per, a.sequences - first);
    len = (uint32_t)lane < count ? length_of(a, first + lane) : 0u;
    own = span_of(a, len).tiles;
    const uint32_t u = own + (own != 0), ti = wave_scan(own), ui = wave_scan(u);
    begin = __builtin_amdgcn_readlane(usums, at);
    tbefore = __builtin_amdgcn_readlane(tsums, at) + ti - own;
    ubefore = begin + ui - u;
    end = begin + __builtin_amdgcn_readlane(ui, 63);
  }
  // Where unit u of the line, below all of them, lies. (The last lane with no more units before it: empty ones are passed over.)
  __device__ __forceinline__ Place find(const PagedAttnArgs& a, uint32_t u, int lane) {
    const uint32_t heads = a.layout.kv_heads;
    if (u < begin * heads || u >= end * heads) window(a, (uint32_t)__builtin_popcountll(__ballot(usums * heads <= u)) - 1u, lane);
    Place p;
    p.lane = (uint32_t)__builtin_popcountll(__ballot((uint32_t)lane < count && ubefore * heads <= u)) - 1u;
    const uint32_t t = __builtin_amdgcn_readlane(own, p.lane), into = u - (uint32_t)__builtin_amdgcn_readlane(ubefore, p.lane) * heads;
    p.kv = into / (t + 1);
    const uint32_t r = into - p.kv * (t + 1);
    p.unit = r;
    p.tile = r ? r - 1 : 0u;
    p.x = (uint32_t)__builtin_amdgcn_readlane(tbefore, p.lane) * heads + p.kv * t + p.tile;
    return p;
  }
  // The first tile of the pair behind p's; there is one.
  __device__ __forceinline__ void next(const PagedAttnArgs& a, Place& p, int lane) {
    p.tile = 0;
    if (++p.kv < a.layout.kv_heads) return;
    p.kv = 0;
    for (;;) {
      const uint64_t more = __ballot((uint32_t)lane > p.lane && (uint32_t)lane < count && own != 0);
      if (more) {
        p.lane = (uint32_t)__builtin_ctzll(more);
        return;
      }
      window(a, first / per + 1, lane);
      if (__builtin_amdgcn_readlane(own, 0)) {
        p.lane = 0;
        return;
      }
      p.lane = 0;
    }
  }
};

// x / d for x < 2^31, with r = floor((2^32 - 1) / d): one too small at most before the correction.
__device__ __forceinline__ uint32_t quotient(uint32_t x, uint32_t d, uint32_t r) {
  const uint32_t q = __umulhi(x, r);
  return x - q * d >= d ? q + 1u : q;
}
// How the line of n units is cut: workgroup b begins at ceil(b n / groups), so that a workgroup has one unit more than another at
// most, and the one at the front of a pair that fills several has it; up to `groups` units, the first workgroups have one each.
struct Cut {
  uint32_t n, base, rest;
  __device__ __forceinline__ Cut(uint32_t units, const PagedAttnArgs& a) : n(units) {
    base = quotient(n, a.groups, a.groups_r);
    rest = n - base * a.groups;
  }
  __device__ __forceinline__ uint32_t begin(uint32_t b, const PagedAttnArgs& a) const {
    return base ? b * base + quotient(b * rest + a.groups - 1, a.groups, a.groups_r) : min(b, n);
  }
  __device__ __forceinline__ uint32_t group_of(uint32_t u, const PagedAttnArgs& a) const {
    if (!base) return u;
    uint32_t b = min((uint32_t)((float)u * (float)a.groups / (float)n), a.groups - 1);   // off by one at most
    if (begin(b, a) > u) --b;
    return begin(b + 1, a) <= u ? b + 1 : b;
  }
};
// Unit of a workgroup's run of n units at which wave w begins (no empty wave lies between others).
__device__ __forceinline__ uint32_t wave_begin(uint32_t n, uint32_t w) { return n < W ? min(w, n) : w * (n / W) + (w * (n % W) + W - 1) / W; }

// The workspace: four words per workgroup, then slots of partial results (maxima and sums of eight heads, and the accumulators as
// the lanes hold them): of each workgroup one of the pair that comes from the workgroups before and ends in it, one of the pair
// that goes on behind it; then one per wave, of the pair that ends inside its run. The four words: the last workgroup of the pair
// that begins in this one and goes on behind it, plus one (0: there is none), its sequence and its KV head.
constexpr uint32_t left_slot(uint32_t group) { return 2 * group; }
constexpr uint32_t right_slot(uint32_t group) { return 2 * group + 1; }
__device__ __forceinline__ uint32_t wave_slot(uint32_t groups, uint32_t group, uint32_t wave) { return 2 * groups + group * W + wave; }
constexpr uint32_t slot_floats(int nh) { return 16 + NC * 4 * (nh == 4 ? 32 : 64); }

// ---------------------------------------------------------------------------------------------------- output
// acc: a lane (n, g) has coordinates 2 (NC n + c) + (g >> 1) of head v (NH = 4) or v + 4 (g & 1); the transform back runs over its
// registers and across lanes. A sum of weights of zero (all that was visible had scores of minus infinity) gives zeros; one that is
// NaN (a query, a scale or a score of plus infinity that is no number) gives NaN.
template <int NH, int IO>
__device__ __forceinline__ void write_output(const PagedAttnArgs& a, uint32_t b, uint32_t kv, v4f (&acc)[NC], const float (&m)[NH],
                                             const float (&l)[NH], int lane) {
  const int n = lane & 15, g = lane >> 4;
  const bool odd = g & 1;
  const uint32_t upper = odd ? ~0u : 0u;   // this lane has heads 4 - 7 of eight
#pragma unroll
  for (int v = 0; v < 4; ++v) {
    const float total = NH == 8 ? pick(upper, l[v], l[NH - 4 + v]) : l[v];
    const float f = total != 0.f ? a.oscale / total : 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[c][v]), __float_as_uint(acc[c][v]), false, false);
      const float x = __uint_as_float(r[0]), y = __uint_as_float(r[1]);
      acc[c][v] = total != 0.f ? (g >= 2 ? x - y : x + y) * f : 0.f;
    }
  }
#pragma unroll
  for (int s = 1; s < NC; s *= 2)
#pragma unroll
    for (int c = 0; c < NC; ++c)
      if (!(c & s)) {
        const v4f x = acc[c], y = acc[c | s];
        acc[c] = x + y;
        acc[c | s] = x - y;
      }
  static_for<0, 4>([&](auto bit_c) {
    constexpr int lm = 1 << decltype(bit_c)::value;
    const float sg = (n & lm) ? -1.f : 1.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int v = 0; v < 4; ++v) acc[c][v] = __builtin_fmaf(acc[c][v], sg, xchg<lm>(acc[c][v]));
  });
  // pairs of coordinates: lanes g < 2 take heads 0 and 1 (of their four), the others 2 and 3
  const uint32_t signs = a.v.signs[(2 * NC * n) >> 5] >> ((2 * NC * n) & 31);
#pragma unroll
  for (int v = 0; v < 2; ++v) {
    uint32_t word[NC];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(acc[c][v]), __float_as_uint(acc[c][v + 2]), false, false);
      word[c] = narrow2<IO>(__uint_as_float(r[0] ^ (signs >> (2 * c) & 1u) << 31), __uint_as_float(r[1] ^ (signs >> (2 * c + 1) & 1u) << 31));
    }
    const uint32_t h = (g >= 2 ? v + 2 : v) + (NH == 8 && odd ? 4 : 0);
    if (h < a.nq && (NH == 8 || !odd)) {
      uint32_t* dst = (uint32_t*)((uint16_t*)a.out.data + b * a.out.token_stride + (kv * a.nq + h) * a.out.head_stride + 2 * NC * n);
      store_words<NC>(dst, word);
    }
  }
  if (a.lse && lane == 0) {
#pragma unroll
    for (int h = 0; h < NH; ++h)
      if (h < (int)a.nq)
        a.lse[((uint64_t)b * a.layout.kv_heads + kv) * a.nq + h] = l[h] != 0.f ? (m[h] + log2f(l[h])) * kLn2 : -__builtin_inff();
  }
}

// The outputs of an empty sequence.
__device__ __forceinline__ void write_zeros(const PagedAttnArgs& a, uint32_t b, int lane) {
  const uint32_t heads = a.layout.kv_heads * a.nq;
  for (uint32_t h = 0; h < heads; ++h)
    if (lane < D / 2) *((uint32_t*)((uint16_t*)a.out.data + b * a.out.token_stride + h * a.out.head_stride) + lane) = 0u;
  if (a.lse)
    for (uint32_t h = lane; h < heads; h += 64) a.lse[(uint64_t)b * heads + h] = -__builtin_inff();
}

// The kernel's arguments read again where they are used: what a part or the end of a run needs is not kept in scalar registers (or
// spilled from them) through the tiles' loop.
__device__ __forceinline__ const PagedAttnArgs& again() {
  auto p = (const __attribute__((address_space(4))) PagedAttnArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const PagedAttnArgs*)p;
}

// ---------------------------------------------------------------------------------------------------- the kernel
template <int KB, int VB, int NH, bool TWO>
struct Lds {  // dwords
  static constexpr uint32_t kTab = tables_bytes(KB, VB, TWO) / 4;
  static constexpr uint32_t kMerge = W * (2 * NH + NC * 4 * (NH == 4 ? 32 : 64));
  static constexpr uint32_t kRows = TWO && NH == 8 ? 8 : 4;   // of staged weights per wave
  static constexpr uint32_t kHead = kTab > kMerge ? kTab : kMerge;
  static constexpr uint32_t kWords = kHead + W * kRows * kPRow + 2 * W + 1;
};

template <int KB, int VB, int NH, int IO>
__global__ __launch_bounds__(64 * W) void paged_attn(PagedAttnArgs a) {
  constexpr bool TWO = IO == 1;
  using L = Lds<KB, VB, NH, TWO>;
  constexpr int GC = D / 4;                                  // codes of a key row that one lane group holds
  constexpr int KW = KB ? (GC * (KB ? KB : 1) + 31) / 32 : GC / 4;   // words a lane holds of them
  constexpr int RC = D / 16;                                 // codes of a value row that one lane holds
  constexpr int VW = VB == 0 && D == 128 ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) uint32_t s_mem[];   // at LDS address 0
  uint32_t* const s_stage = s_mem + L::kHead;
  uint32_t* const s_key = s_stage + W * L::kRows * kPRow;
  uint32_t* const s_run = s_key + W;   // the waves' first tiles, and the last one's end
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wid = __builtin_amdgcn_readfirstlane(tid >> 6), upper = g & 1 ? ~0u : 0u;
  const uint32_t heads = a.layout.kv_heads;

  const int32_t raw = a.lengths[min((uint32_t)lane, a.sequences - 1)];   // (in front of the tables' loads: they return in order)
  int32_t raw_own = a.lengths[min(blockIdx.x * W + wid, a.sequences - 1)];
  __builtin_amdgcn_sched_barrier(0);
  Table<KB, TWO> ktab;
  Table<VB, TWO> vtab;
  ktab.load(a.k, tid);
  vtab.load(a.v, tid);
  Line line;
  line.load(a, raw, lane);
  const uint32_t total = line.units * heads;
  // empty sequences: zeros
  for (uint32_t b = blockIdx.x * W + wid; b < a.sequences; b += a.groups * W) {
    if (span_of(a, cut_length(a, raw_own)).tiles == 0) write_zeros(a, b, lane);
    raw_own = a.lengths[min(b + a.groups * W, a.sequences - 1)];
  }
  const Cut cut(total, a);
  uint32_t u0 = cut.begin(blockIdx.x, a), u1 = cut.begin(blockIdx.x + 1, a);
  if (a.whole) {
    if (u0 < total) u0 -= line.find(a, u0, lane).unit;
    if (u1 < total) u1 -= line.find(a, u1, lane).unit;
  }
  if (u0 >= u1) {
    if (tid == 0) ((uint32_t*)a.ws)[4 * blockIdx.x] = 0u;
    return;
  }
  const uint32_t from = u0 + wave_begin(u1 - u0, wid), to = u0 + wave_begin(u1 - u0, wid + 1);
  const uint32_t x1 = to < total ? line.find(a, to, lane).x : line.tiles * heads;
  Place place{0u, 0u, 0u, 0u, x1};
  if (from < to) place = line.find(a, from, lane);
  const uint32_t x0 = place.x;   // this wave's tiles: [x0, x1) of the line
  const uint32_t klb = lane_byte<KB, TWO>(lane) + key_base(KB, VB, TWO), vlb = lane_byte<VB, TWO>(lane) + value_base(KB, VB, TWO);
  uint32_t* const s_w = s_stage + wid * L::kRows * kPRow;

  // A part of a pair of sequence and KV head: tiles [.., end) of the line belong to it and to this wave's run.
  struct Part {
    uint32_t seq, kv, pair_begin, pair_end, end;
    bool whole;
  };
  // ---- offsets of this lane inside a row of codes
  const uint32_t kstep = a.kslot;
  uint32_t koff[KB ? 1 : KW / 2], ksh[KB ? 1 : KW / 2];
  if constexpr (KB != 0) {
    koff[0] = (uint32_t)n * kstep + (uint32_t)((GC * KB * g) >> 5) * 4u;
    ksh[0] = (uint32_t)((GC * KB * g) & 31);
  } else {  // groups of eight codes, `bits` bytes each, read as eight bytes that stay inside the row
#pragma unroll
    for (int i = 0; i < KW / 2; ++i) {
      const uint32_t at = ((uint32_t)g * (GC / 8) + i) * a.k.bits, lo = min(at, a.k.row_bytes - 8u);
      koff[i] = (uint32_t)n * kstep + lo;
      ksh[i] = 8u * (at - lo);
    }
  }
  const uint32_t vbit = (uint32_t)(RC * n) * a.v.bits, vlo = min(vbit >> 3, a.v.row_bytes - 4u * VW), vsh = vbit - 8u * vlo;
  constexpr bool kShiftV = !(VB == 4 && D == 128);

  // ---- the loads run a tile ahead of the computation: the part of the next tile to load, this lane's page and offset (of its 16
  // tokens) in it
  uint32_t xl = x0, tok = 0, col = 0, off = 0, run_end = 0, page = ~0u, span_begin = 0, span_end = 0;
  Part part{};
  const int32_t* table = a.tables;
  auto begin_part = [&]() __attribute__((always_inline)) {
    const PagedAttnArgs& a = again();
    const Span sp = span_of(a, (uint32_t)__builtin_amdgcn_readlane(line.len, place.lane));
    const uint32_t tile = place.tile;
    const uint32_t seq = line.first + place.lane;
    part.seq = seq;
    part.kv = place.kv;
    part.pair_begin = xl - tile;
    part.pair_end = part.pair_begin + sp.tiles;
    part.end = min(part.pair_end, x1);
    part.whole = tile == 0 && part.end == part.pair_end;
    tok = sp.base + tile * 64u + 16u * g;
    col = quotient(tok >> 4, a.layout.page_size >> 4, a.page_r);
    off = tok - col * a.layout.page_size;
    run_end = min(sp.end, sp.base + (tile + part.end - xl) * 64u);
    span_begin = sp.begin;
    span_end = sp.end;
    table = a.tables + (uint64_t)seq * a.table_width;
  };
  auto page_of = [&]() __attribute__((always_inline)) { return tok < run_end ? (uint32_t)table[col] : ~0u; };   // no page beyond the part is looked up
  // A tile's loads run ahead of its computation: the keys' are issued when the tile before has its scores, the values' and the
  // scales' when it is done. A page outside the pool, or past the run, is read as the one before it (first: 0; in bounds, weight zero); there is no
  // branch around a load, so that the compiler knows how many are in flight.
  uint32_t kw[4][KW], vw[16][VW], safe = 0, offs = 0;
  float nk = 0.f, nv = 0.f, dist = 0.f;
  bool in = false;
  Part loaded{};
  auto load_keys = [&]() __attribute__((always_inline)) {
    loaded = part;
    const bool there = page < a.layout.pages;
    safe = there ? page : safe;
    offs = there ? off : offs;
    in = there && tok + n < span_end && tok + n >= span_begin;
    dist = (float)(int32_t)(tok + n - (span_end - 1u));
    // the first row of this lane's 16 tokens; of all four groups of 16 in scalar registers
    const uint64_t row = (uint64_t)(a.k.codes + (uint64_t)part.kv * a.khead) + (uint64_t)safe * a.kpage + (uint64_t)(offs * a.kslot);
    uint32_t k0[KB ? 1 : KW / 2];
#pragma unroll
    for (int i = 0; i < (KB ? 1 : KW / 2); ++i) {
      k0[i] = koff[i];
      asm volatile("" : "+v"(k0[i]));   // a 32-bit lane offset to a scalar base, not a 64-bit sum kept in registers
    }
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const global_u8* const base = (const global_u8*)((uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)row, 16 * m) |
                                                   (uint64_t)(uint32_t)__builtin_amdgcn_readlane((uint32_t)(row >> 32), 16 * m) << 32);
      if constexpr (KB != 0) {
        const global<uint32_t>* const q = (const global<uint32_t>*)(base + k0[0]);
        if constexpr (KW == 4) {
          const u32x4 v = *(const global<u32x4>*)q;
          kw[m][0] = v.x; kw[m][1] = v.y; kw[m][2] = v.z; kw[m][3] = v.w;
        } else if constexpr (KW == 3) {
          const u32x3 v = *(const global<u32x3>*)q;
          kw[m][0] = v.x; kw[m][1] = v.y; kw[m][2] = v.z;
        } else if constexpr (KW == 2) {
          const u32x2 v = *(const global<u32x2>*)q;
          kw[m][0] = v.x; kw[m][1] = v.y;
        } else {
          kw[m][0] = *q;
        }
      } else {
#pragma unroll
        for (int i = 0; i < KW / 2; ++i) {
          const uint64_t v = *(const global<u64_any>*)(base + k0[i]);
          kw[m][2 * i] = (uint32_t)v;
          kw[m][2 * i + 1] = (uint32_t)(v >> 32);
        }
      }
    }
    ++xl;
    tok += 64u;
    col += a.tile_cols;
    off += a.tile_rest;
    if (off >= a.layout.page_size) {
      off -= a.layout.page_size;
      ++col;
    }
    if (xl < x1 && xl == part.end) {
      line.next(again(), place, lane);
      begin_part();
    }
    page = page_of();
  };
  // values: a lane group takes the 16 tokens of its own page, so that a lane's rows follow each other
  auto load_values = [&]() __attribute__((always_inline)) {
    const uint8_t* base = a.v.codes + (uint64_t)loaded.kv * a.vhead + (uint64_t)safe * a.vpage + (uint64_t)(offs * a.vslot + vlo);
    auto load_row = [&](int j, const uint8_t* q) __attribute__((always_inline)) {
      if constexpr (VW == 2) {
        const uint64_t v = *(const u64_any*)q;
        vw[j][0] = (uint32_t)v;
        vw[j][1] = (uint32_t)(v >> 32);
      } else {
        vw[j][0] = *(const u32_any*)q;
      }
    };
    if (VB != 0 && a.layout.slot_step == 1) {   // head-major pages: constant distances
#pragma unroll
      for (int j = 0; j < 16; ++j) load_row(j, base + j * (D * VB / 8));
    } else {
#pragma unroll
      for (int j = 0; j < 16; ++j, base += a.vslot) load_row(j, base);
    }
    const uint64_t row = (uint64_t)loaded.kv * a.layout.head_step + (uint64_t)safe * (uint32_t)a.layout.page_stride +
                         (uint64_t)((offs + n) * a.layout.slot_step);
    nk = a.k.scales[row];
    nv = a.v.scales[row];
  };

  // Queries: a lane (head, group) loads eight coordinates from 32 t + 8 g of its head for every t, the other operand of the rotation.
  uint32_t yraw[KS][4];
  auto load_queries = [&](const Part& p) __attribute__((always_inline)) {
    const PagedAttnArgs& a = again();
    const uint32_t h = NH == 4 ? n & 3 : n & 7;
    const uint16_t* const q = (const uint16_t*)a.q.data + p.seq * a.q.token_stride + (p.kv * a.nq + min(h, a.nq - 1u)) * a.q.head_stride + 8 * g;
#pragma unroll
    for (int t = 0; t < KS; ++t) {
      const u32x4 v = *(const u32x4*)(q + 32 * t);
      yraw[t][0] = v.x; yraw[t][1] = v.y; yraw[t][2] = v.z; yraw[t][3] = v.w;
    }
  };

  uint32_t qa[KS][4];
  float qs[NH], slope[NH], M[NH], l[NH], S[NH];
  v4f acc[NC];
  bool tail = false;
  Part cur{};
  // ---- a part begins: the score operand of its queries, which are in yraw
  auto prepare = [&]() __attribute__((always_inline)) {
    const PagedAttnArgs& a = again();
    {
      const uint32_t h = NH == 4 ? n & 3 : n & 7, part = NH == 4 ? n >> 2 : n >> 3;
      // H (s q) on the matrix cores, exactly: rows of +1 and -1 times the raw queries with their signs flipped. Instruction b
      // gives this lane (head n, group g) coordinates GC g + 4 b .. + 3: its row r is coordinate i = GC (r / 4) + 4 b + r % 4, and
      // the entry at coordinate j = 32 t + 8 g + e is the parity of i & j.
#pragma unroll
      for (int t = 0; t < KS; ++t) {
        const uint32_t sg = a.k.signs[t] >> (8 * g);
#pragma unroll
        for (int k = 0; k < 4; ++k) yraw[t][k] ^= (sg >> (2 * k) & 1u) << 15 | (sg >> (2 * k + 1) & 1u) << 31;
      }
      constexpr uint32_t kOne = IO == 1 ? 0x3C003C00u : 0x3F803F80u;
      uint32_t row = n, grp = g;   // (opaque: the matrix's rows are formed here, not kept in registers for all parts)
      asm volatile("" : "+v"(row), "+v"(grp));
      uint32_t one[2][4];   // b even, odd: parity of (4 b + r % 4) & e for e = 2 k, 2 k + 1
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint32_t r = row & 3, lo = (uint32_t)__builtin_popcount(r & (2 * k)) & 1u, hi = (uint32_t)__builtin_popcount(r & (2 * k + 1)) & 1u;
        one[0][k] = kOne ^ (lo << 15 | hi << 31);
        one[1][k] = one[0][k] ^ (k >= 2 ? 0x80008000u : 0u);
      }
      const uint32_t rt = row >> 2;
      float y[GC];
#pragma unroll
      for (int b = 0; b < GC / 4; ++b) {
        // i's bits 3 and up within a quarter go with g, its quarter with t
        const uint32_t sb = (uint32_t)__builtin_popcount((b >> 1) & grp) & 1u;
        v4f c{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < KS; ++t) {
          const uint32_t flip = (D == 128 ? sb ^ ((uint32_t)__builtin_popcount(rt & t) & 1u)
                                          : (uint32_t)__builtin_popcount((((rt & 1) << 1) | (b >> 1)) & grp) + (rt >> 1 & (uint32_t)t) & 1u) ? 0x80008000u : 0u;
          const w4 hrow{one[b & 1][0] ^ flip, one[b & 1][1] ^ flip, one[b & 1][2] ^ flip, one[b & 1][3] ^ flip};
          const w4 q{yraw[t][0], yraw[t][1], yraw[t][2], yraw[t][3]};
          c = IO == 1 ? mfma_f16(hrow, q, c) : mfma_bf16(hrow, q, c);
        }
#pragma unroll
        for (int v = 0; v < 4; ++v) y[4 * b + v] = c[v];
      }
      float mx = 0.f;
#pragma unroll
      for (int e = 0; e < GC; ++e) mx = fmax_hw(mx, __builtin_fabsf(y[e]));
      mx = max16(mx, mx);
      mx = max32(mx, mx);
      const int ex = min(max(exponent_of(mx), -100), 126);
      // heads that the call has not, and the rows of further parts, are zero
      const float sc = h < a.nq && part < 2 ? pow2i(14 - ex > 127 ? 127 : 14 - ex) : 0.f;
#pragma unroll
      for (int h2 = 0; h2 < NH; ++h2) qs[h2] = lane_value(pow2i(ex - 14) * a.kinv * a.qscale, h2);
#pragma unroll
      for (int e = 0; e < GC; e += 2) {
        const float p = y[e] * sc, r = y[e + 1] * sc;
        const uint32_t hi = f16_pair(p, r);
        float hp, hr;
        widen2<1>(hi, hp, hr);
        const uint32_t low = f16_pair(p - hp, r - hr);
        qa[e / 8][(e % 8) / 2] = part == 0 ? hi : low;
      }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      slope[h] = a.slopes && h < (int)a.nq ? a.slopes[cur.kv * a.nq + h] * a.slope_scale : 0.f;
      M[h] = -__FLT_MAX__;   // the lowest finite value: a score of minus infinity weighs nothing, also before any other
      l[h] = 0.f;
      S[h] = 1.f;
    }
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] = v4f{0.f, 0.f, 0.f, 0.f};
  };

  auto compute = [&]() __attribute__((always_inline)) {
    // ---- scores: rows 4 g .. 4 g + 3 (parts, heads) of token 16 m + n
    v4f cs[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      cs[m] = v4f{0.f, 0.f, 0.f, 0.f};
      if constexpr (KB == 0) {
        if (a.k.bits == 8) continue;   // a row's words are whole codes
#pragma unroll
        for (int j = 0; j < KW / 2; ++j) {
          const uint64_t v = ((uint64_t)kw[m][2 * j + 1] << 32 | kw[m][2 * j]) >> ksh[j];
          kw[m][2 * j] = spread((uint32_t)v, a.k.bits);
          kw[m][2 * j + 1] = spread((uint32_t)(v >> 4 * a.k.bits), a.k.bits);
        }
      } else if constexpr (GC * KB % 32 != 0) {
#pragma unroll
        for (int k = 0; k < KW; ++k) kw[m][k] = __builtin_amdgcn_alignbit(k + 1 < KW ? kw[m][k + 1] : 0u, kw[m][k], ksh[0]);
      }
    }
    {
      // the table reads of three instructions' operands ahead (12 or so are what the LDS counter tells apart)
      uint32_t hi[4][4], lo[4][4];
      auto look = [&](int k) {
        const int s = k >> 2, m = k & 3;
        look_pairs<KB, TWO, 4>(kw[m], 8 * (KB ? KB : 8) * s, klb, a.k.polar != 0, hi[k & 3], lo[k & 3]);
      };
      constexpr int kAhead = KB == 0 ? 1 : 2;
#pragma unroll
      for (int k = 0; k < kAhead; ++k) look(k);
#pragma unroll
      for (int k = 0; k < 4 * KS; ++k) {
        if (k + kAhead < 4 * KS) look(k + kAhead);
        __builtin_amdgcn_sched_barrier(0);
        const int s = k >> 2, m = k & 3;
        const w4 q{qa[s][0], qa[s][1], qa[s][2], qa[s][3]};
        cs[m] = mfma_f16(q, w4{hi[k & 3][0], hi[k & 3][1], hi[k & 3][2], hi[k & 3][3]}, cs[m]);
        if constexpr (TWO) cs[m] = mfma_f16(q, w4{lo[k & 3][0], lo[k & 3][1], lo[k & 3][2], lo[k & 3][3]}, cs[m]);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    // sum of the parts; lane l gets the scores of token l of the tile
    float z[NH];
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float p = fold32(cs[0][v], cs[2][v]), r = fold32(cs[1][v], cs[3][v]);
      if constexpr (NH == 8) {
        const auto x = __builtin_amdgcn_permlane16_swap(__float_as_uint(p), __float_as_uint(r), false, false);
        z[v] = __uint_as_float(x[0]);
        z[4 + v] = __uint_as_float(x[1]);
      } else {
        z[v] = fold16(p, r);
      }
    }

    const bool now_in = in;
    const float now_dist = dist, now_nk = nk, now_nv = nv;
    load_keys();
    __builtin_amdgcn_sched_barrier(0);
    // ---- online softmax. The maximum and the weights' factor S are kept until a score or a weight leaves their range.
    const float n_t = now_in ? now_nv : 0.f;
#pragma unroll
    for (int h = 0; h < NH; ++h) z[h] *= qs[h] * now_nk;
    if (a.cap > 0.f) {
      asm volatile("");   // a branch: no instruction of it runs where no score is capped
      // cap tanh(t), t = z / cap. Up to 0.4 the odd series, whose next term is 2^-24 of the value: the score keeps its bits however
      // large the cap is (1 - 2 / (1 + exp(2 t)) cancels: 1e-7 of the cap, 0.1 of a score at a cap of 1e6). The exponentials only
      // where a tile has a larger t.
      bool far = false;
#pragma unroll
      for (int h = 0; h < NH; ++h) far |= now_in && !(__builtin_fabsf(z[h] * a.cap_r) <= 0.4f);
      auto series = [](float t) {
        const float s = t * t;
        float x = __builtin_fmaf(s, -1382.f / 155925.f, 62.f / 2835.f);
        x = __builtin_fmaf(s, x, -17.f / 315.f);
        x = __builtin_fmaf(s, x, 2.f / 15.f);
        x = __builtin_fmaf(s, x, -1.f / 3.f);
        return __builtin_fmaf(s, x, 1.f);
      };
      if (!__any(far)) {
#pragma unroll
        for (int h = 0; h < NH; ++h) z[h] *= series(z[h] * a.cap_r);
      } else {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          const float t = z[h] * a.cap_r;
          const float y = a.cap * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(t * 2.885390082f)));   // 2 log2(e)
          z[h] = __builtin_fabsf(t) <= 0.4f ? z[h] * series(t) : y;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) z[h] = now_in ? __builtin_fmaf(slope[h], now_dist, z[h]) : -__builtin_inff();
    float p[NH], y[NH], top = -__FLT_MAX__, most = 0.f;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const float x = z[h] - M[h];
      p[h] = __builtin_amdgcn_exp2f(x);
      y[h] = p[h] * n_t * S[h];
      top = fmax_hw(top, x);
      most = fmax_hw(most, __builtin_fabsf(y[h]));
    }
    const bool over = top > 6.f || most > kTop;
    if (__any(over)) {
      float f[NH], mx[NH];
      wave_max_heads(z, mx);
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        const float m = fmax_hw(M[h], mx[h]), al = __builtin_amdgcn_exp2f(M[h] - m);
        M[h] = m;
        l[h] *= al;
        f[h] = al >= 0x1p-126f ? al : 0.f;
        p[h] = __builtin_amdgcn_exp2f(z[h] - m);
        y[h] = __builtin_fabsf(p[h] * n_t);
      }
      wave_max_heads(y, mx);
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        // the accumulators are relative to M and times S: a new maximum leaves them as they are with S / al. Otherwise S follows the
        // tile's largest weight (from 2^-127 on; without any, it waits at 2^60 for the next), and the accumulators never grow.
        const float keep = S[h] * __builtin_amdgcn_rcpf(f[h]);
        float s_new = keep, fac = 1.f;
        if (!(keep <= 0x1p60f && mx[h] * keep <= kTop)) {
          s_new = fmin_hw(pow2i(mx[h] > 0.f ? min(13 - max(exponent_of(mx[h]), -100), 113) : 60), keep);
          fac = f[h] * s_new * __builtin_amdgcn_rcpf(S[h]);
        }
        S[h] = s_new;
        f[h] = fac;
        y[h] = p[h] * n_t * S[h];
      }
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float fv = NH == 8 ? pick(upper, f[v], f[NH - 4 + v]) : f[v];
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c][v] *= fv;
      }
    }
#pragma unroll
    for (int h = 0; h < NH; ++h) l[h] += p[h];
    // row r of the staged weights: four heads, head r's two parts; eight, the weights of heads r and r + 4 (float16: row 4 + r
    // their rests)
    constexpr bool REST = TWO && NH == 8;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (NH == 4) {
        const float hi = (float)(_Float16)y[r];
        s_w[r * kPRow + lane] = f16_pair(hi, (y[r] - hi) * kLoScale);
      } else {
        const uint32_t hi = f16_pair(y[r], y[r + 4]);
        s_w[r * kPRow + lane] = hi;
        if constexpr (REST) {
          float p0, p1;
          widen2<1>(hi, p0, p1);
          s_w[(4 + r) * kPRow + lane] = f16_pair(y[r] - p0, y[r + 4] - p1);
        }
      }
    }
    wave_lds_fence();

    // ---- weighted values: the accumulators' rows 0 - 7 weigh a pair's first coordinate, 8 - 15 its second
    if (kShiftV && (VB != 0 || a.v.bits != 8)) {
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if constexpr (VW == 2) {
          const uint64_t v = ((uint64_t)vw[j][1] << 32 | vw[j][0]) >> vsh;
          vw[j][0] = spread((uint32_t)v, a.v.bits);
          vw[j][1] = spread((uint32_t)(v >> 4 * a.v.bits), a.v.bits);
        } else {
          vw[j][0] >>= vsh;
          if constexpr (VB == 0) vw[j][0] = spread(vw[j][0], a.v.bits);
        }
      }
    }
    const uint32_t* const s_row = s_w + (n & 3) * kPRow + 16 * g;   // tokens 16 g + 4 m + j
    const uint32_t sel = n < 8 ? (n & 4 ? 0x0C0C0302u : 0x0C0C0100u) : (n & 4 ? 0x03020C0Cu : 0x01000C0Cu);
    // a step: the pairs c (two bits: c and c + 1, which one table read gives) of four tokens
    constexpr int PC = VB == 2 ? 2 : 1, NS = 4 * NC / PC, kAhead = VB == 0 ? 1 : 2;
    uint32_t v[4][4][PC], rest[4][4][PC];
    w4 d[4], dr[4], wa{}, wr{};
    auto look = [&](int k) __attribute__((always_inline)) {
      const int m = k / (NC / PC), c = k % (NC / PC) * PC;
      if (c == 0) d[m] = *(const w4*)(s_row + 4 * m);
      if (REST && c == 0) dr[m] = *(const w4*)(s_row + 4 * kPRow + 4 * m);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        look_pairs<VB, TWO, PC>(vw[4 * m + j], 2 * (VB ? VB : 8) * c, vlb, a.v.polar != 0, v[k & 3][j], rest[k & 3][j]);
      }
    };
#pragma unroll
    for (int k = 0; k < kAhead; ++k) look(k);
#pragma unroll
    for (int k = 0; k < NS; ++k) {
      if (k + kAhead < NS) look(k + kAhead);
      __builtin_amdgcn_sched_barrier(0);
      const int m = k / (NC / PC), c = k % (NC / PC) * PC;
      if (c == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          wa[j] = __builtin_amdgcn_perm(0u, d[m][j], sel);
          if (REST) wr[j] = __builtin_amdgcn_perm(0u, dr[m][j], sel);
        }
      }
#pragma unroll
      for (int i = 0; i < PC; ++i) {
        const w4 x{v[k & 3][0][i], v[k & 3][1][i], v[k & 3][2][i], v[k & 3][3][i]};
        acc[c + i] = mfma_f16(wa, x, acc[c + i]);
        if (REST) acc[c + i] = mfma_f16(wr, x, acc[c + i]);
        if (TWO) acc[c + i] = mfma_f16(wa, w4{rest[k & 3][0][i], rest[k & 3][1][i], rest[k & 3][2][i], rest[k & 3][3][i]}, acc[c + i]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    wave_lds_fence();
  };

  // ---- a part is done: sums over the lanes, parts added, factors taken out
  auto finish = [&]() __attribute__((always_inline)) {
    const PagedAttnArgs& a = again();
    float* const ws = a.ws + 4 * a.groups;
#pragma unroll
    for (int h = 0; h < NH; ++h) l[h] = wave_sum(l[h]);
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = a.vinv * __builtin_amdgcn_rcpf(NH == 8 ? pick(upper, S[v], S[NH - 4 + v]) : S[v]);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        if constexpr (NH == 4) {
          const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[c][v]), __float_as_uint(acc[c][v]), false, false);
          acc[c][v] = __builtin_fmaf(__uint_as_float(r[1]), 1.f / kLoScale, __uint_as_float(r[0]));
        }
        acc[c][v] *= f;
      }
    }
    if (cur.whole) {
      write_output<NH, IO>(a, cur.seq, cur.kv, acc, M, l, lane);
    } else if (cur.end == x1) {
      tail = true;
    } else {
      float* const out = ws + (uint64_t)(wid ? wave_slot(a.groups, blockIdx.x, wid) : left_slot(blockIdx.x)) * slot_floats(NH);
      if (lane == 0) {
#pragma unroll
        for (int h = 0; h < NH; ++h) {
          out[h] = M[h];
          out[8 + h] = l[h];
        }
      }
      if (NH == 8 || !(g & 1)) {
        const int at = NH == 8 ? lane : n + 16 * (g >> 1);
#pragma unroll
        for (int c = 0; c < NC; ++c) *(v4f*)(out + 16 + (c * (NH == 4 ? 32 : 64) + at) * 4) = acc[c];
      }
    }
  };
  if (x0 < x1) {
    begin_part();
    page = page_of();
    cur = part;
    load_queries(cur);
  }
  // the tables are written while the page is looked up
  ktab.write(s_mem + key_base(KB, VB, TWO) / 4, a.k, a.kfactor, tid);
  vtab.write(s_mem + value_base(KB, VB, TWO) / 4, a.v, a.vfactor, tid);
  __builtin_amdgcn_sched_barrier(0);
  if (x0 < x1) {
    load_keys();
    load_values();
  }
  // (orders LDS only: the loads of the first tile stay on their way)
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
  if (x0 < x1) {
    prepare();
    for (uint32_t xc = x0;;) {
      compute();
      if (++xc == x1) break;
      load_values();
      __builtin_amdgcn_sched_barrier(0);
      if (xc == cur.end) {
        const Part next = loaded;
        load_queries(next);
        finish();
        cur = next;
        prepare();
      }
    }
    finish();
  }
  const uint32_t key = tail ? cur.seq * heads + cur.kv : ~0u;   // (pairs with tiles: below 2^31)

  const PagedAttnArgs& e = again();
  float* const ws = e.ws + 4 * e.groups;
  // ---- the last parts of neighbouring waves, where they are of one pair, merge through LDS (the tables' space)
  __syncthreads();
  constexpr int kMl = 2 * NH, kLanes = NH == 4 ? 32 : 64;
  float* const s_ml = (float*)s_mem;
  v4f* const s_acc = (v4f*)(s_mem + W * kMl);
  const int at = NH == 8 ? lane : n + 16 * (g >> 1);
  if (lane == 0) {
    s_key[wid] = key;
    s_run[wid] = x0;
    if (wid == W - 1) s_run[W] = x1;
  }
  if (tail) {
    if (lane == 0) {
#pragma unroll
      for (int h = 0; h < NH; ++h) {
        s_ml[wid * kMl + h] = M[h];
        s_ml[wid * kMl + NH + h] = l[h];
      }
    }
    if (NH == 8 || !(g & 1)) {
#pragma unroll
      for (int c = 0; c < NC; ++c) s_acc[(wid * NC + c) * kLanes + at] = acc[c];
    }
  }
  __syncthreads();
  auto key_of = [&](uint32_t w) { return (uint32_t)__builtin_amdgcn_readfirstlane(s_key[w]); };
  uint32_t first = wid, last = wid;
  if (tail) {
    ++last;
    while (first > 0 && key_of(first - 1) == key) --first;
    while (last < W && key_of(last) == key) ++last;
  }
  // the waves [first, last) have the pair's tiles [begin, end); the next one may have the rest of it, which ends inside its run
  auto run_of = [&](uint32_t w) { return (uint32_t)__builtin_amdgcn_readfirstlane(s_run[w]); };
  const uint32_t g0 = run_of(0), g1 = run_of(W), begin = run_of(first), end = run_of(last);
  const bool rest = tail && end < g1 && cur.pair_end > end;
  const bool whole = tail && begin <= cur.pair_begin && (rest || end >= cur.pair_end);
  const float* const rest_in = ws + (uint64_t)wave_slot(e.groups, blockIdx.x, last) * slot_floats(NH);
  float* const out = ws + (uint64_t)(cur.pair_end <= g1 ? left_slot(blockIdx.x) : right_slot(blockIdx.x)) * slot_floats(NH);
  float mm[NH], lm[NH];
  if (tail) {
    // maxima and sums: lane NH w + h has head h's of wave w
    const uint32_t lw = (uint32_t)lane / NH, lh = (uint32_t)lane % NH;
    const bool mine = lw >= first && lw < last;
    const uint32_t from = mine ? lw : wid;
    const float pm = mine ? s_ml[from * kMl + lh] : -__FLT_MAX__, pl = mine ? s_ml[from * kMl + NH + lh] : 0.f;
    const float rm = rest ? rest_in[lh] : -__FLT_MAX__, rl = rest ? rest_in[8 + lh] : 0.f;
    auto other = [&](float x, int d) { return __uint_as_float((uint32_t)__builtin_amdgcn_ds_bpermute((lane ^ d) << 2, (int)__float_as_uint(x))); };
    float top = fmax_hw(pm, rm);
#pragma unroll
    for (int d = NH; d < NH * W; d *= 2) top = fmax_hw(top, other(top, d));
    const float pe = mine ? __builtin_amdgcn_exp2f(pm - top) : 0.f, re = __builtin_amdgcn_exp2f(rm - top);
    float sum = pl * pe;
#pragma unroll
    for (int d = NH; d < NH * W; d *= 2) sum += other(sum, d);
    sum = __builtin_fmaf(rl, re, sum);
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      mm[h] = lane_value(top, h);
      lm[h] = lane_value(sum, h);
    }
    if (last - first == 1 && !rest) {   // nothing to add
      if (!whole && (NH == 8 || !(g & 1))) {
#pragma unroll
        for (int c = 0; c < NC; ++c) *(v4f*)(out + 16 + (c * kLanes + at) * 4) = acc[c];
      }
    } else
    // the accumulators' columns, shared out over these waves: column c is read and written by one wave alone
    for (uint32_t c = wid - first; c < NC; c += last - first) {
      v4f x[W], col{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < W; ++w) x[w] = s_acc[(w * NC + c) * kLanes + at];
      if (rest) {
        const v4f y = *(const v4f*)(rest_in + 16 + (c * kLanes + at) * 4);
#pragma unroll
        for (int v = 0; v < 4; ++v) col[v] = y[v] * (NH == 8 ? pick(upper, lane_value(re, v), lane_value(re, NH - 4 + v)) : lane_value(re, v));
      }
#pragma unroll
      for (int w = 0; w < W; ++w) {
        const bool in = (uint32_t)w >= first && (uint32_t)w < last;   // (uniform; other waves' words are not looked at)
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float e = NH == 8 ? pick(upper, lane_value(pe, NH * w + v), lane_value(pe, NH * w + NH - 4 + v)) : lane_value(pe, NH * w + v);
          col[v] = __builtin_fmaf(in ? x[w][v] : 0.f, e, col[v]);
        }
      }
      if (NH == 8 || !(g & 1)) {
        if (whole) s_acc[(first * NC + c) * kLanes + at] = col;
        else *(v4f*)(out + 16 + (c * kLanes + at) * 4) = col;
      }
    }
  }
  __syncthreads();
  if (x0 < x1 && x1 == g1 && lane == 0) {
    const bool more = cur.pair_end > g1 && cur.pair_begin >= g0;
    const uint32_t unit = to + (cur.pair_end - x1);   // (the run ends inside the pair: only tiles are left of it)
    *(w4*)((uint32_t*)e.ws + 4 * blockIdx.x) = w4{more ? cut.group_of(unit - 1, e) + 1 : 0u, cur.seq, cur.kv, 0u};
  } else if (g0 == g1 && tid == 0) {
    ((uint32_t*)e.ws)[4 * blockIdx.x] = 0u;
  }
  if (!tail || first != wid) return;
  if (whole) {
    if (last - first > 1 || rest)
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[c] = s_acc[(first * NC + c) * kLanes + at];
    write_output<NH, IO>(e, cur.seq, cur.kv, acc, mm, lm, lane);
  } else if (lane == 0) {
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      out[h] = mm[h];
      out[8 + h] = lm[h];
    }
  }
}

// Joins the partial results of the pair of sequence and KV head that begins in a workgroup of paged_attn and goes on behind it: the
// waves share its parts out, a lane each has a part's maxima and sums.
constexpr int kJoinWaves = 8;
constexpr int kJoinParts = 4;   // of a wave at a time
template <int NH, int IO>
__global__ __launch_bounds__(64 * kJoinWaves) void paged_join(PagedAttnArgs a) {
  constexpr int kLanes = NH == 4 ? 32 : 64, kAtOnce = kJoinWaves * kJoinParts;
  __shared__ v4f s_acc[kJoinWaves - 1][NC][kLanes];
  const uint32_t heads = a.layout.kv_heads;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const uint32_t wid = __builtin_amdgcn_readfirstlane(tid >> 6), upper = g & 1 ? ~0u : 0u;
  const w4 pair = *(const w4*)((const uint32_t*)a.ws + 4 * blockIdx.x);
  const float* const ws = a.ws + 4 * a.groups;
  const int at = NH == 8 ? lane : n + 16 * (g >> 1);
  if (!pair[0]) return;   // (uniform over the workgroup)
  const uint32_t parts = pair[0] - blockIdx.x;
  auto part_of = [&](uint32_t c) {   // the last one ends in its workgroup
    return ws + (uint64_t)(c + 1 < parts ? right_slot(blockIdx.x + c) : left_slot(blockIdx.x + c)) * slot_floats(NH);
  };
  float M[NH], l[NH];
  v4f acc[NC];
#pragma unroll
  for (int h = 0; h < NH; ++h) {
    M[h] = -__FLT_MAX__;
    l[h] = 0.f;
  }
#pragma unroll
  for (int c = 0; c < NC; ++c) acc[c] = v4f{0.f, 0.f, 0.f, 0.f};
  for (uint32_t c0 = 0; c0 < parts; c0 += kAtOnce) {
    const bool there = lane < kAtOnce && c0 + lane < parts;
    const float* const in = part_of(min(c0 + (uint32_t)lane % kAtOnce, parts - 1));
    float pm[NH], pl[NH], mx[NH];
#pragma unroll
    for (int h = 0; h < NH; h += 4) {
      const v4f x = *(const v4f*)(in + h), y = *(const v4f*)(in + 8 + h);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        pm[h + k] = there ? x[k] : -__FLT_MAX__;
        pl[h + k] = there ? y[k] : 0.f;
      }
    }
    v4f y[kJoinParts][NC];   // (parts that are not there are read as the last one, and weigh nothing)
#pragma unroll
    for (int k = 0; k < kJoinParts; ++k) {
      const float* const part = part_of(min(c0 + k * kJoinWaves + wid, parts - 1)) + 16;
#pragma unroll
      for (int c = 0; c < NC; ++c) y[k][c] = *(const v4f*)(part + (c * kLanes + at) * 4);
    }
    wave_max_heads(pm, mx);
#pragma unroll
    for (int h = 0; h < NH; ++h) {
      const float m = fmax_hw(M[h], mx[h]), al = __builtin_amdgcn_exp2f(M[h] - m);
      pm[h] = there ? __builtin_amdgcn_exp2f(pm[h] - m) : 0.f;
      l[h] = __builtin_fmaf(l[h], al, wave_sum(pl[h] * pm[h]));
      M[h] = m;
      mx[h] = al;
    }
#pragma unroll
    for (int v = 0; v < 4; ++v) {
      const float f = NH == 8 ? pick(upper, mx[v], mx[NH - 4 + v]) : mx[v];
#pragma unroll
      for (int c = 0; c < NC; ++c) acc[c][v] *= f;
    }
#pragma unroll
    for (int k = 0; k < kJoinParts; ++k) {
      if (c0 + k * kJoinWaves + wid >= parts) break;
      float f[NH];
#pragma unroll
      for (int h = 0; h < NH; ++h) f[h] = lane_value(pm[h], (int)(k * kJoinWaves + wid));
#pragma unroll
      for (int v = 0; v < 4; ++v) {
        const float fv = NH == 8 ? pick(upper, f[v], f[NH - 4 + v]) : f[v];
#pragma unroll
        for (int c = 0; c < NC; ++c) acc[c][v] = __builtin_fmaf(y[k][c][v], fv, acc[c][v]);
      }
    }
  }
  if (wid > 0 && (NH == 8 || !(g & 1))) {
#pragma unroll
    for (int c = 0; c < NC; ++c) s_acc[wid - 1][c][at] = acc[c];
  }
  __syncthreads();
  if (wid != 0) return;
#pragma unroll
  for (int w = 0; w < kJoinWaves - 1; ++w)
#pragma unroll
    for (int c = 0; c < NC; ++c) acc[c] += s_acc[w][c][at];
  write_output<NH, IO>(a, pair[1], pair[2], acc, M, l, lane);
}

// ---------------------------------------------------------------------------------------------------- launch
template <int KB, int VB, int NH, int IO>
hipError_t launch_one(const PagedAttnArgs& a, hipStream_t s) {
  using L = Lds<KB, VB, NH, IO == 1>;
  constexpr uint32_t bytes = 4u * L::kWords;
  static_assert(bytes <= 160u * 1024u, "LDS of one workgroup");
  static_assert(slot_floats(NH) <= paged_slot_floats(D, NH), "a partial result fits its slot");
  if constexpr (bytes > 65536u) {   // once per device and kernel: the call takes as long as a launch
    static std::atomic<uint64_t> done{0};
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (dev > 63 || !(done.load(std::memory_order_relaxed) & bit)) {
      e = hipFuncSetAttribute((const void*)paged_attn<KB, VB, NH, IO>, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
      if (e != hipSuccess) return e;
      if (dev <= 63) done.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  hipLaunchKernelGGL((paged_attn<KB, VB, NH, IO>), dim3(a.groups), dim3(64 * W), bytes, s, a);
  if (!a.whole) hipLaunchKernelGGL((paged_join<NH, IO>), dim3(a.groups), dim3(64 * kJoinWaves), 0, s, a);
  return hipGetLastError();
}
template <int VB>
hipError_t launch_heads(const PagedAttnArgs& a, uint32_t io, hipStream_t s) {
  if (a.nq <= 4) return io == 1 ? launch_one<PITCH_KB, VB, 4, 1>(a, s) : launch_one<PITCH_KB, VB, 4, 2>(a, s);
  return io == 1 ? launch_one<PITCH_KB, VB, 8, 1>(a, s) : launch_one<PITCH_KB, VB, 8, 2>(a, s);
}

}  // namespace

#define PITCH_CAT4_(a, b, c, d) a##b##c##d
#define PITCH_CAT4(a, b, c, d) PITCH_CAT4_(a, b, c, d)
hipError_t PITCH_CAT4(launch_paged_attention_d, PITCH_DIM, _k, PITCH_KB)(const PagedAttnArgs& a0, uint32_t io, hipStream_t s) {
  PagedAttnArgs a = a0;
  a.kfactor = pitch_f16_factor(ilog2(D), a.k.polar, (int)a.k.bits);
  a.vfactor = pitch_f16_factor(ilog2(D), a.v.polar, (int)a.v.bits);
  a.kinv = 1.f / a.kfactor;
  a.vinv = 1.f / a.vfactor;
  a.groups_r = 0xFFFFFFFFu / a.groups;
  a.kpage = (uint32_t)a.layout.page_stride * a.k.row_bytes;
  a.vpage = (uint32_t)a.layout.page_stride * a.v.row_bytes;
  a.khead = a.layout.head_step * a.k.row_bytes;
  a.vhead = a.layout.head_step * a.v.row_bytes;
  a.kslot = a.layout.slot_step * a.k.row_bytes;
  a.vslot = a.layout.slot_step * a.v.row_bytes;
  const uint32_t most = a.window ? min(a.window + 15u, a.most_tokens) : a.most_tokens;
  // Pairs of a tile per wave at most: workgroups take whole ones, and there is no join (one sequence of up to 500 tokens and 8 KV
  // heads 13.0 us, 13.7 with the join; 100 22.3 and 23.8; 200 of 12 heads of 64 28 and 31). At 16 tiles one sequence takes 15.9 and
  // 14.0 us, 64 of eight bits 37 and 31: the waves of the longest pair are what the call waits for.
  a.whole = (most + 63) / 64 <= (uint32_t)W;
  a.page_r = 0xFFFFFFFFu / (a.layout.page_size / 16);
  a.tile_cols = 64 / a.layout.page_size;
  a.tile_rest = 64 % a.layout.page_size;
  switch (a.v.bits) {
    case 2: return launch_heads<2>(a, io, s);
    case 3: return launch_heads<3>(a, io, s);
    case 4: return launch_heads<4>(a, io, s);
    default: return launch_heads<0>(a, io, s);
  }
}

}  // namespace pitch
