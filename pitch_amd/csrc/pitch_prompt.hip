// Attention over whole prompts, for one dimension (PITCH_DIM = 64 or 128) and one 16-bit type (PITCH_IO = 1: float16, 2: bfloat16).
//
//   out_i = sum_j softmax(z_i)_j v_j,  z_ij = cap(scale q_i . k_j) + slope (j - p_i),  p_i = nk - nq + i,  p_i - window < j <= p_i
//
// Work split. The query heads of a KV head share its keys, so a row is a pair of token and head, and 128 neighbouring rows of a sequence
// are a query tile, a workgroup's work: four waves of 32 rows, two workgroups on a compute unit. It goes over the keys 64 at a time
// with the running maximum and sum of a softmax (Milakov and Gimelshein 2018; Rabe and Staats 2021). Workgroups that follow each other
// have different KV heads, so that an XCD, every eighth workgroup, finds the keys of few heads in its L2; tiles that see most keys
// come first, of each sequence or of all. Grid and workspace follow from sizes that the host knows, the lengths stay on the device.
//
// Products. v_mfma_f32_32x32x16 gives 32 x 32 scores as K Q^T, keys down and queries across: a lane holds 16 scores of one query, its
// partner at distance 32 the other 16, and maxima, sums and rescaling stay within the lane but for one exchange a tile. The weights
// are then the second operand of V^T P^T as they lie, if the 16 keys of a product are taken in the order 4 h .. 4 h + 3, 8 + 4 h ..
// 8 + 4 h + 3 in the lanes' halves h; V^T is read in that order by the transposing LDS reads (ds_read_b64_tr_b16, four keys by 16
// coordinates). Weights are rounded to the values' type, once; scores, maxima, sums and accumulators are float32. With bfloat16 the
// rounding of the weights is as large as the output's own, and averages like it: errors of outputs are 1.04 to 1.41 times those
// of the exact result's rounding (0.0021 to 0.0016 of the norm in a batch of prompts; float16 0.00029 to 0.00021 in chunks).
//
// Data. Tiles go from memory to LDS without registers (buffer_load ... lds), one ahead; chunks of 16 bytes lie swizzled, by the address
// that each lane asks for, so that no read finds a bank conflict (the counter says none). Rows behind the sequence come back as zeros
// (the buffers' bounds), and a mask is applied only in tiles that need one. The maximum in use lags by up to 2^8 behind a row's true
// one, so that the accumulators are rarely rescaled; weights up to 256 are as exact as those below 1.
//
// What bounds it. 16,381 tokens of 8 KV and 32 query heads of 128, bfloat16, causal: 2.02 to 2.18 ms on different cards, up to 1,090
// TFLOP/s, where a large library product reaches 1,400. Matrix instructions are on their way in 57 % of the cycles; the rest is mostly
// the softmax, 32 exponentials and about 120 other vector instructions for each 32 matrix instructions. The card lowers its clock under
// this load (1.9 GHz): a step that took 12 % of the cycles out took 8 % of the time. Twelve ragged prompts of up to 3,000 tokens 400 to
// 440 us (820 to 900 TFLOP/s): of a workgroup's 17 tiles of keys, 1.8 us each beside another's, 5 us are its beginning (0.8 until it knows its
// tile, 2.2 until queries and keys are there, 0.6 of the slowest wave) and its end (1.3), and 30 us pass while places run empty. Heads
// of 64 with soft caps in a window, 25.5 us, are bound by vector instructions (two in three cycles): the cap's polynomial, five a score
// (27.8 with nine; 11,486 tokens of four heads of 128 351 us, with nine 405), and the softmax. Slower were: 64 rows a wave (half the LDS
// reads, but one wave a SIMD); eight waves that share a tile of keys for 256 rows (2,050 us instead of 2,100, but 47 instead of 30 in
// the window and 137 instead of 124 for drafts) or by twos (2,250 us; the waves keep step); two tiles an iteration (2,110 us, spills);
// the next tile's scores among this one's weights (2,115 us beside 2,020, the second pass over what is not finite apart: two tiles of
// scores leave too few registers, and 30 are moved for each tile); and skipping of tiles that all rows of a wave are blind to, and the
// longest sequence first (no change). Queries that are waited for inside the loop cost 14 % (the counter of loads also counts the tiles
// on their way).
#include "pitch_attn_shared.h"
#include "pitch_prompt.h"

#ifndef PITCH_DIM
#error "compile with -DPITCH_DIM=<dim>"
#endif
#ifndef PITCH_IO
#error "compile with -DPITCH_IO=<io type>"
#endif

namespace pitch {
namespace {

constexpr int D = PITCH_DIM;
constexpr int kWaves = 4;            // of a workgroup, 32 rows each
constexpr int kRows = kWaves * 32;   // rows of a query tile
constexpr int kKeys = 64;            // keys of a tile
constexpr int kSteps = D / 16;       // steps of the contraction over the coordinates
constexpr int kBlocks = D / 32;      // blocks of 32 output coordinates
constexpr int kTileBytes = kKeys * D * 2;
constexpr int kLaneRows = 1024 / (D * 2);            // rows of a tile that a wave loads at once
constexpr int kLoads = kKeys / (kLaneRows * kWaves); // loads of a wave for a tile of keys or values
constexpr float kGrow = 8.f;         // log2 units that a row's scores may exceed the maximum in use by
constexpr float kNoScore = -__builtin_inff();
constexpr float kTanhSplit = 0.55f;

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t w2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) uint8_t lds_u8;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
typedef __attribute__((address_space(3))) w4 lds_w4;
typedef __attribute__((address_space(3))) void lds_void;

__device__ __forceinline__ v16f mfma(w4 a, w4 b, v16f c) {
  if constexpr (PITCH_IO == 1)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// Two values rounded to nearest even, in a word.
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  const f32x2 v = {x, y};
  if constexpr (PITCH_IO == 1)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
}
__device__ __forceinline__ uint32_t of_wave(uint32_t x) { return __builtin_amdgcn_readfirstlane(x); }

__device__ __forceinline__ float fmax3_abs(float a, float b, float c) {
  float r;
  asm("v_max3_f32 %0, %1, |%2|, |%3|" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// pre s tanh(x) / x, x = k s, for |x| below kTanhSplit: an even polynomial fitted at Chebyshev's points.
__device__ __forceinline__ float capped(float s, float k, float pre) {
  const float x = s * k, t = x * x, z = s * pre;
  float f = __builtin_fmaf(t, -0x1.b191fep-8f, 0x1.5d3024p-6f);
  f = __builtin_fmaf(t, f, -0x1.b9a19ap-5f);
  f = __builtin_fmaf(t, f, 0x1.110ff0p-3f);
  f = __builtin_fmaf(t, f, -0x1.555554p-2f);
  return __builtin_fmaf(z * t, f, z);
}
// x *= f where `go` is not zero. The branch is inside the statement: with one around it, the compiler keeps two copies of the
// accumulators and moves them, 64 registers there and back for every tile (2,190 us for 16,381 tokens; 2,016 without, and with maxima of
// three).
// Waits: 16 states behind the matrix instructions that wrote x, two before those that read it.
__device__ __forceinline__ void scale_where(uint64_t go, float f, v16f& x) {
  float y[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) y[r] = x[r];
  asm("s_cmp_eq_u64 %16, 0\n\t"
      "s_cbranch_scc1 .Lkept%=\n\t"
      "s_nop 7\n\ts_nop 7\n\t"
      "v_mul_f32 %0, %0, %17\n\tv_mul_f32 %1, %1, %17\n\tv_mul_f32 %2, %2, %17\n\tv_mul_f32 %3, %3, %17\n\t"
      "v_mul_f32 %4, %4, %17\n\tv_mul_f32 %5, %5, %17\n\tv_mul_f32 %6, %6, %17\n\tv_mul_f32 %7, %7, %17\n\t"
      "v_mul_f32 %8, %8, %17\n\tv_mul_f32 %9, %9, %17\n\tv_mul_f32 %10, %10, %17\n\tv_mul_f32 %11, %11, %17\n\t"
      "v_mul_f32 %12, %12, %17\n\tv_mul_f32 %13, %13, %17\n\tv_mul_f32 %14, %14, %17\n\tv_mul_f32 %15, %15, %17\n\t"
      "s_nop 1\n"
      ".Lkept%=:"
      : "+v"(y[0]), "+v"(y[1]), "+v"(y[2]), "+v"(y[3]), "+v"(y[4]), "+v"(y[5]), "+v"(y[6]), "+v"(y[7]), "+v"(y[8]), "+v"(y[9]),
        "+v"(y[10]), "+v"(y[11]), "+v"(y[12]), "+v"(y[13]), "+v"(y[14]), "+v"(y[15])
      : "s"(go), "v"(f)
      : "scc");
#pragma unroll
  for (int r = 0; r < 16; ++r) x[r] = y[r];
}

// The sum over this lane and those below it.
__device__ __forceinline__ uint32_t lanes_up_to(uint32_t x) {
  x += __builtin_amdgcn_update_dpp(0u, x, 0x111, 0xF, 0xF, false);  // row_shr:1
  x += __builtin_amdgcn_update_dpp(0u, x, 0x112, 0xF, 0xF, false);  // row_shr:2
  x += __builtin_amdgcn_update_dpp(0u, x, 0x114, 0xF, 0xF, false);  // row_shr:4
  x += __builtin_amdgcn_update_dpp(0u, x, 0x118, 0xF, 0xF, false);  // row_shr:8
  x += __builtin_amdgcn_update_dpp(0u, x, 0x142, 0xA, 0xF, false);  // row_bcast:15, to rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0u, x, 0x143, 0xC, 0xF, false);  // row_bcast:31, to rows 2 and 3
  return x;
}
__device__ __forceinline__ uint32_t of_lane(uint32_t x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
// The largest of all lanes.
__device__ __forceinline__ uint32_t most(uint32_t x) {
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x111, 0xF, 0xF, false));  // row_shr:1
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x112, 0xF, 0xF, false));  // row_shr:2
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x114, 0xF, 0xF, false));  // row_shr:4
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x118, 0xF, 0xF, false));  // row_shr:8
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x142, 0xA, 0xF, false));  // row_bcast:15, to rows 1 and 3
  x = max(x, __builtin_amdgcn_update_dpp(x, x, 0x143, 0xC, 0xF, false));  // row_bcast:31, to rows 2 and 3
  return of_lane(x, 63);
}

// A sequence's queries and keys, within the buffers.
struct Sequence {
  uint32_t first_query, queries, first_key, keys, tiles;
};
__device__ __forceinline__ Sequence sequence(const PromptArgs& a, uint32_t b) {
  Sequence s{};
  if (b >= a.sequences) return s;
  const int32_t q0 = a.row_starts[b], q1 = a.row_starts[b + 1], k0 = a.key_starts[b], k1 = a.key_starts[b + 1];
  s.first_query = min((uint32_t)max(q0, 0), a.rows);
  s.queries = max((int32_t)(min((uint32_t)max(q1, 0), a.rows) - s.first_query), 0);
  s.first_key = min((uint32_t)max(k0, 0), a.keys);
  s.keys = max((int32_t)(min((uint32_t)max(k1, 0), a.keys) - s.first_key), 0);
  s.tiles = (s.queries * a.nq + kRows - 1) / kRows;
  return s;
}

// A query tile: the rows [row, row + kRows) of (token, head) pairs of a sequence.
struct Tile {
  Sequence s;
  uint32_t row;
  bool any;
};
// Tile number `at` of all sequences, found by all of the waves alike. A sequence's last tile, whose rows see most, comes first; with
// by_height the highest of 64 sequences do, a tile's height being its number in its sequence and those that the keys before the queries
// would fill, and tiles of a height lie in the order of the sequences.
__device__ __forceinline__ Tile find_tile(const PromptArgs& a, uint32_t at) {
  const uint32_t lane = threadIdx.x & 63;
  Tile t{};
  for (uint32_t base = 0; base < a.sequences; base += 64) {
    const Sequence s = sequence(a, base + lane);
    const uint32_t sum = lanes_up_to(s.tiles), total = of_lane(sum, 63);
    if (at >= total) {
      at -= total;
      continue;
    }
    int who;
    if (!a.by_height) {
      who = __ffsll((unsigned long long)__ballot(sum > at)) - 1;
      t.row = (of_lane(sum, who) - 1 - at) * kRows;
    } else {
      const uint32_t before = (uint32_t)max((int32_t)(s.keys - s.queries), 0);
      const uint32_t bottom = (uint32_t)min((uint64_t)before * a.nq / kRows, (uint64_t)1 << 30), top = bottom + s.tiles;
      uint32_t lo = 0, hi = most(top), more = 0;   // the tile's height is in (lo, hi]; as many tiles lie above hi
      while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) / 2, above = s.tiles - min(s.tiles, max(mid, bottom) - bottom);
        const uint32_t n = of_lane(lanes_up_to(above), 63);
        if (n > at)
          lo = mid;
        else
          hi = mid, more = n;
      }
      const uint64_t here = __ballot(hi > bottom && hi <= top);
      const uint32_t rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(here >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)here, 0u));
      who = __ffsll((unsigned long long)__ballot((here >> lane & 1) && rank == at - more)) - 1;
      t.row = (hi - of_lane(bottom, who) - 1) * kRows;
    }
    t.s = Sequence{of_lane(s.first_query, who), of_lane(s.queries, who), of_lane(s.first_key, who), of_lane(s.keys, who), 0};
    t.any = true;
    return t;
  }
  return t;
}

// The first key that a query at position pos sees through a window (0: all). Written so that no window, however long, overflows.
__device__ __forceinline__ int32_t window_start(int32_t pos, uint32_t window) {
  return !window || pos < (int32_t)window ? 0 : pos - (int32_t)window + 1;
}
// The keys [lo, hi) of a tile, from its first row's first to its last row's last.
struct Range {
  int32_t lo, hi;
};
__device__ __forceinline__ Range keys_of(const PromptArgs& a, const Sequence& s, uint32_t row) {
  const int32_t offset = (int32_t)s.keys - (int32_t)s.queries;   // a query's position in its sequence, less its number
  const uint32_t last = min(row + kRows, s.queries * a.nq) - 1;
  const int32_t pos0 = offset + (int32_t)(row / a.nq), pos1 = offset + (int32_t)(last / a.nq);
  return Range{window_start(pos0, a.window), a.causal ? min(pos1 + 1, (int32_t)s.keys) : (int32_t)s.keys};
}

// ------------------------------------------------------------------------------------------------ keys in parts
// Where query tiles are few, or of very different lengths, the keys of a sequence are cut into parts, the same for all of its tiles, and
// a workgroup takes one part of one tile: it leaves maxima, sums and values in the workspace, and prompt_join puts a tile's parts
// together, in their order. Parts of a sequence are numbered part by part and within one tile by tile, so that workgroups that run at the
// same time read the same keys (all tiles as one line, cut into equal runs at keys of their own, found a fifth of their reads in L2: eight
// chunks of up to 500 tokens behind up to 8,000, 245 us without the join, 217 so; with all 240).
struct Cut {   // the workspace's first part: for each sequence, those with the longest parts first
  uint32_t* items;     // [sequences + 1] parts of tiles before its own
  uint32_t* tiles;     // [sequences + 1] tiles before its own
  uint32_t* parts;     // [sequences]
  uint32_t* each;      // [sequences] tiles of keys of a part
  uint32_t* sequence;  // [sequences] its number
  __device__ explicit Cut(const PromptArgs& a)
      : items((uint32_t*)a.ws), tiles(items + a.sequences + 1), parts(tiles + a.sequences + 1), each(parts + a.sequences),
        sequence(each + a.sequences) {}
};
constexpr uint32_t kPartFloats = kPromptRows * (PITCH_DIM + 2);   // [rows][2] maxima and sums, [rows][dim] values
__device__ __forceinline__ float* part_of(const PromptArgs& a, uint32_t head, uint32_t item) {
  return a.ws + a.parts_at + ((uint64_t)item * a.kv_heads + head) * kPartFloats;
}

// Chooses the longest part, of 64 candidates (the longest sequence in 1 .. 64 parts), by an estimate of the time, in sixteenths
// of a tile of keys: all tiles of keys, 2 for each part's beginning and end and kPromptCut for a part of 128 rows that is written and
// joined, over the workgroup places, and half of the longest part for the end, when places run empty; or, where there is a place for
// each part, the longest and, if any are cut, a part's join (five sequences of 100 queries over 600 keys: 35.5 us cut, 26.7 with no cut
// found; 19.8 are the attention alone, in a call whose plan does not look).
__global__ __launch_bounds__(1024) void prompt_cut(PromptArgs a) {
  __shared__ uint32_t sums[2][16], longest, lengths[1024], counts[2][1024];
  __shared__ unsigned long long cost[64], items[64];
  const uint32_t me = threadIdx.x, lane = me & 63, wave = of_wave(me >> 6);
  static_assert(kPromptCutSequences == 1024, "a thread for each sequence");
  const Sequence s = sequence(a, me);
  const uint32_t seen = a.window ? min(s.keys, (uint32_t)min((uint64_t)a.window + kRows, (uint64_t)0x7FFFFFFFu)) : s.keys;
  const uint32_t units = s.tiles ? max((seen + kKeys - 1) / kKeys, 1u) : 0;
  const uint32_t join = kPromptCut * 16 * min(s.queries * a.nq, (uint32_t)kRows) / kRows;
  if (me == 0) longest = 0;
  if (me < 64) cost[me] = items[me] = 0;
  __syncthreads();
  if (units) atomicMax(&longest, units);
  __syncthreads();
  const uint32_t run = max((longest + lane) / (lane + 1), 1u);   // the lane's candidate
  uint64_t my_cost = 0, my_items = 0;
  const uint32_t here = min(max((int32_t)(a.sequences - wave * 64), 0), 64);
  for (uint32_t k = 0; k < here; ++k) {
    const uint32_t u = of_lane(units, k), n = of_lane(s.tiles, k), j = of_lane(join, k);
    if (n == 0) continue;
    const uint32_t parts = (u + run - 1) / run;
    my_items += (uint64_t)n * parts;
    my_cost += (uint64_t)n * (16ull * u + parts * (32ull + (parts > 1 ? j : 0)));
  }
  if (here) {
    atomicAdd(&cost[lane], (unsigned long long)my_cost);
    atomicAdd(&items[lane], (unsigned long long)my_items);
  }
  __syncthreads();
  // the cheapest candidate that the workspace has room for, the same in every wave; uncut is always possible
  float best = items[lane] <= a.places ? 16.f * (float)run + 32.f + (lane ? kPromptCut * 16.f : 0.f)
                                       : (float)cost[lane] / (float)a.places + 8.f * (float)run;
  if (lane > 0 && items[lane] > a.most_items) best = __builtin_inff();
  uint32_t choice = run;
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const float other = __shfl_xor(best, d);
    const uint32_t its = __shfl_xor(choice, d);
    if (other < best || (other == best && its > choice)) best = other, choice = its;
  }
  const uint32_t parts = s.tiles ? (units + choice - 1) / choice : 0, each = parts ? (units + parts - 1) / parts : 0;
  // the sequences by the length of their parts: the shortest come last, when places run empty
  lengths[me] = each;
  __syncthreads();
  uint32_t place = 0;
  for (uint32_t i = 0; i < a.sequences; ++i) place += lengths[i] > each || (lengths[i] == each && i < me);
  const Cut cut(a);
  if (me < a.sequences) {
    counts[0][place] = s.tiles * parts;
    counts[1][place] = s.tiles;
    cut.parts[place] = parts;
    cut.each[place] = each;
    cut.sequence[place] = me;
  }
  __syncthreads();
  uint32_t mine[2], before[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    mine[i] = me < a.sequences ? counts[i][me] : 0;
    const uint32_t x = lanes_up_to(mine[i]);
    if (lane == 63) sums[i][wave] = x;
    before[i] = x - mine[i];
  }
  __syncthreads();
  for (uint32_t w = 0; w < wave; ++w) before[0] += sums[0][w], before[1] += sums[1][w];
  if (me < a.sequences) {
    cut.items[me] = before[0];
    cut.tiles[me] = before[1];
  }
  if (me == a.sequences - 1) {
    cut.items[a.sequences] = before[0] + mine[0];
    cut.tiles[a.sequences] = before[1] + mine[1];
  }
}

// The last sequence with at most `at` items (or tiles) before its own, found by the wave: every 64th sequence, then 64 of them.
__device__ __forceinline__ uint32_t find_sequence(const uint32_t* before, uint32_t sequences, uint32_t at) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t from = 0;
  for (uint32_t step = 64; step; step /= 64) {
    const uint32_t i = from + lane * step;
    from += (max(__popcll(__ballot(i < sequences && before[i] <= at)), 1) - 1) * step;
  }
  return of_wave(from);
}

// Chunks of 16 bytes of a tile's row lie at places that depend on the row: 16 lanes that read the same chunk of 16 rows (keys), or
// 32 that read 64 neighbouring bytes of four rows (values), find 64 banks.
__device__ __forceinline__ uint32_t key_place(uint32_t row, uint32_t chunk) {
  return D == 128 ? chunk ^ (row & 15) : chunk ^ ((row >> 1) & 7);
}
__device__ __forceinline__ uint32_t value_place(uint32_t row, uint32_t chunk) {
  return D == 128 ? chunk ^ ((row & 3) << 2) : chunk ^ ((row & 2) << 1);
}

// w x, where a weight that has become zero leaves what is not finite.
__device__ __forceinline__ float weighed(float w, float x) { return w == 0.f && x - x == 0.f ? 0.f : w == 0.f ? x : w * x; }

// A workgroup's shared memory: two tiles of keys and of values, and whether a result is not finite.
struct Shared {
  __align__(1024) uint8_t tile[2][2][kTileBytes];
  uint32_t odd;
};

// Attention of a query tile over its keys [from, to) of the range that it sees. The results go to the output, or with `part` there.
template <bool MOD>
__device__ __forceinline__ void attend(const PromptArgs& a, Shared& shared, uint32_t head, const Tile& t, Range range, float* part) {
  const uint32_t lane = threadIdx.x & 63, wave = of_wave(threadIdx.x >> 6), half = lane >> 5;
  const int32_t offset = (int32_t)t.s.keys - (int32_t)t.s.queries;
  const uint32_t rows = t.s.queries * a.nq;
  const int32_t lo = range.lo, hi = range.hi;
  const uint32_t ktb = (uint32_t)a.k.token_stride * 2, vtb = (uint32_t)a.v.token_stride * 2;
  const uint8_t* const kbase = (const uint8_t*)a.k.data + head * a.k.head_stride * 2 + (uint64_t)t.s.first_key * ktb;
  const uint8_t* const vbase = (const uint8_t*)a.v.data + head * a.v.head_stride * 2 + (uint64_t)t.s.first_key * vtb;
  const uint32_t load_row = wave * kLaneRows + lane / (D / 8), place = lane % (D / 8);
  const uint32_t koff = load_row * ktb + key_place(load_row, place) * 16;
  const uint32_t voff = load_row * vtb + value_place(load_row, place) * 16;
  // Tiles go from memory straight to LDS. The loads are written out: the compiler, which cannot tell the two halves of the buffer
  // apart, would wait for the next tile before it reads this one.
  auto load_rows = [&](const uint8_t* base, uint32_t stride, uint32_t more, uint32_t at, uint32_t to) {
    const uint64_t p = (uint64_t)base;
    const w4 r = {of_wave((uint32_t)p), of_wave((uint32_t)(p >> 32) & 0xFFFFu), of_wave(more * stride + D * 2), 0x00027000u};
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                   :: "s"(of_wave(to + (i * kWaves + wave) * 1024)), "v"(at + i * kWaves * kLaneRows * stride), "s"(r) : "memory", "m0");
  };
  auto load = [&](int32_t k0, int buf) {
    if (k0 >= hi) return;
    const uint32_t more = (uint32_t)min((int32_t)t.s.keys - k0, kKeys) - 1;  // rows behind the sequence are zeros
    load_rows(kbase + (uint64_t)(uint32_t)k0 * ktb, ktb, more, koff, (uint32_t)(uintptr_t)(lds_u8*)shared.tile[buf][0]);
    load_rows(vbase + (uint64_t)(uint32_t)k0 * vtb, vtb, more, voff, (uint32_t)(uintptr_t)(lds_u8*)shared.tile[buf][1]);
  };
  if (threadIdx.x == 0) shared.odd = 0;
  load(lo, 0);   // (on its way while the queries are read)

  // this lane's row, and the keys [seen_lo, seen_hi] that it sees
  const uint32_t m = t.row + wave * 32 + (lane & 31);
  const bool live = m < rows;
  const uint32_t mm = min(m, rows - 1), token_in = mm / a.nq;
  const uint32_t token_of = t.s.first_query + token_in, head_of = head * a.nq + (mm - token_in * a.nq);
  const int32_t pos = offset + (int32_t)token_in;
  const int32_t seen_hi = a.causal ? min(pos, (int32_t)t.s.keys - 1) : (int32_t)t.s.keys - 1, seen_lo = window_start(pos, a.window);
  w4 q[kSteps];
  float slope = 0.f;
  {
    const uint16_t* const p = (const uint16_t*)a.q.data + token_of * a.q.token_stride + head_of * a.q.head_stride;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) q[s] = *(const w4*)(p + s * 16 + half * 8);
    if (a.negate) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) q[s] ^= 0x80008000u;
    }
    // (used here, so that the compiler waits for them here and not in the loop over the keys, for every tile on its way)
#pragma unroll
    for (int s = 0; s < kSteps; ++s) asm volatile("" : "+v"(q[s]));
    if (MOD && a.slopes) {
      slope = a.slopes[head_of] * 1.44269504088896341f;
      asm volatile("" : "+v"(slope));
    }
  }
  // the wave's rows
  const uint32_t wave_row = t.row + wave * 32, wave_last = min(wave_row + 32, rows) - 1;
  const bool wave_live = wave_row < rows;
  const int32_t whi0 = a.causal ? offset + (int32_t)(wave_row / a.nq) : 0x7FFFFFFF;
  const int32_t wlo1 = window_start(offset + (int32_t)(wave_last / a.nq), a.window);

  v16f o[kBlocks];
  float m_run, mc, sum;

  // Where a lane finds its operands in a tile. Keys: row lane % 32, chunk 2 s + half. Values: of the 16 lanes that a transposing
  // read serves, lanes 4 j .. 4 j + 3 name 16 neighbouring coordinates of key j.
  const uint32_t krow = lane & 31;
  const uint32_t vrow = half * 4 + ((lane >> 2) & 3), vchunk = ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1), vbyte = (lane & 1) * 8;

  auto tile = [&](int32_t k0, int buf, auto careful, uint32_t kind) {
    v16f s[2];
    const lds_u8* const kt = (const lds_u8*)shared.tile[buf][0];
    const lds_u8* const vt = (const lds_u8*)shared.tile[buf][1];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      s[b] = v16f{};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const w4 k = *(const lds_w4*)(kt + (b * 32 + krow) * (D * 2) + key_place(krow, i * 2 + half) * 16);
        s[b] = mfma(k, q[i], s[b]);
      }
    }
    // (the compiler does not see that the statements below read what matrix instructions write: 16 wait states, 12 are needed)
    asm("s_nop 7\n\ts_nop 7" : "+v"(s[0]), "+v"(s[1]));
    if constexpr (MOD) {
      if (a.cap > 0.f) {
        // cap tanh(x) = (cap x) (tanh(x) / x), x = k s. The quotient is a polynomial in s^2 below 0.3 (1.2e-8 off, five instructions
        // with its factors made by the host), in x^2 below 0.55 (6e-9 off, for caps of any size); above that cap (1 - 2 / (e^2x + 1)),
        // which would lose digits to the 1 for small x.
        float big = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) big = fmax3_abs(big, s[0][r], s[1][r]);
        const float k = a.cap_k, pre = a.pre;
        if (!__ballot(big >= a.cap_small)) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float t = s[b][r] * s[b][r];
              s[b][r] *= __builtin_fmaf(t, __builtin_fmaf(t, __builtin_fmaf(t, a.cap_p[2], a.cap_p[1]), a.cap_p[0]), pre);
            }
        } else if (__ballot(big * __builtin_fabsf(k) >= kTanhSplit)) {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const float e = __builtin_amdgcn_exp2f(s[b][r] * a.cap_r);
              const float y = __builtin_fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(e + 1.f), a.cap);
              s[b][r] = __builtin_fabsf(s[b][r] * k) < kTanhSplit ? capped(s[b][r], k, pre) : y;
            }
        } else {
#pragma unroll
          for (int b = 0; b < 2; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) s[b][r] = capped(s[b][r], k, pre);
        }
      } else {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] *= a.pre;
      }
      if (a.slopes) {
        const float away = slope * (float)(int32_t)((uint32_t)k0 + half * 4 - (uint32_t)offset - token_in);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[b][r] += __builtin_fmaf(slope, (float)(b * 32 + (r & 3) + 8 * (r >> 2)), away);
      }
    }
    const bool masked = k0 + kKeys - 1 > whi0 || k0 < wlo1 || k0 + kKeys > (int32_t)t.s.keys;
    if (masked) {
      const int32_t up = seen_hi - k0 - (int32_t)half * 4, down = seen_lo - k0 - (int32_t)half * 4;
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int32_t j = b * 32 + (r & 3) + 8 * (r >> 2);
          if (j > up || j < down) s[b][r] = kNoScore;
        }
    }
    // weights exp2(c (s - m)), with a maximum m that is followed only where scores outgrow it by kGrow
    if (careful && kind) {
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[b][r] = s[b][r] > kNoScore ? 1.f : 0.f;
    } else {
      float top = fmax3_hw(s[0][0], s[1][0], s[0][1]);
      float top2 = fmax3_hw(s[1][1], s[0][2], s[1][2]);
#pragma unroll
      for (int r = 3; r < 15; r += 2) {
        top = fmax3_hw(top, s[0][r], s[1][r]);
        top2 = fmax3_hw(top2, s[0][r + 1], s[1][r + 1]);
      }
      top = fmax_hw(fmax3_hw(top, s[0][15], s[1][15]), top2);
      top = max32(top, top);
      const uint64_t grown = __ballot(__builtin_fmaf(top, a.c, -m_run * a.c) > kGrow);
      float keep = 1.f;
      if (grown) {
        const float next = fmax_hw(m_run, top);
        const float nc = next == kNoScore ? 0.f : next * a.c;
        keep = __builtin_amdgcn_exp2f(__builtin_fmaf(m_run, a.c, -nc));
        sum *= keep;
        m_run = next;
        mc = nc;
      }
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) scale_where(grown, keep, o[d]);
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[b][r], a.c, -mc));
          s[b][r] = w;
          sum += w;
        }
    }
    // the weights, rounded to the values' type: all that is held in fewer bits than float32 here (in two parts of that type they would
    // cost the second product, half of the matrix work, twice); `sum` is that of the weights before it
    w4 p[4];
#pragma unroll
    for (int b = 0; b < 2; ++b)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) p[b * 2 + i][j] = pack2(s[b][i * 8 + j * 2], s[b][i * 8 + j * 2 + 1]);
    // the weights lie as a product's second operand wants them, if its 16 keys are taken in the order 4 h .. 4 h + 3, 8 + 4 h ..
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) {
        w4 v;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint32_t row = i * 16 + u * 8 + vrow;
          const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_s16x4*)(vt + row * (D * 2) + value_place(row, d * 4 + vchunk) * 16 + vbyte));
          const w2 y = __builtin_bit_cast(w2, x);
          v[u * 2] = y[0];
          v[u * 2 + 1] = y[1];
        }
        if constexpr (careful) {
          // kind 0: finite values, others as 0; kinds 1, 2, 3: 1 for NaN, plus infinity, minus infinity, else 0
          constexpr uint32_t inf = PITCH_IO == 1 ? 0x7C00u : 0x7F80u, one = PITCH_IO == 1 ? 0x3C00u : 0x3F80u;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint32_t out = 0;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const uint32_t x = v[j] >> (16 * h) & 0xFFFFu, size = x & 0x7FFFu;
              const uint32_t is = size < inf ? 0u : size > inf ? 1u : x < 0x8000u ? 2u : 3u;
              out |= (kind == 0 ? (is == 0 ? x : 0u) : is == kind ? one : 0u) << (16 * h);
            }
            v[j] = out;
          }
        }
        o[d] = mfma(v, p[i], o[d]);
      }
  };
  // (the first tile is on its way when a pass begins)
  auto pass = [&](auto careful, uint32_t kind) {
    m_run = kNoScore;
    mc = sum = 0.f;
#pragma unroll
    for (int d = 0; d < kBlocks; ++d) o[d] = v16f{};
    int buf = 0;
    if (!wave_live) {   // a wave without rows loads its share for the others
      for (int32_t k0 = lo; k0 < hi; k0 += kKeys, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        load(k0 + kKeys, buf ^ 1);
      }
    } else {
      for (int32_t k0 = lo; k0 < hi; k0 += kKeys, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        load(k0 + kKeys, buf ^ 1);
        tile(k0, buf, careful, kind);
      }
    }
  };

  struct Plain { constexpr operator bool() const { return false; } };
  struct Careful { constexpr operator bool() const { return true; } };
  pass(Plain{}, 0);
  // A value that is not finite reaches every row of a product, also those whose mask hides it (0 * inf). Results that are not finite
  // are therefore computed again: where NaN and infinities are among a row's own values, then the finite values' sum.
  float check[4] = {};
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; ++r) check[r & 3] = __builtin_fmaf(o[d][r], 0.f, check[r & 3]);
  if ((check[0] + check[1]) + (check[2] + check[3]) != 0.f) shared.odd = 1;
  __syncthreads();
  if (shared.odd) {
    uint64_t is[3];
    for (uint32_t kind = 1; kind <= 3; ++kind) {
      __syncthreads();   // (the pass before has read its tiles)
      load(lo, 0);
      pass(Careful{}, kind);
      uint64_t bits = 0;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) bits |= (uint64_t)(o[d][r] > 0.f) << (d * 16 + r);
      if (kind == 1) is[0] = bits;
      if (kind == 2) is[1] = bits;
      if (kind == 3) is[2] = bits;
    }
    __syncthreads();
    load(lo, 0);
    pass(Careful{}, 0);
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = d * 16 + r;
        const bool up = is[1] >> j & 1, down = is[2] >> j & 1;
        if ((is[0] >> j & 1) || (up && down)) o[d][r] = __builtin_nanf("");
        else if (up || down) o[d][r] += up ? __builtin_inff() : -__builtin_inff();
      }
  }

  const float total = fold32(sum, sum);
  if (!wave_live) return;
  if (part) {
    if (live) {
      const uint32_t r = wave * 32 + (lane & 31);
      if (half == 0) {
        part[r * 2] = total == 0.f ? kNoScore : mc;
        part[r * 2 + 1] = total;
      }
      float* const ov = part + kRows * 2 + r * D;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int j = 0; j < 16; j += 4) *(v4f*)(ov + d * 32 + j * 2 + half * 4) = v4f{o[d][j], o[d][j + 1], o[d][j + 2], o[d][j + 3]};
    }
    return;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  if (a.lse && live && half == 0)
    a.lse[(uint64_t)token_of * a.kv_heads * a.nq + head_of] = total == 0.f ? kNoScore : (mc + __builtin_amdgcn_logf(total)) * kLn2;
  uint16_t* const out = (uint16_t*)a.out.data + token_of * a.out.token_stride + head_of * a.out.head_stride;
#pragma unroll
  for (int d = 0; d < kBlocks; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 8) {
      // of 16 coordinates a lane has 0 - 3 and 8 - 11, its partner at distance 32 the others; each stores eight neighbours
      uint32_t x[2], y[2];
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        x[j] = pack2(o[d][r + j * 2] * inv, o[d][r + j * 2 + 1] * inv);
        y[j] = pack2(o[d][r + 4 + j * 2] * inv, o[d][r + 4 + j * 2 + 1] * inv);
        const auto z = __builtin_amdgcn_permlane32_swap(x[j], y[j], false, false);
        x[j] = z[0];
        y[j] = z[1];
      }
      if (live) *(w4*)(out + d * 32 + r * 2 + half * 8) = w4{x[0], x[1], y[0], y[1]};
    }
}

template <bool MOD, bool CUT>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void prompt_attention(PromptArgs a) {
  __shared__ Shared shared;
  // Of the waves that share a SIMD (one of each workgroup on the compute unit) those in odd places go first, so that one's softmax
  // falls together with the other's matrix instructions: 16 sequences in a window 35.3 us without, 31.6 with; chunks 246, 237.
  if (__builtin_amdgcn_s_getreg((3 << 11) | 4) & 1) __builtin_amdgcn_s_setprio(1);   // (the wave's place: four bits of HW_ID)
  const uint32_t head = blockIdx.x % a.kv_heads, number = blockIdx.x / a.kv_heads;
  if constexpr (!CUT) {
    const Tile t = find_tile(a, number);
    if (t.any) attend<MOD>(a, shared, head, t, keys_of(a, t.s, t.row), nullptr);
  } else {
    const Cut cut(a);
    if (number >= cut.items[a.sequences]) return;
    const uint32_t b = find_sequence(cut.items, a.sequences, number), parts = cut.parts[b], rest = number - cut.items[b];
    Tile t{};
    t.s = sequence(a, of_wave(cut.sequence[b]));
    if (t.s.tiles == 0) return;
    const uint32_t part = rest / t.s.tiles;
    if (part >= parts) return;   // (starts that decrease)
    t.row = (t.s.tiles - 1 - (rest - part * t.s.tiles)) * kRows;
    Range r = keys_of(a, t.s, t.row);
    if (parts > 1 && r.lo < r.hi) {   // (unsigned: a part may begin behind the last key)
      const uint32_t each = cut.each[b] * kKeys, from = (uint32_t)r.lo + part * each;
      r.lo = (int32_t)min(from, (uint32_t)r.hi);
      r.hi = (int32_t)min((uint64_t)from + each, (uint64_t)(uint32_t)r.hi);
    }
    attend<MOD>(a, shared, head, t, r, parts > 1 ? part_of(a, head, number) : nullptr);
  }
}

// The parts of a query tile, joined: a lane has four coordinates of a row, a wave as many rows as it has lanes for, so many times one
// after the other. A workgroup's beginning is a chain of five reads, which four turns share where there are workgroups enough (chunks:
// 26 us, with one turn 28 to 33; a join of few rows 7.4 either way, but then a workgroup should not take more than it must).
constexpr uint32_t kRowLanes = D / 4, kWaveRows = 64 / kRowLanes, kJoinRows = 4 * kWaveRows;
__global__ __launch_bounds__(256) void prompt_join(PromptArgs a, uint32_t turns) {
  constexpr uint32_t kDepth = 8;   // parts on their way at once
  const uint32_t lane = threadIdx.x & 63, wave = of_wave(threadIdx.x >> 6);
  const uint32_t blocks = kRows / kJoinRows / turns;   // of a query tile
  const uint32_t head = blockIdx.x % a.kv_heads, rest = blockIdx.x / a.kv_heads, block = rest % blocks, number = rest / blocks;
  const Cut cut(a);
  if (number >= cut.tiles[a.sequences] || cut.items[a.sequences] == cut.tiles[a.sequences]) return;
  const uint32_t b = find_sequence(cut.tiles, a.sequences, number), parts = cut.parts[b];
  if (parts < 2) return;   // its results are in the output
  const Sequence s = sequence(a, of_wave(cut.sequence[b]));
  const uint32_t tile = number - cut.tiles[b], first = cut.items[b] + (s.tiles - 1 - tile);
  if (tile >= s.tiles || first + (parts - 1) * s.tiles >= cut.items[b + 1]) return;   // (starts that decrease)
  const uint32_t left = s.queries * a.nq - tile * kRows;
  for (uint32_t turn = 0; turn < turns; ++turn) {
    const uint32_t row0 = (block * turns + turn) * kJoinRows + wave * kWaveRows;
    if (row0 >= left) return;
    const uint32_t own = min(left - row0, kWaveRows), mine = lane / kRowLanes;   // the wave's rows, the lane's among them
    const uint32_t at = kRows * 2 + (row0 + min(mine, own - 1)) * D + lane % kRowLanes * 4;
    auto part = [&](uint32_t p) { return part_of(a, head, first + p * s.tiles); };
    v4f x[kDepth];
    auto read = [&](uint32_t p) {
#pragma unroll
      for (uint32_t i = 0; i < kDepth; ++i) x[i] = *(const v4f*)(part(min(p + i, parts - 1)) + at);
    };
    read(0);
    // a lane for each part (there are 64 at most): the rows' maxima, sums and weights
    float weight[kWaveRows], sum = 0.f, m = 0.f;
#pragma unroll
    for (uint32_t k = 0; k < kWaveRows; ++k) {
      const uint32_t r = row0 + min(k, own - 1);
      const float top = lane < parts ? part(lane)[r * 2] : kNoScore, total = lane < parts ? part(lane)[r * 2 + 1] : 0.f;
      float most = wave_max(top);
      if (__ballot(top != top)) most = __builtin_nanf("");
      if (most == kNoScore) most = 0.f;
      weight[k] = __builtin_amdgcn_exp2f(top - most);
      const float all = wave_sum(top == kNoScore ? 0.f : weighed(weight[k], total));
      if (mine == k) sum = all, m = most;
    }
    // this row's weight of a part; behind the last part 0
    auto weight_of = [&](uint32_t p) {
      float w = lane_value(weight[0], (int)p);
#pragma unroll
      for (uint32_t k = 1; k < kWaveRows; ++k) w = mine == k ? lane_value(weight[k], (int)p) : w;
      return w;
    };
    v4f o = {};
    for (uint32_t p = 0;;) {
#pragma unroll
      for (uint32_t i = 0; i < kDepth; ++i) {
        const float w = weight_of(p + i);
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] = __builtin_fmaf(w, x[i][d], o[d]);   // (a part that sees no key holds zeros)
      }
      if ((p += kDepth) >= parts) break;
      read(p);
    }
    if (__ballot(((o[0] + o[1]) + (o[2] + o[3])) * 0.f != 0.f)) {   // something is not finite: a weight of zero leaves it so
      o = v4f{};
      for (uint32_t p = 0; p < parts; ++p) {
        const float w = weight_of(p);
        const v4f y = *(const v4f*)(part(p) + at);
#pragma unroll
        for (int d = 0; d < 4; ++d) o[d] += weighed(w, y[d]);
      }
    }
    if (mine >= own) continue;
    const uint32_t row = tile * kRows + row0 + mine, token = row / a.nq, h = head * a.nq + (row - token * a.nq);
    const uint64_t to = s.first_query + token;
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (a.lse && lane % kRowLanes == 0)
      a.lse[to * a.kv_heads * a.nq + h] = sum == 0.f ? kNoScore : (m + __builtin_amdgcn_logf(sum)) * kLn2;
    uint16_t* const out = (uint16_t*)a.out.data + to * a.out.token_stride + h * a.out.head_stride + lane % kRowLanes * 4;
    *(w2*)out = w2{pack2(o[0] * inv, o[1] * inv), pack2(o[2] * inv, o[3] * inv)};
  }
}

}  // namespace

#define PITCH_CAT_(a, b, c, d) a##b##c##d
#define PITCH_CAT(a, b, c, d) PITCH_CAT_(a, b, c, d)
hipError_t PITCH_CAT(launch_prompt_d, PITCH_DIM, _io, PITCH_IO)(const PromptArgs& a, hipStream_t s) {
  const bool mod = a.slopes || a.cap > 0.f;
  if (!a.places) {
    const dim3 grid(a.tiles * a.kv_heads);
    if (mod)
      prompt_attention<true, false><<<grid, dim3(256), 0, s>>>(a);
    else
      prompt_attention<false, false><<<grid, dim3(256), 0, s>>>(a);
    return hipGetLastError();
  }
  prompt_cut<<<dim3(1), dim3(1024), 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 grid((a.tiles > a.most_items ? a.tiles : a.most_items) * a.kv_heads);
  if (mod)
    prompt_attention<true, true><<<grid, dim3(256), 0, s>>>(a);
  else
    prompt_attention<false, true><<<grid, dim3(256), 0, s>>>(a);
  e = hipGetLastError();
  if (e != hipSuccess) return e;
  const uint32_t blocks = a.tiles * a.kv_heads * (kRows / kJoinRows), turns = blocks > 8 * a.places * a.kv_heads ? 4 : 1;
  prompt_join<<<dim3(blocks / turns), dim3(256), 0, s>>>(a, turns);
  return hipGetLastError();
}

}  // namespace pitch
