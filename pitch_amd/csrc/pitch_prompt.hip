// Attention over whole prompts, for one dimension (PITCH_DIM = 64 or 128) and one 16-bit type (PITCH_IO = 1: float16, 2: bfloat16).
#include "pitch_attn_shared.h"
#include "pitch_prompt.h"

#ifndef PITCH_DIM
#error "compile with -DPITCH_DIM=<dim>"
#endif
#ifndef PITCH_IO
#error "compile with -DPITCH_IO=<io type>"
#endif
#ifndef PITCH_PROMPT_NB
#define PITCH_PROMPT_NB 1
#endif

namespace pitch {
namespace {

constexpr int D = PITCH_DIM;
constexpr int kWaves = 4;
constexpr int NB = PITCH_PROMPT_NB;  // blocks of 32 rows of a wave
constexpr int kRows = kWaves * 32 * NB;
constexpr int kKeys = 64;            // keys of a tile
constexpr int kSteps = D / 16;       // steps of the contraction over the coordinates
constexpr int kBlocks = D / 32;      // blocks of 32 output coordinates
constexpr int kTileBytes = kKeys * D * 2;
constexpr int kLaneRows = 1024 / (D * 2);            // rows of a tile that a wave loads at once
constexpr int kLoads = kKeys / (kLaneRows * kWaves); // loads of a wave for a tile of keys or values
constexpr float kGrow = 8.f;         // log2 units that a row's scores may exceed the maximum in use by
constexpr float kNoScore = -__builtin_inff();

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

// x *= f where `go` is not zero. The branch is inside the statement: with one around it, the compiler keeps two copies of the
// accumulators and moves them, 64 registers there and back for every tile (2,190 us of a prompt of 16,381 tokens, 8 KV and 32 query heads; XXX without).
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

// A query tile: the rows [row, row + kRows) of (token, head) pairs of a sequence.
struct Tile {
  uint32_t first_query, queries;  // the sequence's
  uint32_t first_key, keys;
  uint32_t row;
  bool any;
};

// The sequence of tile number `at`, found by all of the waves alike; a sequence's last tile, whose rows see most, comes first.
__device__ __forceinline__ Tile find_tile(const PromptArgs& a, uint32_t at) {
  const uint32_t lane = threadIdx.x & 63;
  Tile t{};
  for (uint32_t base = 0; base < a.sequences; base += 64) {
    const uint32_t b = base + lane;
    uint32_t n = 0, q0 = 0;
    if (b < a.sequences) {
      const int32_t lo = a.row_starts[b], hi = a.row_starts[b + 1];
      q0 = min((uint32_t)max(lo, 0), a.rows);
      n = max((int32_t)(min((uint32_t)max(hi, 0), a.rows) - q0), 0);
    }
    const uint32_t tiles = (n * a.nq + kRows - 1) / kRows;
    uint32_t sum = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint32_t up = __shfl_up(sum, d);
      if (lane >= (uint32_t)d) sum += up;
    }
    const uint32_t total = of_wave(__shfl(sum, 63));
    if (at < total) {
      const int who = __ffsll((unsigned long long)__ballot(sum > at)) - 1;
      t.any = true;
      t.first_query = of_wave(__shfl(q0, who));
      t.queries = of_wave(__shfl(n, who));
      t.row = (of_wave(__shfl(sum, who)) - 1 - at) * kRows;
      const int32_t lo = a.key_starts[base + who], hi = a.key_starts[base + who + 1];
      t.first_key = min((uint32_t)max(lo, 0), a.keys);
      t.keys = max((int32_t)(min((uint32_t)max(hi, 0), a.keys) - t.first_key), 0);
      return t;
    }
    at -= total;
  }
  return t;
}

// Chunks of 16 bytes of a tile's row lie at places that depend on the row: 16 lanes that read the same chunk of 16 rows (keys), or
// 32 that read 64 neighbouring bytes of four rows (values), find 64 banks.
__device__ __forceinline__ uint32_t key_place(uint32_t row, uint32_t chunk) {
  return D == 128 ? chunk ^ (row & 15) : chunk ^ ((row >> 1) & 7);
}
__device__ __forceinline__ uint32_t value_place(uint32_t row, uint32_t chunk) {
  return D == 128 ? chunk ^ ((row & 3) << 2) : chunk ^ ((row & 2) << 1);
}

// The first key that a query at position pos sees through a window (0: all). Written so that no window, however long, overflows.
__device__ __forceinline__ int32_t window_start(int32_t pos, uint32_t window) {
  return !window || pos < (int32_t)window ? 0 : pos - (int32_t)window + 1;
}

template <bool MOD>
__global__ __launch_bounds__(256, NB == 1 ? 2 : 1) void prompt_attention(PromptArgs a) {
  __shared__ __align__(1024) uint8_t lds[2][2][kTileBytes];
  __shared__ uint32_t odd;
  const uint32_t head = blockIdx.x % a.kv_heads, part = blockIdx.x / a.kv_heads % a.splits;
  const Tile t = find_tile(a, blockIdx.x / (a.kv_heads * a.splits));
  if (!t.any) return;
  const uint32_t lane = threadIdx.x & 63, wave = of_wave(threadIdx.x >> 6), half = lane >> 5;
  const int32_t offset = (int32_t)t.keys - (int32_t)t.queries;  // a query's position in its sequence, less its number
  const uint32_t rows = t.queries * a.nq;

  // the rows of this lane, and the keys [lo, hi] that they see
  int32_t seen_hi[NB], seen_lo[NB];
  uint64_t q_at[NB], o_at[NB];
  uint32_t head_of[NB], token_of[NB];
  bool live[NB];
  w4 q[NB][kSteps];
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const uint32_t m = t.row + (wave * NB + n) * 32 + (lane & 31);
    live[n] = m < rows;
    const uint32_t mm = min(m, rows - 1), token = mm / a.nq;
    token_of[n] = t.first_query + token;
    head_of[n] = head * a.nq + (mm - token * a.nq);
    const int32_t pos = offset + (int32_t)token;
    seen_hi[n] = a.causal ? min(pos, (int32_t)t.keys - 1) : (int32_t)t.keys - 1;
    seen_lo[n] = window_start(pos, a.window);
    const uint16_t* const p = (const uint16_t*)a.q.data + token_of[n] * a.q.token_stride + head_of[n] * a.q.head_stride;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      q[n][s] = *(const w4*)(p + s * 16 + half * 8);
      if (a.negate) q[n][s] ^= 0x80008000u;
    }
  }
  // the tile's keys, from its first row's first to its last row's last
  const uint32_t last_row = min(t.row + kRows, rows) - 1;
  const int32_t pos0 = offset + (int32_t)(t.row / a.nq), pos1 = offset + (int32_t)(last_row / a.nq);
  int32_t lo = window_start(pos0, a.window);
  int32_t hi = a.causal ? min(pos1 + 1, (int32_t)t.keys) : (int32_t)t.keys;
  if (a.splits > 1 && lo < hi) {   // (unsigned: the last parts may begin behind the last key)
    const uint32_t each = (((uint32_t)(hi - lo) + a.splits - 1) / a.splits + kKeys - 1) / kKeys * kKeys;
    const uint32_t from = (uint32_t)lo + part * each;
    lo = (int32_t)min(from, (uint32_t)hi);
    hi = (int32_t)min(from + each, (uint32_t)hi);
  }
  // the wave's own rows
  const uint32_t wave_row = t.row + wave * NB * 32, wave_last = min(wave_row + NB * 32, rows) - 1;
  const bool wave_live = wave_row < rows;
  const int32_t wpos0 = offset + (int32_t)(wave_row / a.nq), wpos1 = offset + (int32_t)(wave_last / a.nq);
  const int32_t whi0 = a.causal ? wpos0 : 0x7FFFFFFF, wlo1 = window_start(wpos1, a.window);

  const uint32_t ktb = (uint32_t)a.k.token_stride * 2, vtb = (uint32_t)a.v.token_stride * 2;
  const uint8_t* const kbase = (const uint8_t*)a.k.data + head * a.k.head_stride * 2 + (uint64_t)t.first_key * ktb;
  const uint8_t* const vbase = (const uint8_t*)a.v.data + head * a.v.head_stride * 2 + (uint64_t)t.first_key * vtb;
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
                   :: "s"(of_wave(to + (i * kWaves + wave) * 1024)), "v"(at + i * kWaves * kLaneRows * stride), "s"(r) : "memory");
  };
  auto load = [&](int32_t k0, int buf) {
    const uint32_t more = (uint32_t)min((int32_t)t.keys - k0, kKeys) - 1;  // rows behind the sequence are zeros
    load_rows(kbase + (uint64_t)(uint32_t)k0 * ktb, ktb, more, koff, (uint32_t)(uintptr_t)(lds_u8*)lds[buf][0]);
    load_rows(vbase + (uint64_t)(uint32_t)k0 * vtb, vtb, more, voff, (uint32_t)(uintptr_t)(lds_u8*)lds[buf][1]);
  };

  v16f o[NB][kBlocks];
  float m_run[NB], mc[NB], sum[NB];

  // Where a lane finds its operands in a tile. Keys: row lane % 32, chunk 2 s + half. Values: of the 16 lanes that a transposing
  // read serves, lanes 4 j .. 4 j + 3 name 16 neighbouring coordinates of key j.
  const uint32_t krow = lane & 31;
  const uint32_t vrow = half * 4 + ((lane >> 2) & 3), vchunk = ((lane >> 4) & 1) * 2 + ((lane >> 1) & 1), vbyte = (lane & 1) * 8;

  auto tile = [&](int32_t k0, int buf, auto careful, uint32_t kind) {
    v16f s[NB][2];
    const lds_u8* const kt = (const lds_u8*)lds[buf][0];
    const lds_u8* const vt = (const lds_u8*)lds[buf][1];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
      for (int n = 0; n < NB; ++n) s[n][b] = v16f{};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const w4 k = *(const lds_w4*)(kt + (b * 32 + krow) * (D * 2) + key_place(krow, i * 2 + half) * 16);
#pragma unroll
        for (int n = 0; n < NB; ++n) s[n][b] = mfma(k, q[n][i], s[n][b]);
      }
    }
    if constexpr (MOD) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const float slope = a.slopes ? a.slopes[head_of[n]] * 1.44269504088896341f : 0.f;
        const int32_t away = (int32_t)((uint32_t)k0 + half * 4 - (uint32_t)offset - (token_of[n] - t.first_query));
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            float z = s[n][b][r] * a.pre;
            if (a.cap > 0.f) {
              // tanh(x) = sign(x) (1 - 2 / (e^2|x| + 1))
              const float e = __builtin_amdgcn_exp2f(__builtin_fabsf(z) * a.cap_r);
              z = __builtin_copysignf(__builtin_fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(e + 1.f), a.cap), z);
            }
            s[n][b][r] = __builtin_fmaf(slope, (float)(away + b * 32 + (r & 3) + 8 * (r >> 2)), z);
          }
      }
    }
    const bool masked = k0 + kKeys - 1 > whi0 || k0 < wlo1 || k0 + kKeys > (int32_t)t.keys;
    if (masked) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        const int32_t up = seen_hi[n] - k0 - (int32_t)half * 4, down = seen_lo[n] - k0 - (int32_t)half * 4;
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int32_t j = b * 32 + (r & 3) + 8 * (r >> 2);
            if (j > up || j < down) s[n][b][r] = kNoScore;
          }
      }
    }
    // weights exp2(c (s - m)), with a maximum m that is followed only where scores outgrow it by kGrow
    w4 p[NB][4];
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      if constexpr (careful) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (kind) s[n][b][r] = s[n][b][r] > kNoScore ? 1.f : 0.f;
      }
      if (!careful || !kind) {
        // (the compiler does not see that the maxima below read what matrix instructions write: 16 wait states, 11 are needed)
        asm("s_nop 7\n\ts_nop 7" : "+v"(s[n][0]), "+v"(s[n][1]));
        float top = fmax3_hw(s[n][0][0], s[n][1][0], s[n][0][1]);
        float top2 = fmax3_hw(s[n][1][1], s[n][0][2], s[n][1][2]);
#pragma unroll
        for (int r = 3; r < 15; r += 2) {
          top = fmax3_hw(top, s[n][0][r], s[n][1][r]);
          top2 = fmax3_hw(top2, s[n][0][r + 1], s[n][1][r + 1]);
        }
        top = fmax3_hw(top, s[n][0][15], s[n][1][15]);
        top = max32(fmax_hw(top, top2), fmax_hw(top, top2));
        const uint64_t grown = __ballot(__builtin_fmaf(top, a.c, -m_run[n] * a.c) > kGrow);
        float keep = 1.f;
        if (grown) {
          const float next = fmax_hw(m_run[n], top);
          const float nc = next == kNoScore ? 0.f : next * a.c;
          keep = __builtin_amdgcn_exp2f(__builtin_fmaf(m_run[n], a.c, -nc));
          sum[n] *= keep;
          m_run[n] = next;
          mc[n] = nc;
        }
#pragma unroll
        for (int d = 0; d < kBlocks; ++d) scale_where(grown, keep, o[n][d]);
#pragma unroll
        for (int b = 0; b < 2; ++b)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float w = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][b][r], a.c, -mc[n]));
            s[n][b][r] = w;
            sum[n] += w;
          }
      }
#pragma unroll
      for (int b = 0; b < 2; ++b)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) p[n][b * 2 + i][j] = pack2(s[n][b][i * 8 + j * 2], s[n][b][i * 8 + j * 2 + 1]);
    }
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
#pragma unroll
        for (int n = 0; n < NB; ++n) o[n][d] = mfma(v, p[n][i], o[n][d]);
      }
  };
  auto pass = [&](auto careful, uint32_t kind) {
#pragma unroll
    for (int n = 0; n < NB; ++n) {
      m_run[n] = kNoScore;
      mc[n] = sum[n] = 0.f;
#pragma unroll
      for (int d = 0; d < kBlocks; ++d) o[n][d] = v16f{};
    }
    if (lo >= hi) return;
    load(lo, 0);
    int buf = 0;
    if (!wave_live) {   // a wave without rows loads its share for the others
      for (int32_t k0 = lo; k0 < hi; k0 += kKeys, buf ^= 1) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
        if (k0 + kKeys < hi) load(k0 + kKeys, buf ^ 1);
      }
      __syncthreads();
      return;
    }
    for (int32_t k0 = lo; k0 < hi; k0 += kKeys, buf ^= 1) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads();
      if (k0 + kKeys < hi) load(k0 + kKeys, buf ^ 1);
      tile(k0, buf, careful, kind);
    }
    __syncthreads();
  };

  struct Plain { constexpr operator bool() const { return false; } };
  struct Careful { constexpr operator bool() const { return true; } };
  if (threadIdx.x == 0) odd = 0;
  pass(Plain{}, 0);
  // A value that is not finite reaches every row of a product, also those whose mask hides it (0 * inf). Results that are not finite
  // are therefore computed again: where NaN and infinities are among a row's own values, then the finite values' sum.
  float check = 0.f;
#pragma unroll
  for (int n = 0; n < NB; ++n)
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; ++r) check = __builtin_fmaf(o[n][d][r], 0.f, check);
  if (lo >= hi) __syncthreads();
  if (check != 0.f) odd = 1;
  __syncthreads();
  if (odd) {
    uint64_t is[3][NB];
    for (uint32_t kind = 1; kind <= 3; ++kind) {
      pass(Careful{}, kind);
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        uint64_t bits = 0;
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) bits |= (uint64_t)(o[n][d][r] > 0.f) << (d * 16 + r);
        if (kind == 1) is[0][n] = bits;
        if (kind == 2) is[1][n] = bits;
        if (kind == 3) is[2][n] = bits;
      }
    }
    pass(Careful{}, 0);
#pragma unroll
    for (int n = 0; n < NB; ++n)
#pragma unroll
      for (int d = 0; d < kBlocks; ++d)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = d * 16 + r;
          const bool up = is[1][n] >> j & 1, down = is[2][n] >> j & 1;
          if ((is[0][n] >> j & 1) || (up && down)) o[n][d][r] = __builtin_nanf("");
          else if (up || down) o[n][d][r] += up ? __builtin_inff() : -__builtin_inff();
        }
  }

  if (!wave_live) return;
#pragma unroll
  for (int n = 0; n < NB; ++n) {
    const float total = fold32(sum[n], sum[n]);
    if (a.splits > 1) {
      // (maximum, sum, values) of the part, values by output coordinate
      const uint64_t heads = (uint64_t)a.kv_heads * a.nq, at = (uint64_t)token_of[n] * heads + head_of[n], all = (uint64_t)a.rows * heads;
      float* const ms = a.ws + (part * all + at) * 2;
      float* const ov = a.ws + (uint64_t)a.splits * all * 2 + (part * all + at) * D;
      if (live[n]) {
        if (half == 0) {
          ms[0] = total == 0.f ? kNoScore : mc[n];
          ms[1] = total;
        }
#pragma unroll
        for (int d = 0; d < kBlocks; ++d)
#pragma unroll
          for (int r = 0; r < 16; r += 4) *(v4f*)(ov + d * 32 + r * 2 + half * 4) = v4f{o[n][d][r], o[n][d][r + 1], o[n][d][r + 2], o[n][d][r + 3]};
      }
      continue;
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    if (a.lse && live[n] && half == 0)
      a.lse[(uint64_t)token_of[n] * a.kv_heads * a.nq + head_of[n]] = total == 0.f ? kNoScore : (mc[n] + __builtin_amdgcn_logf(total)) * kLn2;
    uint16_t* const out = (uint16_t*)a.out.data + token_of[n] * a.out.token_stride + head_of[n] * a.out.head_stride;
#pragma unroll
    for (int d = 0; d < kBlocks; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 8) {
        // of 16 coordinates a lane has 0 - 3 and 8 - 11, its partner at distance 32 the others; each stores eight neighbours
        uint32_t x[2], y[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          x[j] = pack2(o[n][d][r + j * 2] * inv, o[n][d][r + j * 2 + 1] * inv);
          y[j] = pack2(o[n][d][r + 4 + j * 2] * inv, o[n][d][r + 4 + j * 2 + 1] * inv);
          const auto z = __builtin_amdgcn_permlane32_swap(x[j], y[j], false, false);
          x[j] = z[0];
          y[j] = z[1];
        }
        if (live[n]) *(w4*)(out + d * 32 + r * 2 + half * 8) = w4{x[0], x[1], y[0], y[1]};
      }
  }
}

// The parts of split keys, joined: one wave for each row of (token, head), parts in their order.
__global__ __launch_bounds__(256) void prompt_join(PromptArgs a) {
  const uint64_t heads = (uint64_t)a.kv_heads * a.nq, all = (uint64_t)a.rows * heads;
  const uint64_t at = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= all) return;
  const uint32_t lane = threadIdx.x & 63, token = (uint32_t)(at / heads), head = (uint32_t)(at % heads);
  // a token of no sequence has no result
  bool inside = false;
  for (uint32_t b = lane; b < a.sequences; b += 64)
    inside |= (int32_t)token >= a.row_starts[b] && (int32_t)token < a.row_starts[b + 1];
  if (!__ballot(inside)) return;
  // a lane for each part (64 at most): its maximum and its sum
  const bool part = lane < a.splits;
  const float mine = part ? a.ws[(lane * all + at) * 2] : kNoScore, mine_sum = part ? a.ws[(lane * all + at) * 2 + 1] : 0.f;
  const bool nan = __ballot(mine != mine) != 0;
  float m = wave_max(mine);
  if (m == kNoScore) m = 0.f;
  const float weight = nan ? __builtin_nanf("") : __builtin_amdgcn_exp2f(mine - m);
  const float sum = wave_sum(weight == 0.f ? 0.f : weight * mine_sum);
  float o[D / 64] = {};
  const float* const ov = a.ws + (uint64_t)a.splits * all * 2;
  // (parts without a visible key have not written values that count)
  for (uint64_t todo = __ballot(part && weight != 0.f); todo;) {
    float w[8], x[8][D / 64];
#pragma unroll
    for (int i = 0; i < 8; ++i) {   // eight parts on their way at once
      w[i] = 0.f;
      if (!todo) continue;
      const int p = __ffsll((unsigned long long)todo) - 1;
      todo &= todo - 1;
      w[i] = lane_value(weight, p);
#pragma unroll
      for (int d = 0; d < D / 64; ++d) x[i][d] = ov[(p * all + at) * D + lane * (D / 64) + d];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int d = 0; d < D / 64; ++d)
        if (w[i] != 0.f) o[d] = __builtin_fmaf(w[i], x[i][d], o[d]);
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (a.lse && lane == 0) a.lse[at] = sum == 0.f ? kNoScore : (m + __builtin_amdgcn_logf(sum)) * kLn2;
  uint16_t* const out = (uint16_t*)a.out.data + token * a.out.token_stride + head * a.out.head_stride + lane * (D / 64);
  if constexpr (D == 128)
    *(uint32_t*)out = pack2(o[0] * inv, o[1] * inv);
  else
    *out = (uint16_t)pack2(o[0] * inv, 0.f);
}

}  // namespace

#define PITCH_CAT_(a, b, c, d) a##b##c##d
#define PITCH_CAT(a, b, c, d) PITCH_CAT_(a, b, c, d)
hipError_t PITCH_CAT(launch_prompt_d, PITCH_DIM, _io, PITCH_IO)(const PromptArgs& a, hipStream_t s) {
  const uint64_t groups = (uint64_t)a.tiles * a.kv_heads * a.splits;
  if (a.slopes || a.cap > 0.f)
    prompt_attention<true><<<dim3((uint32_t)groups), dim3(256), 0, s>>>(a);
  else
    prompt_attention<false><<<dim3((uint32_t)groups), dim3(256), 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.splits == 1) return e;
  const uint64_t rows = (uint64_t)a.rows * a.kv_heads * a.nq;
  prompt_join<<<dim3((uint32_t)((rows + 3) / 4)), dim3(256), 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace pitch
