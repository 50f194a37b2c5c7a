// The paged cache's writes and reads for one dimension (PITCH_DIM = 64 or 128) and one element type of the vectors
// (PITCH_IO): paged_append quantises a step's keys and values into the slots of a pool's pages, with the queries' and
// keys' norms and position rotation in the same pass; paged_decode reads ranges of tokens back through page tables.
//
// A vector is held by a team of D / 8 lanes, eight neighbouring coordinates each: one 16-byte load or store of 16-bit
// elements per lane, and the eight codes of a lane are `bits` whole bytes of the vector's row, whatever the width, so
// every width runs one body with the width as a wave-uniform value.
#include "pitch_device.h"
#include "pitch_paged.h"

#ifndef PITCH_DIM
#error "compile with -DPITCH_DIM=<dim>"
#endif
#ifndef PITCH_IO
#error "compile with -DPITCH_IO=<io>"
#endif

namespace pitch {
namespace {

constexpr int D = PITCH_DIM, IO = PITCH_IO, T = D / 8;
constexpr int V = 64 / T;                 // vectors of a wave
constexpr int VPB = V * (kBlock / 64);    // vectors of a workgroup's pass
constexpr double kInvSqrtD = D == 64 ? 0.125 : 0x1.6a09e667f3bcdp-4;
static_assert(D == 64 || D == 128, "dimensions of the paged cache");

typedef uint16_t u16_any __attribute__((aligned(1)));
typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint64_t u64_any __attribute__((aligned(1)));

// This lane's eight rotation signs.
__device__ __forceinline__ uint32_t lane_signs(const PagedPool& p, int t) {
  const uint32_t w = D == 64 ? (t < 4 ? p.signs[0] : p.signs[1])
                             : (t < 8 ? (t < 4 ? p.signs[0] : p.signs[1]) : (t < 12 ? p.signs[2] : p.signs[3]));
  return w >> (8 * (t & 3));
}

// The low `bytes` (2 .. 8, uniform) bytes of w.
__device__ __forceinline__ void store_bytes(uint8_t* p, uint64_t w, uint32_t bytes) {
  const uint32_t lo = (uint32_t)w, hi = (uint32_t)(w >> 32);
  switch (bytes) {
    case 2: *(u16_any*)p = (uint16_t)lo; break;
    case 3: *(u16_any*)p = (uint16_t)lo; p[2] = (uint8_t)(lo >> 16); break;
    case 4: *(u32_any*)p = lo; break;
    case 5: *(u32_any*)p = lo; p[4] = (uint8_t)hi; break;
    case 6: *(u32_any*)p = lo; *(u16_any*)(p + 4) = (uint16_t)hi; break;
    case 7: *(u32_any*)p = lo; *(u16_any*)(p + 4) = (uint16_t)hi; p[6] = (uint8_t)(hi >> 16); break;
    default: *(u64_any*)p = w; break;
  }
}

// ----------------------------------------------------------------------------------------------------
// Append. Keys and values are normed, rotated to their positions and transformed in float64, which on this hardware costs
// what float32 costs, so a code is that of the exact vector unless a value lies within 1e-15 of an edge: the write does not
// depend on how the work is split. The norm's factor 1 / rms multiplies every coordinate alike: it changes no code and only
// scales the stored norm (TurboQuant) or largest radius (PolarQuant). Queries are computed in float32 and rounded once.
// A team takes one token and H of its heads: the token's weights and rotation are read and multiplied once, all heads are
// loaded at once, and a rotation's partner coordinates come from their lane. Bound by arithmetic beside the copies: 8,191
// tokens of 8 KV and 32 query heads (d = 128 bf16, norms, full rotation, 4 bits), 185 MB, take 48 us (3.9 TB/s); the queries
// alone 36, keys and values alone 28. One token 4.8 us, 64 tokens 4.9. (Times in this file are those of a call among others.)

// 1 / sqrt(x) of a normal positive x, to 2^-51: the hardware's estimate and two steps of Newton's, a third of what a division by
// the correctly rounded root takes.
__device__ __forceinline__ double inv_sqrt(double x) {
  const double h = 0.5 * x;
  double r = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) r = __builtin_fma(r, __builtin_fma(-(h * r), r, 0.5), r);
  return r;
}
// The same in float32, to 2^-23 (the hardware's, which takes no subnormal numbers).
__device__ __forceinline__ float inv_sqrt(float x) {
  const bool tiny = x < 0x1p-96f;
  return __builtin_amdgcn_rsqf(tiny ? x * 0x1p96f : x) * (tiny ? 0x1p48f : 1.f);
}

// Eight coordinates as they lie in memory.
constexpr int kRawWords = IO == 0 ? 8 : 4;
struct Raw {
  uint32_t w[kRawWords];
};
__device__ __forceinline__ Raw load_raw(const void* base, uint64_t i) {
  Raw r;
#pragma unroll
  for (int k = 0; k < kRawWords; k += 4) {
    const u32x4 v = *(const u32x4*)((const char*)base + i * Io<IO>::kBytes + 4 * k);
    r.w[k] = v.x; r.w[k + 1] = v.y; r.w[k + 2] = v.z; r.w[k + 3] = v.w;
  }
  return r;
}
__device__ __forceinline__ void widen(const Raw& r, float (&f)[8]) {
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    if constexpr (IO == 0) f[k] = __uint_as_float(r.w[k]);
    else if (k % 2 == 0) widen2<IO>(r.w[k / 2], f[k], f[k + 1]);
  }
}

// The norm's weights and the rotation of one token, for this lane's coordinates: y = own . x + other . x of the partner lane.
template <typename F>
struct Turn {
  F own[8], other[8];
  int partner;    // lane (times 4) that holds the coordinates turned with these
  bool scaled, turned;   // uniform: weights or a rotation are given; this lane's coordinates are rotated

  __device__ __forceinline__ void set(const PagedAppendArgs& a, const void* weight, uint64_t pos, int lane, int t) {
    const uint32_t half = a.rotary / 16;   // in lanes
    scaled = weight || a.positions;
    turned = a.positions && 2u * half > (uint32_t)t;
    const int pt = turned ? ((uint32_t)t < half ? t + (int)half : t - (int)half) : t;
    partner = (lane - t + pt) * 4;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      own[e] = F(1);
      other[e] = F(0);
    }
    if (weight) {
      float f[8];
      load_elems<IO, 8>(weight, 8u * t, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) own[e] = (F)f[e];
    }
    if (turned) {
      float c[8], s[8], f[8];
      load_elems<0, 8>(a.cos, pos * a.rotary + 8u * t, c);
      load_elems<0, 8>(a.sin, pos * a.rotary + 8u * t, s);
      if (weight) load_elems<IO, 8>(weight, 8u * pt, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        own[e] *= (F)c[e];
        other[e] = (uint32_t)t < half ? -(F)s[e] : (F)s[e];
        if (weight) other[e] *= (F)f[e];
      }
    }
  }
  // ss = sum of the x^2 over the vector (where norm).
  __device__ __forceinline__ void apply(const Raw& r, bool norm, F (&y)[8], F& ss) const {
    float f[8];
    widen(r, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (F)f[e];
    if (norm) {
      ss = F(0);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fma_t(y[e], y[e], ss);
      ss = team_reduce<T>(ss, [](F p, F q) { return p + q; });
    }
    if (!scaled) return;
    Raw o;
#pragma unroll
    for (int k = 0; k < kRawWords; ++k) o.w[k] = (uint32_t)__builtin_amdgcn_ds_bpermute(partner, (int)r.w[k]);
    widen(o, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const F u = y[e] * own[e];
      y[e] = turned ? fma_t((F)f[e], other[e], u) : u;
    }
  }
};

// The radius and angle codes of a pair near a rounding point, in float64 and the definition's order (see
// polar_codes_exact in pitch_vector.hip; here the number of levels is a run-time value).
__device__ __attribute__((noinline)) uint32_t polar_pair_exact(double a, double c, double r2, double safe, uint32_t levels) {
  const double top = (double)(levels - 1);
  double rq = __builtin_floor(__builtin_sqrt(r2) / safe * top + 0.5);
  rq = rq < 0.0 ? 0.0 : (rq > top ? top : rq);
  double th = atan2(c, a);
  if (th < 0.0) th += kTwoPi;
  const double tq = __builtin_floor(th / kTwoPi * (double)levels + 0.5);
  return (uint32_t)rq | (((uint32_t)tq & (levels - 1)) << 8);
}

// Eight codes of p.bits bits each as the bytes of a row.
__device__ __forceinline__ uint64_t pack(const uint32_t (&c)[8], uint32_t bits) {
  uint32_t lo = c[0], hi = c[4];
#pragma unroll
  for (int e = 1; e < 4; ++e) {
    lo |= c[e] << (bits * e);
    hi |= c[4 + e] << (bits * e);
  }
  return (uint64_t)lo | (uint64_t)hi << (4 * bits);
}

// The codes of this lane's eight coordinates of a vector, given in float64 times their signs; scale = the vector's scale.
template <bool POLAR>
__device__ __forceinline__ uint64_t quantise(const PagedPool& p, double (&y)[8], int t, const uint2* s_lut, double& scale) {
  uint32_t codes[8];
  if (!POLAR || !p.polar) {
    double n2 = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) n2 = __builtin_fma(y[e], y[e], n2);
    n2 = team_reduce<T>(n2, [](double x, double z) { return x + z; });
    const bool some = n2 > 0.0 && n2 < (double)__builtin_inf();
    const double inv = some ? inv_sqrt(n2) : 1.0, us = inv * kInvSqrtD;
    scale = some ? n2 * inv : n2;
    fwht_contig<8, T, double>(y, t);
    // bucket u * 2^m + off holds at most one edge: code = edges below the bucket + [u > edge]
    const double um = us * p.lut_scale;
    uint2 entry[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = (int)__builtin_fma(y[e], um, p.lut_off);
      entry[e] = s_lut[min(max(j, 0), p.lut_entries - 1)];
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      codes[e] = entry[e].y + (y[e] * us > (double)__uint_as_float(entry[e].x) ? 1u : 0u);
    }
    return pack(codes, p.bits);
  }
  fwht_contig<8, T, double>(y, t);
  double r2[4], top = 0.0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    r2[q] = __builtin_fma(y[2 * q], y[2 * q], y[2 * q + 1] * y[2 * q + 1]);
    top = r2[q] <= top ? top : r2[q];   // (NaN is kept: every transformed coordinate of a vector that is not finite is infinite or NaN)
  }
  top = team_reduce<T>(top, [](double x, double z) { return x <= z ? z : x; });
  const double rmax = __builtin_sqrt(top), safe = rmax > 0.0 ? rmax : 1.0, inv = 1.0 / safe;
  scale = rmax * kInvSqrtD;
  const uint32_t levels = 1u << p.bits;
  const float fl = (float)levels;
  uint32_t code[4], need = 0u;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    // float32 on the pair relative to the largest radius; what lies near a rounding point is decided in float64
    const float af = (float)(y[2 * q] * inv), cf = (float)(y[2 * q + 1] * inv);
    const float rf = __builtin_amdgcn_sqrtf(__builtin_fmaf(af, af, cf * cf));
    bool ok = r2[q] > 0.0;
    const float kr = guarded_floor(__builtin_fmaf(rf, fl - 1.f, 0.5f), ok);
    const float ka = guarded_floor(__builtin_fmaf(angle_turns<8>(cf, af), fl, 0.5f), ok);
    code[q] = min((uint32_t)kr, levels - 1) | (((uint32_t)ka & (levels - 1)) << 8);
    need |= ok ? 0u : 1u << q;
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    if (need & (1u << q)) code[q] = polar_pair_exact(y[2 * q], y[2 * q + 1], r2[q], safe, levels);
    codes[2 * q] = code[q] & 255u;
    codes[2 * q + 1] = code[q] >> 8;
  }
  return pack(codes, p.bits);
}

// A team's token and its H heads from head on.
struct Item {
  uint32_t token, head;
  bool any;
  __device__ __forceinline__ Item(uint32_t block, int team, uint32_t tokens, uint32_t heads, int h) {
    const uint32_t groups = (heads + h - 1) / h, count = tokens * groups, nominal = block * VPB + (uint32_t)team;
    const uint32_t v = min(nominal, count - 1);
    any = nominal < count;
    token = v / groups;
    head = (v - token * groups) * h;
  }
};
template <int H>
__device__ __forceinline__ void load_heads(const PagedVectors& in, const Item& it, uint32_t heads, int t, Raw (&x)[H]) {
#pragma unroll
  for (int n = 0; n < H; ++n)
    x[n] = load_raw(in.data, it.token * in.token_stride + min(it.head + n, heads - 1) * in.head_stride + 8u * t);
}
// The token's row of the rotation tables; false if it lies outside them.
__device__ __forceinline__ bool position_of(const PagedAppendArgs& a, uint32_t token, uint64_t& pos) {
  pos = 0;
  if (!a.positions) return true;
  pos = (uint64_t)a.positions[token];
  const bool ok = pos < a.table_rows;
  pos = ok ? pos : 0;
  return ok;
}

// Keys (normed and rotated) or values.
template <int H, bool POLAR, bool KEYS>
__device__ __forceinline__ void append_vectors(const PagedAppendArgs& a, uint32_t block, uint2* s_lut) {
  const PagedPool& p = a.pool[KEYS ? 0 : 1];
  const int tid = threadIdx.x, lane = tid & 63, t = lane & (T - 1);
  const uint32_t heads = a.layout.kv_heads;
  const Item it(block, (tid >> 6) * V + lane / T, a.tokens, heads, H);
  Raw x[H];
  load_heads<H>(a.in[KEYS ? 0 : 1], it, heads, t, x);
  const int64_t slot = a.slots[it.token];
  uint64_t pos;
  const bool write = it.any & position_of(a, it.token, pos) & ((uint64_t)slot < (uint64_t)a.layout.pages * a.layout.page_size);
  const void* const weight = KEYS ? a.k_norm : nullptr;
  Turn<double> turn;
  const uint32_t signs = lane_signs(p, t);
  if constexpr (KEYS) {
    turn.set(a, weight, pos, lane, t);
#pragma unroll
    for (int e = 0; e < 8; ++e) {   // the vector's signs go with the factors, without any onto the words as they lie in memory
      turn.own[e] = (signs >> e) & 1u ? -turn.own[e] : turn.own[e];
      turn.other[e] = (signs >> e) & 1u ? -turn.other[e] : turn.other[e];
    }
  }
  uint32_t flip[kRawWords];
#pragma unroll
  for (int k = 0; k < kRawWords; ++k) {
    flip[k] = IO == 0 ? signs << (31 - k) & 0x80000000u : (signs >> (2 * k) & 1u) << 15 | (signs >> (2 * k + 1) & 1u) << 31;
    if (KEYS && turn.scaled) flip[k] = 0u;
  }
  if (!POLAR || !p.polar) {
    for (int i = tid; i < p.lut_entries; i += kBlock) s_lut[i] = ((const uint2*)pitch_lut_tab)[p.lut + i];
    __syncthreads();
  }
  const uint64_t page = (uint64_t)slot / a.layout.page_size, in_page = (uint64_t)slot - page * a.layout.page_size;
  uint64_t row = page * a.layout.page_stride + (uint64_t)it.head * a.layout.head_step + in_page * a.layout.slot_step;
#pragma unroll 1
  for (int n = 0; n < H; ++n) {
    double y[8], ss = 0.0, scale;
#pragma unroll
    for (int k = 0; k < kRawWords; ++k) x[0].w[k] ^= flip[k];
    if constexpr (KEYS) {
      turn.apply(x[0], weight != nullptr, y, ss);
    } else {
      float f[8];
      widen(x[0], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (double)f[e];
    }
    const uint64_t w = quantise<POLAR>(p, y, t, s_lut, scale);
    if (weight) scale *= inv_sqrt(ss * (1.0 / D) + (double)a.eps);
    if (write && it.head + n < heads) {
      store_bytes(p.codes + row * p.row_bytes + (uint32_t)t * p.bits, w, p.bits);
      if (t == 0) p.scales[row] = (float)scale;
    }
    row += a.layout.head_step;
#pragma unroll
    for (int i = 0; i + 1 < H; ++i) x[i] = x[i + 1];
  }
}

template <int H>
__device__ __forceinline__ void append_queries(const PagedAppendArgs& a, uint32_t block) {
  const int tid = threadIdx.x, lane = tid & 63, t = lane & (T - 1);
  const Item it(block, (tid >> 6) * V + lane / T, a.tokens, a.q_heads, H);
  Raw x[H];
  load_heads<H>(a.q, it, a.q_heads, t, x);
  uint64_t pos;
  const bool write = it.any & position_of(a, it.token, pos);
  Turn<float> turn;
  turn.set(a, a.q_norm, pos, lane, t);
#pragma unroll
  for (int n = 0; n < H; ++n) {
    float y[8], ss = 0.f;
    turn.apply(x[n], a.q_norm != nullptr, y, ss);
    if (a.q_norm) {
      const float r = inv_sqrt(ss * (1.f / D) + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= r;
    }
    if (write && it.head + n < a.q_heads)
      store_elems<IO, 8>(a.q_out.data, it.token * a.q_out.token_stride + (it.head + n) * a.q_out.head_stride + 8u * t, y, false);
  }
}

// Workgroups take keys, values and q_turn times queries in turn, so that the keys' and values' arithmetic runs beside the queries'
// copies; queries that are left come last. (POLAR: a pool is PolarQuant's. Its exact path's call costs registers.)
template <int H, bool POLAR>
__global__ __launch_bounds__(kBlock) void paged_append(PagedAppendArgs a, uint32_t kv_blocks, uint32_t q_blocks, uint32_t q_turn) {
  __shared__ uint2 s_lut[2048];
  const uint32_t mixed = kv_blocks * (2 + q_turn), cycle = blockIdx.x / (2 + q_turn);
  const uint32_t part = blockIdx.x < mixed ? (blockIdx.x - cycle * (2 + q_turn) + cycle) % (2 + q_turn) : 2;
  const uint32_t q = blockIdx.x < mixed ? cycle * q_turn + part - 2 : blockIdx.x - 2 * kv_blocks;
  if (part == 0 && cycle < kv_blocks) append_vectors<H, POLAR, true>(a, cycle, s_lut);
  else if (part == 1 && cycle < kv_blocks) append_vectors<H, POLAR, false>(a, cycle, s_lut);
  else if (part >= 2 && q < q_blocks) append_queries<H>(a, q);
}

// ----------------------------------------------------------------------------------------------------
// Read back. Row r of the output is token first_tokens[b] + r - row_starts[b] of the sequence b whose range holds it. A workgroup
// takes kReadRows rows of up to four KV heads, keys or values: it looks their pages up once (a chain of three loads), then asks
// for the codes and scales of all its heads, and decodes two vectors per team at a time, whose transforms share the cross-lane
// instructions. The arithmetic and its order are those of vec_decode (pitch_vector.hip), so a row's bytes are those of the
// contiguous decode. Bound by the writes: a read waits long behind them, which is what asking for four heads at once hides
// (with one head at a time 47 us, with the stores under a branch, which makes the next reads' wait one for all stores
// before them, 40-54 us). Measured: 31,616 rows of 8 heads, d = 128 bf16, 4 / 3 bits: 36.9 us for 156 MB (4.2 TB/s); 32,767
// rows of 12 heads, d = 64 float32: 52.5 us for 227 MB (4.3 TB/s; 57 us when each store instruction writes every other
// 16 bytes).

// The sequence whose rows hold row: the last b with starts[b] <= row (starts does not decrease).
template <typename P>
__device__ __forceinline__ uint32_t sequence_of(P starts, uint32_t sequences, int32_t row) {
  uint32_t lo = 0, hi = sequences;
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

constexpr uint32_t kStarts = 1024;   // row starts that are kept in LDS
constexpr uint64_t kNoVector = ~0ull;
constexpr uint32_t kRangeBytes = 0x7FFFFF00u;   // of the buffer that a workgroup's rows are written through

// The vector (of head 0) that a row reads, kNoVector if its page lies outside the pool or the row outside the ranges.
__device__ __forceinline__ uint64_t vector_of(const PagedDecodeArgs& a, const int32_t* s_starts, uint32_t row) {
  const bool local = a.sequences < kStarts;
  const uint32_t b = local ? sequence_of(s_starts, a.sequences, (int32_t)row) : sequence_of(a.row_starts, a.sequences, (int32_t)row);
  const int64_t begin = local ? s_starts[b] : a.row_starts[b], end = local ? s_starts[b + 1] : a.row_starts[b + 1];
  const int64_t token = (int64_t)row - begin + (a.first_tokens ? a.first_tokens[b] : 0);
  if (row >= a.rows || (int64_t)row < begin || (int64_t)row >= end || token < 0 || token > 0x7FFFFFFF) return kNoVector;
  const uint32_t col = (uint32_t)token / a.layout.page_size, slot = (uint32_t)token - col * a.layout.page_size;
  if (col >= a.table_width) return kNoVector;
  const int32_t page = a.tables[(uint64_t)b * a.table_width + col];
  if ((uint32_t)page >= a.layout.pages) return kNoVector;
  return (uint64_t)(uint32_t)page * a.layout.page_stride + (uint64_t)slot * a.layout.slot_step;
}

// The value of the lane of this quad that a DPP quad permutation names.
template <int P>
__device__ __forceinline__ float quad_of(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), P, 0xF, 0xF, true));
}

// Tables of the read-back: four two-bit codes, or two codes of up to five bits, look up the values of their coordinates with the
// transform's first stages applied (as DecTab of pitch_vector.hip); wider codes look up one value each (PolarQuant: radius,
// cosine and sine).
template <int B, bool POLAR>
struct ReadTab {
  static constexpr int L = 1 << B, G = B == 2 && !POLAR ? 4 : B <= 5 ? 2 : 1;
  static constexpr int kEntries = G == 4 ? 256 : G == 2 ? L * L : L, kFloats = G == 1 ? (POLAR ? 3 * L : L) : kEntries * G;
  __device__ static __forceinline__ void build(float* tab, int tid) {
    const float* const book = pitch_codebook_tab + pitch_codebook_offset(ilog2(D), B);
    const float *const radius = pitch_polar_radius_tab + pitch_polar_offset(B), *const cosine = pitch_polar_cos_tab + pitch_polar_offset(B),
                *const sine = pitch_polar_sin_tab + pitch_polar_offset(B);
    for (int i = tid; i < kEntries; i += kBlock) {
      if constexpr (G == 4) {
        const float q0 = book[i & 3], q1 = book[(i >> 2) & 3], q2 = book[(i >> 4) & 3], q3 = book[i >> 6];
        const float a0 = q0 + q1, a1 = q0 - q1, a2 = q2 + q3, a3 = q2 - q3;
        *(f32x4*)(tab + 4 * i) = f32x4{a0 + a2, a1 + a3, a0 - a2, a1 - a3};
      } else if constexpr (G == 2) {
        const int c0 = i & (L - 1), c1 = i >> B;
        const float x = POLAR ? radius[c0] * cosine[c1] : book[c0], y = POLAR ? radius[c0] * sine[c1] : book[c1];
        *(f32x2*)(tab + 2 * i) = f32x2{x + y, x - y};
      } else if constexpr (POLAR) {
        tab[i] = radius[i];
        tab[L + i] = cosine[i];
        tab[2 * L + i] = sine[i];
      } else {
        tab[i] = book[i];
      }
    }
  }
  // The values of the eight codes in x, with the first log2 G stages applied.
  template <typename X>
  __device__ static __forceinline__ void look(const float* tab, X x, float* y) {
    if constexpr (G == 1) {
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        const uint32_t c0 = (uint32_t)(x >> (B * e)) & (L - 1), c1 = (uint32_t)(x >> (B * (e + 1))) & (L - 1);
        const float u = tab[c0];
        y[e] = POLAR ? u * tab[L + c1] : u;
        y[e + 1] = POLAR ? u * tab[2 * L + c1] : tab[c1];
      }
    } else {
      constexpr uint32_t kMask = (uint32_t)(kEntries - 1) * (4 * G);   // an entry's byte offset
#pragma unroll
      for (int k = 0; k < 8 / G; ++k) {
        constexpr int up = G == 4 ? 4 : 3;
        const int pos = G * B * k;
        const uint32_t at = (pos >= up ? (uint32_t)(x >> (pos >= up ? pos - up : 0)) : (uint32_t)x << (up - pos)) & kMask;
        if constexpr (G == 4) {
          const f32x4 v = *(const f32x4*)((const char*)tab + at);
          y[4 * k] = v.x; y[4 * k + 1] = v.y; y[4 * k + 2] = v.z; y[4 * k + 3] = v.w;
        } else {
          const f32x2 v = *(const f32x2*)((const char*)tab + at);
          y[2 * k] = v.x; y[2 * k + 1] = v.y;
        }
      }
    }
  }
};
constexpr int kReadTabFloats = 2048;

// Keys or values of B bits of the workgroup's rows, heads [head, head + count): the codes and scales of all of them are asked for
// at once, since a read takes long among the writes.
template <int B, bool POLAR, int H>
__device__ __forceinline__ void decode_rows(const PagedDecodeArgs& a, const PagedPool& p, const PagedVectors& out, uint32_t head,
                                            uint32_t count, uint32_t row0, const uint64_t* s_vec, const float* s_tab) {
  using TB = ReadTab<B, POLAR>;
  static_assert(TB::kFloats <= kReadTabFloats, "table");
  constexpr int kLoad = B == 2 ? 2 : B <= 4 ? 4 : 8, kRow = D * B / 8;   // bytes of a load, of a row
  using X = std::conditional_t<(B <= 4), uint32_t, uint64_t>;
  const int lane = threadIdx.x & 63, wid = threadIdx.x >> 6, t = lane & (T - 1), team = lane / T;
  const uint32_t at = (uint32_t)(t * B), lo = min(at, (uint32_t)(kRow - kLoad)), sh = 8u * (at - lo);
  // dpp_lane_sign_bit<D, 8, true>: the transform's results are negated on some lanes
  const uint32_t lane_sign = (uint32_t)(__builtin_popcount((unsigned)(t & 11)) & 1) << 31;
  const uint32_t signs = lane_signs(p, t);
  uint32_t flip[IO == 0 ? 8 : 4];   // of the values, or of the pairs of 16-bit values
#pragma unroll
  for (int e = 0; e < (IO == 0 ? 8 : 4); ++e)
    flip[e] = IO == 0 ? signs << (31 - e) & 0x80000000u : (signs >> (2 * e) & 1u) << 15 | (signs >> (2 * e + 1) & 1u) << 31;
  const uint64_t step = a.layout.head_step;
  X w[H][2];
  float scale[H][2];
  uint32_t o[2];   // byte offsets from the workgroup's first row, past the range for rows that are not written
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint32_t r = (uint32_t)((wid * 2 + i) * V + team);
    const uint64_t v = s_vec[r];
    const bool good = v != kNoVector;
    const uint64_t u = (good ? v : 0) + (uint64_t)head * step;
    const uint8_t* const q = p.codes + u * kRow + lo;
    const float* const f = p.scales + u;
    o[i] = good ? (r * (uint32_t)out.token_stride + (IO == 0 ? 8u * (t & ~3) + 4u * (t & 3) : 8u * t)) * Io<IO>::kBytes : kRangeBytes;
#pragma unroll
    for (int n = 0; n < H; ++n) {
      const uint64_t s = min((uint32_t)n, count - 1) * step;
      const uint8_t* const c = q + s * kRow;
      w[n][i] = kLoad == 2 ? *(const u16_any*)c : kLoad == 4 ? *(const u32_any*)c : (X) * (const u64_any*)c;
      scale[n][i] = f[s];
    }
  }
  const float s1 = t & 1 ? -1.f : 1.f, s2 = t & 2 ? -1.f : 1.f, s8 = t & 8 ? -1.f : 1.f;
#pragma unroll
  for (int n = 0; n < H; ++n) {
    if ((uint32_t)n >= count) break;
    const __amdgpu_buffer_rsrc_t to = __builtin_amdgcn_make_buffer_rsrc(
        (char*)out.data + (row0 * out.token_stride + (head + n) * out.head_stride) * Io<IO>::kBytes, 0, kRangeBytes, 0x00027000);
    float y[16];
    TB::look(s_tab, (X)(w[n][0] >> sh), y);
    TB::look(s_tab, (X)(w[n][1] >> sh), y + 8);
#pragma unroll
    for (int m = TB::G; m < 8; m *= 2)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (!(e & m)) {
          const float u = y[e], v = y[e | m];
          y[e] = u + v;
          y[e | m] = u - v;
        }
    fmac_dpp16<1, 0>(y, s1);
    fmac_dpp16<2, 0>(y, s2);
    bfly4_dpp8<0>(y);
    bfly4_dpp8<8>(y);
    if constexpr (T == 16) fmac_dpp16<8, 0>(y, s8);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float fac = __uint_as_float(__float_as_uint(scale[n][i] * (float)kInvSqrtD) ^ lane_sign);
      float r[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) r[e] = __builtin_fmaf(y[8 * i + e], fac, 0.f);
      if constexpr (IO == 0) {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = __uint_as_float(__float_as_uint(r[e]) ^ flip[e]);
        // four lanes exchange their halves: each of the two stores then writes 64 bytes in a row instead of four times 16
        f32x4 z[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float lo0 = quad_of<0x50>(r[e]), hi0 = quad_of<0x50>(r[4 + e]), lo1 = quad_of<0xFA>(r[e]), hi1 = quad_of<0xFA>(r[4 + e]);
          z[0][e] = t & 1 ? hi0 : lo0;
          z[1][e] = t & 1 ? hi1 : lo1;
        }
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, z[0]), to, (int)o[i], 0, 0);
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, z[1]), to, (int)(o[i] + 64), 0, 0);
      } else {   // (rounding to nearest even commutes with the sign)
        const u32x4 v{narrow2<IO>(r[0], r[1]) ^ flip[0], narrow2<IO>(r[2], r[3]) ^ flip[1], narrow2<IO>(r[4], r[5]) ^ flip[2],
                      narrow2<IO>(r[6], r[7]) ^ flip[3]};
        __builtin_amdgcn_raw_buffer_store_b128(v, to, (int)o[i], 0, 0);
      }
    }
  }
}

constexpr int kReadRows = 2 * VPB;   // of a workgroup: two vectors per team
// Heads of a workgroup where these leave two workgroups per compute unit and kind, else one: at 16,384 rows of 8 heads, d = 128
// bf16, four take 16.4 us and one 18.4, at 8,192 rows (2 per unit) 10.9 and 11.9, at 4,096 rows 7.9 and 7.7, at 2,048 6.2 and 5.5.
constexpr uint32_t kReadHeads = 4;

template <int H>
__global__ __launch_bounds__(kBlock) void paged_decode(PagedDecodeArgs a, uint32_t groups) {
  __shared__ __attribute__((aligned(16))) float s_tab[kReadTabFloats];
  __shared__ int32_t s_starts[kStarts];
  __shared__ uint64_t s_vec[kReadRows];
  const int tid = threadIdx.x, kind = (int)blockIdx.y;
  const uint32_t block = blockIdx.x / groups, head = (blockIdx.x - block * groups) * H, count = min((uint32_t)H, a.layout.kv_heads - head);
  const uint32_t row0 = block * kReadRows;
  const PagedVectors& out = a.out[kind];
  if (!out.data) return;
  const PagedPool& p = a.pool[kind];
  if (a.sequences < kStarts)
    for (uint32_t i = tid; i <= a.sequences; i += kBlock) s_starts[i] = a.row_starts[i];
#define PITCH_PAGED_WIDTHS(F) F(2) F(3) F(4) F(5) F(6) F(7) F(8)
#define PITCH_PAGED_TAB(B)                                \
  case B:                                                 \
    if (p.polar) ReadTab<B, true>::build(s_tab, tid);     \
    else ReadTab<B, false>::build(s_tab, tid);            \
    break;
#define PITCH_PAGED_DECODE(B)                                                                   \
  case B:                                                                                       \
    if (p.polar) decode_rows<B, true, H>(a, p, out, head, count, row0, s_vec, s_tab);           \
    else decode_rows<B, false, H>(a, p, out, head, count, row0, s_vec, s_tab);                  \
    break;
  switch (p.bits) {
    PITCH_PAGED_WIDTHS(PITCH_PAGED_TAB)
    default: break;
  }
  __syncthreads();
  if (tid < kReadRows) s_vec[tid] = vector_of(a, s_starts, row0 + tid);
  __syncthreads();
  switch (p.bits) {
    PITCH_PAGED_WIDTHS(PITCH_PAGED_DECODE)
    default: break;
  }
#undef PITCH_PAGED_DECODE
#undef PITCH_PAGED_TAB
}

}  // namespace

#define PITCH_CAT4_(a, b, c, d) a##b##c##d
#define PITCH_CAT4(a, b, c, d) PITCH_CAT4_(a, b, c, d)
hipError_t PITCH_CAT4(launch_paged_append_d, PITCH_DIM, _io, PITCH_IO)(const PagedAppendArgs& a0, hipStream_t s) {
  PagedAppendArgs a = a0;
  for (PagedPool& p : a.pool) {
    const PitchLutInfo li = pitch_lut_info(ilog2(D), (int)p.bits);
    if (li.offset < 0 || li.entries > 2048) return hipErrorInvalidValue;   // every width of these dimensions has one
    p.lut = li.offset;
    p.lut_entries = li.entries;
    p.lut_scale = li.scale;
    p.lut_off = li.off;
  }
  // Four heads per team where these make eight workgroups per compute unit, else one: 8 KV and 32 query heads, d = 128 bf16, take
  // 48 us and 65 at 8,191 tokens, 27 and 32 at 4,096, 17.3 and 17.0 at 2,048, 8.6 and 7.0 at 512. PolarQuant takes one, whose kernel
  // holds more waves (2 KV and 12 query heads at 8,000 tokens: 23 us, 32 with four). Among the keys and values come up to three
  // workgroups of queries each (48 us; with one 49, with all of them last 53; an even number gives one XCD all of the keys: with
  // two 62).
  const bool polar = a.pool[0].polar || a.pool[1].polar;
  const uint32_t most = 1u << 25, slice = max(1u, most / max(a.layout.kv_heads, a.q_heads));   // tokens of a launch, whose grid has a limit
  for (uint32_t left = a0.tokens; left;) {
    a.tokens = min(left, slice);
    auto blocks = [&](uint32_t heads, uint32_t h) { return (uint32_t)(((uint64_t)a.tokens * ((heads + h - 1) / h) + VPB - 1) / VPB); };
    const bool four = !polar && 2ull * blocks(a.layout.kv_heads, 4) + blocks(a.q_heads, 4) >= 8ull * (uint64_t)device_cu_count();
    const uint32_t h = four ? 4 : 1, nkv = blocks(a.layout.kv_heads, h), nq = blocks(a.q_heads, h);
    const uint32_t turn = min(3u, (nq + nkv - 1) / nkv) | 1u, grid = nkv * (2 + turn) + (nq > nkv * turn ? nq - nkv * turn : 0u);
    void (*const kernel)(PagedAppendArgs, uint32_t, uint32_t, uint32_t) =
        four ? paged_append<4, false> : polar ? paged_append<1, true> : paged_append<1, false>;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(kBlock), 0, s, a, nkv, nq, turn);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    left -= a.tokens;
    for (PagedVectors* v : {&a.in[0], &a.in[1], &a.q, &a.q_out})
      if (v->data) v->data = (char*)v->data + (uint64_t)a.tokens * v->token_stride * Io<IO>::kBytes;
    a.slots += a.tokens;
    if (a.positions) a.positions += a.tokens;
  }
  return hipSuccess;
}

hipError_t PITCH_CAT4(launch_paged_decode_d, PITCH_DIM, _io, PITCH_IO)(const PagedDecodeArgs& a, hipStream_t s) {
  const uint32_t heads = a.layout.kv_heads, cus = (uint32_t)device_cu_count(), blocks = (a.rows + kReadRows - 1) / kReadRows;
  const uint32_t groups = (heads + kReadHeads - 1) / kReadHeads;
  if ((uint64_t)blocks * groups >= 2ull * cus)
    hipLaunchKernelGGL(paged_decode<kReadHeads>, dim3(blocks * groups, 2), dim3(kBlock), 0, s, a, groups);
  else
    hipLaunchKernelGGL(paged_decode<1>, dim3(blocks * heads, 2), dim3(kBlock), 0, s, a, heads);
  return hipGetLastError();
}

}  // namespace pitch
