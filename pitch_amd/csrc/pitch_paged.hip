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

// y = w . x rotated to position pos, for this lane's coordinates; ss = sum of the x^2 over the vector (with a norm).
template <typename F>
__device__ __forceinline__ void norm_rotate(const PagedAppendArgs& a, const void* x, uint64_t at, const void* weight,
                                            uint64_t pos, int t, F (&y)[8], F& ss) {
  float f[8];
  load_elems<IO, 8>(x, at + 8u * t, f);
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = (F)f[e];
  if (weight) {
    ss = F(0);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fma_t(y[e], y[e], ss);
    ss = team_reduce<T>(ss, [](F p, F q) { return p + q; });
    load_elems<IO, 8>(weight, 8u * t, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] *= (F)f[e];
  }
  if (a.positions && 8u * t < a.rotary) {
    // the partner coordinates are another lane's: read again (they are in the nearest cache)
    const uint32_t half = a.rotary / 2, j = 8u * t, pj = j < half ? j + half : j - half;
    float p[8], c[8], s[8];
    load_elems<IO, 8>(x, at + pj, p);
    load_elems<0, 8>(a.cos, pos * a.rotary + j, c);
    load_elems<0, 8>(a.sin, pos * a.rotary + j, s);
    if (weight) load_elems<IO, 8>(weight, pj, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      F q = (F)p[e];
      if (weight) q *= (F)f[e];
      q = j < half ? -q : q;
      y[e] = fma_t(y[e], (F)c[e], q * (F)s[e]);
    }
  }
}

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

// Keys (kind 0) or values (kind 1) of the workgroup's vectors.
__device__ __forceinline__ void append_vectors(const PagedAppendArgs& a, const PagedPool& p, const PagedVectors& in,
                                               const void* weight, bool rotate, uint32_t block, uint32_t blocks,
                                               uint2* s_lut) {
  const int tid = threadIdx.x, lane = tid & 63, t = lane & (T - 1), team = (tid >> 6) * V + lane / T;
  const uint32_t heads = a.layout.kv_heads, count = a.tokens * heads;   // below 2^32 (checked by the caller)
  const uint32_t signs = lane_signs(p, t);
  if (!p.polar) {
    for (int i = tid; i < p.lut_entries; i += kBlock) s_lut[i] = ((const uint2*)pitch_lut_tab)[p.lut + i];
    __syncthreads();
  }
  for (uint32_t base = block * VPB; base < count; base += blocks * VPB) {
    const uint32_t nominal = base + team, v = min(nominal, count - 1);
    const uint32_t tok = v / heads, head = v - tok * heads;
    const int64_t slot = a.slots[tok];
    bool write = nominal < count && (uint64_t)slot < (uint64_t)a.layout.pages * a.layout.page_size;
    uint64_t pos = 0;
    if (a.positions) {
      pos = (uint64_t)a.positions[tok];
      write = write && pos < a.table_rows;
      pos = pos < a.table_rows ? pos : 0;
    }
    double y[8], ss = 0.0;
    if (rotate) {
      norm_rotate<double>(a, in.data, tok * in.token_stride + head * in.head_stride, weight, pos, t, y, ss);
    } else {
      float f[8];
      load_elems<IO, 8>(in.data, tok * in.token_stride + head * in.head_stride + 8u * t, f);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (double)f[e];
    }
    const double r = weight ? 1.0 / __builtin_sqrt(ss * (1.0 / D) + (double)a.eps) : 1.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = (signs >> e) & 1u ? -y[e] : y[e];
    uint64_t w = 0;
    double scale;
    if (!p.polar) {
      double n2 = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) n2 = __builtin_fma(y[e], y[e], n2);
      n2 = team_reduce<T>(n2, [](double x, double z) { return x + z; });
      const double nrm = __builtin_sqrt(n2), us = (1.0 / (nrm > 0.0 ? nrm : 1.0)) * kInvSqrtD;
      scale = nrm * r;
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
        const uint32_t code = entry[e].y + (y[e] * us > (double)__uint_as_float(entry[e].x) ? 1u : 0u);
        w |= (uint64_t)code << (p.bits * e);
      }
    } else {
      fwht_contig<8, T, double>(y, t);
      double r2[4], top = 0.0;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        r2[q] = __builtin_fma(y[2 * q], y[2 * q], y[2 * q + 1] * y[2 * q + 1]);
        top = r2[q] > top ? r2[q] : top;
      }
      top = team_reduce<T>(top, [](double x, double z) { return x > z ? x : z; });
      const double rmax = __builtin_sqrt(top), safe = rmax > 0.0 ? rmax : 1.0, inv = 1.0 / safe;
      scale = rmax * kInvSqrtD * r;
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
        w |= (uint64_t)(code[q] & 255u) << (2 * p.bits * q) | (uint64_t)(code[q] >> 8) << (2 * p.bits * q + p.bits);
      }
    }
    if (write) {
      const uint64_t page = (uint64_t)slot / a.layout.page_size, in_page = (uint64_t)slot - page * a.layout.page_size;
      const uint64_t row = page * a.layout.page_stride + (uint64_t)head * a.layout.head_step + in_page * a.layout.slot_step;
      store_bytes(p.codes + row * p.row_bytes + (uint32_t)t * p.bits, w, p.bits);
      if (t == 0) p.scales[row] = (float)scale;
    }
  }
}

__device__ __forceinline__ void append_queries(const PagedAppendArgs& a, uint32_t block, uint32_t blocks) {
  const int tid = threadIdx.x, lane = tid & 63, t = lane & (T - 1), team = (tid >> 6) * V + lane / T;
  const uint32_t heads = a.q_heads, count = a.tokens * heads;
  for (uint32_t base = block * VPB; base < count; base += blocks * VPB) {
    const uint32_t nominal = base + team, v = min(nominal, count - 1);
    const uint32_t tok = v / heads, head = v - tok * heads;
    bool write = nominal < count;
    uint64_t pos = 0;
    if (a.positions) {
      pos = (uint64_t)a.positions[tok];
      write = write && pos < a.table_rows;
      pos = pos < a.table_rows ? pos : 0;
    }
    float y[8], ss = 0.f;
    norm_rotate<float>(a, a.q.data, tok * a.q.token_stride + head * a.q.head_stride, a.q_norm, pos, t, y, ss);
    if (a.q_norm) {
      const float r = 1.f / __builtin_sqrtf(ss * (1.f / D) + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] *= r;
    }
    if (write) store_elems<IO, 8>(a.q_out.data, tok * a.q_out.token_stride + head * a.q_out.head_stride + 8u * t, y, false);
  }
}

__global__ __launch_bounds__(kBlock) void paged_append(PagedAppendArgs a) {
  __shared__ uint2 s_lut[2048];
  const uint32_t b = blockIdx.x;
  if (b < a.first[1]) append_vectors(a, a.pool[0], a.in[0], a.k_norm, true, b, a.first[1], s_lut);
  else if (b < a.first[2]) append_vectors(a, a.pool[1], a.in[1], nullptr, false, b - a.first[1], a.first[2] - a.first[1], s_lut);
  else append_queries(a, b - a.first[2], a.first[3] - a.first[2]);
}

// ----------------------------------------------------------------------------------------------------
// Read back. Row r of the output is token first_tokens[b] + r - row_starts[b] of the sequence b whose range holds it.

// The sequence whose rows hold row: the last b with row_starts[b] <= row (row_starts does not decrease).
__device__ __forceinline__ uint32_t sequence_of(const int32_t* row_starts, uint32_t sequences, int32_t row) {
  uint32_t lo = 0, hi = sequences;   // row_starts[lo] <= row < row_starts[hi], where the row is in the ranges at all
  while (hi - lo > 1) {
    const uint32_t mid = (lo + hi) / 2;
    if (row_starts[mid] <= row) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ void decode_vectors(const PagedDecodeArgs& a, const PagedPool& p, const PagedVectors& out,
                                               uint32_t head, uint32_t row, int t, float* s_tab) {
  const uint32_t b = sequence_of(a.row_starts, a.sequences, (int32_t)row);
  const int64_t begin = a.row_starts[b], end = a.row_starts[b + 1];
  const int64_t token = (int64_t)row - begin + (a.first_tokens ? a.first_tokens[b] : 0);
  bool good = (int64_t)row >= begin && (int64_t)row < end && token >= 0;
  const uint64_t col = (uint64_t)token / a.layout.page_size, slot = (uint64_t)token - col * a.layout.page_size;
  good = good && col < a.table_width;
  const int32_t page = good ? a.tables[(uint64_t)b * a.table_width + col] : 0;
  good = good && (uint32_t)page < a.layout.pages;
  const uint64_t v = good ? (uint64_t)page * a.layout.page_stride + (uint64_t)head * a.layout.head_step + slot * a.layout.slot_step
                          : 0;
  // the lane's eight codes: `bits` bytes, read as eight that stay inside the row
  const uint32_t at = (uint32_t)t * p.bits, lo = min(at, p.row_bytes - 8u);
  uint64_t w = *(const u64_any*)(p.codes + v * p.row_bytes + lo);
  w >>= 8u * (at - lo);
  const float scale = p.scales[v];
  const uint32_t levels = 1u << p.bits, mask = levels - 1;
  float y[8];
  if (!p.polar) {
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = s_tab[(uint32_t)(w >> (p.bits * e)) & mask];
  } else {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float r = s_tab[(uint32_t)(w >> (2 * p.bits * q)) & mask];
      const uint32_t k = (uint32_t)(w >> (2 * p.bits * q + p.bits)) & mask;
      y[2 * q] = r * s_tab[levels + k];
      y[2 * q + 1] = r * s_tab[2 * levels + k];
    }
  }
  fwht_contig<8, T, float>(y, t);
  // as dec_out of pitch_vector.hip: the same bytes as the decode of a contiguous cache (a zero is +0 before its sign)
  const float f = scale * (float)kInvSqrtD;
  const uint32_t signs = lane_signs(p, t);
#pragma unroll
  for (int e = 0; e < 8; ++e)
    y[e] = __uint_as_float(__float_as_uint(__builtin_fmaf(y[e], f, 0.f)) ^ ((signs >> e) & 1u) << 31);
  if (good) store_elems<IO, 8>(out.data, row * out.token_stride + head * out.head_stride + 8u * t, y, false);
}

__global__ __launch_bounds__(kBlock) void paged_decode(PagedDecodeArgs a) {
  __shared__ float s_tab[3 * 256];
  const int tid = threadIdx.x, lane = tid & 63, t = lane & (T - 1), team = (tid >> 6) * V + lane / T;
  const uint32_t kind = blockIdx.z, head = blockIdx.y;
  const PagedPool& p = a.pool[kind];
  if (!a.out[kind].data) return;
  const int levels = 1 << p.bits;
  if (p.polar) {
    const int off = pitch_polar_offset(p.bits);
    for (int i = tid; i < levels; i += kBlock) {
      s_tab[i] = pitch_polar_radius_tab[off + i];
      s_tab[levels + i] = pitch_polar_cos_tab[off + i];
      s_tab[2 * levels + i] = pitch_polar_sin_tab[off + i];
    }
  } else {
    const int off = pitch_codebook_offset(ilog2(D), p.bits);
    for (int i = tid; i < levels; i += kBlock) s_tab[i] = pitch_codebook_tab[off + i];
  }
  __syncthreads();
  for (uint64_t base = (uint64_t)blockIdx.x * VPB; base < a.rows; base += (uint64_t)gridDim.x * VPB) {
    const uint64_t row = base + team;
    if (row < a.rows) decode_vectors(a, p, a.out[kind], head, (uint32_t)row, t, s_tab);
  }
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
  const uint64_t most = 8ull * (uint64_t)device_cu_count();
  const uint64_t kv = ((uint64_t)a.tokens * a.layout.kv_heads + VPB - 1) / VPB, q = ((uint64_t)a.tokens * a.q_heads + VPB - 1) / VPB;
  const uint32_t nkv = (uint32_t)(kv < most ? kv : most), nq = (uint32_t)(q < 2 * most ? q : 2 * most);
  a.first[0] = 0;
  a.first[1] = nkv;
  a.first[2] = 2 * nkv;
  a.first[3] = 2 * nkv + nq;
  hipLaunchKernelGGL(paged_append, dim3(a.first[3]), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

hipError_t PITCH_CAT4(launch_paged_decode_d, PITCH_DIM, _io, PITCH_IO)(const PagedDecodeArgs& a, hipStream_t s) {
  const uint64_t need = ((uint64_t)a.rows + VPB - 1) / VPB, most = 8ull * (uint64_t)device_cu_count();
  hipLaunchKernelGGL(paged_decode, dim3((uint32_t)(need < most ? need : most), a.layout.kv_heads, 2), dim3(kBlock), 0, s, a);
  return hipGetLastError();
}

}  // namespace pitch
