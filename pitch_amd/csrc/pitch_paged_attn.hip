// Attention of one new token of every sequence over a paged cache, for one dimension (PITCH_DIM = 64 or 128).
//
// out = softmax(z) V with z_t = cap tanh(scale q . k_t / cap) + slope (t - (L - 1)) over the tokens t of [L - window, L).
// No token is decoded: k_t = s H c(code_t) n_t / sqrt(d), so a query is rotated once (H s q), scores are its products
// with the table values of the codes times the token's scale, and the weighted table values are rotated back once.
#include "pitch_device.h"
#include "pitch_paged.h"

#ifndef PITCH_DIM
#error "compile with -DPITCH_DIM=<dim>"
#endif

namespace pitch {
namespace {

constexpr int D = PITCH_DIM;
constexpr int kChunk = 256;
constexpr float kLn2 = 0x1.62e430p-1f;

typedef uint32_t u32_any __attribute__((aligned(1)));
typedef uint64_t u64_any __attribute__((aligned(1)));

__device__ void load_tab(const PagedPool& p, float* tab) {
  const int levels = 1 << p.bits;
  for (int i = threadIdx.x; i < levels; i += kChunk) {
    if (p.polar) {
      const int off = pitch_polar_offset(p.bits);
      tab[i] = pitch_polar_radius_tab[off + i];
      tab[256 + i] = pitch_polar_cos_tab[off + i];
      tab[512 + i] = pitch_polar_sin_tab[off + i];
    } else {
      tab[i] = pitch_codebook_tab[pitch_codebook_offset(ilog2(D), p.bits) + i];
    }
  }
}

template <int IO>
__global__ __launch_bounds__(kChunk) void paged_attn(PagedAttnArgs a) {
  __shared__ float s_kt[768], s_vt[768], s_q[8][D], s_p[8][kChunk], s_o[8][D], s_red[8], s_m[8], s_l[8], s_al[8];
  __shared__ uint64_t s_row[kChunk];
  const int tid = threadIdx.x;
  const uint32_t b = blockIdx.x / a.layout.kv_heads, kv = blockIdx.x % a.layout.kv_heads, nq = a.nq;
  load_tab(a.k, s_kt);
  load_tab(a.v, s_vt);
  for (int i = tid; i < 8 * D; i += kChunk) {
    const uint32_t h = i / D, j = i % D;
    float x = 0.f;
    if (h < nq) {
      float f[1];
      load_elems<IO, 1>(a.q.data, b * a.q.token_stride + (kv * nq + h) * a.q.head_stride + j, f);
      x = (a.k.signs[j >> 5] >> (j & 31)) & 1 ? -f[0] : f[0];
    }
    s_q[h][j] = x;
    s_o[h][j] = 0.f;
  }
  if (tid < 8) {
    s_m[tid] = -__FLT_MAX__;
    s_l[tid] = 0.f;
  }
  __syncthreads();
  for (int m = 1; m < D; m *= 2) {
    float x[8 * D / 2 / kChunk][2];
    for (int i = tid, k = 0; i < 8 * D / 2; i += kChunk, ++k) {
      const int h = i / (D / 2), r = i % (D / 2), j = (r / m) * 2 * m + r % m;
      x[k][0] = s_q[h][j];
      x[k][1] = s_q[h][j + m];
      s_q[h][j] = x[k][0] + x[k][1];
      s_q[h][j + m] = x[k][0] - x[k][1];
    }
    __syncthreads();
  }
  const uint64_t most = (uint64_t)a.table_width * a.layout.page_size;
  const int64_t len0 = a.lengths[b];
  const uint64_t len = len0 < 0 ? 0 : min((uint64_t)len0, most);
  const uint64_t begin = a.window && len > a.window ? len - a.window : 0;
  for (uint64_t t0 = begin; t0 < len; t0 += kChunk) {
    const uint64_t t = t0 + tid;
    bool in = t < len;
    uint64_t row = 0;
    if (in) {
      const uint64_t col = t / a.layout.page_size;
      const int32_t page = a.tables[(uint64_t)b * a.table_width + col];
      in = (uint32_t)page < a.layout.pages;
      if (in)
        row = (uint64_t)page * a.layout.page_stride + (uint64_t)kv * a.layout.head_step + (t - col * a.layout.page_size) * a.layout.slot_step;
    }
    s_row[tid] = in ? row : ~0ull;
    float s[8] = {};
    const uint8_t* kr = a.k.codes + row * a.k.row_bytes;
    const uint32_t mask = (1u << a.k.bits) - 1;
    for (int g = 0; g < D / 8; ++g) {
      const uint32_t at = g * a.k.bits, lo = min(at, a.k.row_bytes - 8u);
      const uint64_t w = *(const u64_any*)(kr + lo) >> (8u * (at - lo));
      float y[8];
      for (int e = 0; e < 8; e += 2) {
        const uint32_t c0 = (uint32_t)(w >> (a.k.bits * e)) & mask, c1 = (uint32_t)(w >> (a.k.bits * (e + 1))) & mask;
        y[e] = a.k.polar ? s_kt[c0] * s_kt[256 + c1] : s_kt[c0];
        y[e + 1] = a.k.polar ? s_kt[c0] * s_kt[512 + c1] : s_kt[c1];
      }
      for (int h = 0; h < 8; ++h)
        for (int e = 0; e < 8; ++e) s[h] = __builtin_fmaf(s_q[h][8 * g + e], y[e], s[h]);
    }
    const float nk = in ? a.k.scales[row] * a.qscale : 0.f;
    for (int h = 0; h < 8; ++h) {
      float z = s[h] * nk;
      if (a.cap > 0.f) z = a.cap * (1.f - 2.f / (1.f + __builtin_amdgcn_exp2f(z)));
      if (a.slopes && h < (int)nq) z += a.slopes[kv * nq + h] * a.slope_scale * ((float)t - (float)(len - 1));
      s_p[h][tid] = in ? z : -__builtin_inff();
    }
    __syncthreads();
    // the chunk's maximum, the weights and their sum: two heads per wave
    for (int h = (tid >> 6) * 2; h < (tid >> 6) * 2 + 2; ++h) {
      float m = s_m[h], l = 0.f;
      for (int i = tid & 63; i < kChunk; i += 64) m = fmaxf(m, s_p[h][i]);
      for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d));
      for (int i = tid & 63; i < kChunk; i += 64) {
        const float p = __builtin_amdgcn_exp2f(s_p[h][i] - m);
        l += p;
        s_p[h][i] = s_row[i] == ~0ull ? 0.f : p * a.v.scales[s_row[i]];
      }
      for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d);
      if ((tid & 63) == 0) {
        s_al[h] = __builtin_amdgcn_exp2f(s_m[h] - m);
        s_l[h] = s_l[h] * s_al[h] + l;
        s_m[h] = m;
      }
    }
    __syncthreads();
    // values: thread = pair of coordinates x part of the chunk's tokens, four or two heads at a time
    constexpr int P = kChunk / (D / 2);
    const int j = 2 * (tid % (D / 2)), part = tid / (D / 2);
    float o[8][2] = {};
    const uint32_t vmask = (1u << a.v.bits) - 1, vat = (j * a.v.bits) / 8, vlo = min(vat, a.v.row_bytes - 4u);
    const uint32_t vsh = j * a.v.bits - 8 * vlo;
    for (int i = part; i < kChunk; i += P) {
      const uint64_t r = s_row[i];
      if (r == ~0ull) continue;
      const uint32_t w = *(const u32_any*)(a.v.codes + r * a.v.row_bytes + vlo) >> vsh;
      const uint32_t c0 = w & vmask, c1 = (w >> a.v.bits) & vmask;
      const float y0 = a.v.polar ? s_vt[c0] * s_vt[256 + c1] : s_vt[c0], y1 = a.v.polar ? s_vt[c0] * s_vt[512 + c1] : s_vt[c1];
      for (int h = 0; h < 8; ++h) {
        o[h][0] = __builtin_fmaf(s_p[h][i], y0, o[h][0]);
        o[h][1] = __builtin_fmaf(s_p[h][i], y1, o[h][1]);
      }
    }
    for (int k = 0; k < P; ++k) {
      if (part == k)
        for (int h = 0; h < 8; ++h)
          for (int e = 0; e < 2; ++e) s_o[h][j + e] = (k == 0 ? s_o[h][j + e] * s_al[h] : s_o[h][j + e]) + o[h][e];
      __syncthreads();
    }
  }
  for (int m = 1; m < D; m *= 2) {
    for (int i = tid; i < 8 * D / 2; i += kChunk) {
      const int h = i / (D / 2), r = i % (D / 2), j = (r / m) * 2 * m + r % m;
      const float x = s_o[h][j], y = s_o[h][j + m];
      s_o[h][j] = x + y;
      s_o[h][j + m] = x - y;
    }
    __syncthreads();
  }
  for (int i = tid; i < (int)nq * D; i += kChunk) {
    const int h = i / D, j = i % D;
    float f[1] = {s_l[h] > 0.f ? s_o[h][j] * a.oscale / s_l[h] : 0.f};
    if ((a.v.signs[j >> 5] >> (j & 31)) & 1) f[0] = -f[0];
    store_elems<IO, 1>(a.out.data, b * a.out.token_stride + (kv * nq + h) * a.out.head_stride + j, f, false);
  }
  if (a.lse && tid < (int)nq)
    a.lse[(uint64_t)b * a.layout.kv_heads * nq + kv * nq + tid] = s_l[tid] > 0.f ? (s_m[tid] + log2f(s_l[tid])) * kLn2 : -__builtin_inff();
}

}  // namespace

#define PITCH_CAT_(a, b) a##b
#define PITCH_CAT(a, b) PITCH_CAT_(a, b)
hipError_t PITCH_CAT(launch_paged_attention_d, PITCH_DIM)(const PagedAttnArgs& a, uint32_t io, hipStream_t s) {
  const dim3 grid(a.sequences * a.layout.kv_heads);
  if (io == 1) hipLaunchKernelGGL((paged_attn<1>), grid, dim3(kChunk), 0, s, a);
  else hipLaunchKernelGGL((paged_attn<2>), grid, dim3(kChunk), 0, s, a);
  return hipGetLastError();
}

}  // namespace pitch
