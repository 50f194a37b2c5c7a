// Arguments and launches of the paged cache's kernels (pitch_paged.hip, pitch_paged_attn.hip). A pool holds pages of
// page_size token slots for every KV head; the vector of (page, head, slot) is page * page_stride + head * head_step +
// slot * slot_step, for the codes (row_bytes each) and for the scales.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pitch {

// One of a cache's two pools (keys, values) and how its vectors are quantised.
struct PagedPool {
  uint8_t* codes;
  float* scales;
  uint32_t polar, bits, row_bytes;
  uint32_t signs[4];         // rotation signs: bit i of the 128 is 1 where coordinate i has sign -1
  int32_t lut, lut_entries;  // TurboQuant's bucket table (pitch_lut_tab), its scale and offset
  double lut_scale, lut_off;
};

struct PagedLayout {
  uint64_t page_stride;
  uint32_t pages, page_size, kv_heads, head_step, slot_step;
};

// The strided vectors of a call: vector (token t, head h) starts at element t * token_stride + h * head_stride.
struct PagedVectors {
  void* data;
  uint64_t token_stride, head_stride;
};

struct PagedAppendArgs {
  PagedPool pool[2];         // keys, values
  PagedLayout layout;
  PagedVectors in[2], q, q_out;
  const int64_t* slots;      // page * page_size + slot of each token; others are not written
  const int64_t* positions;  // null: no rotation
  const float* cos;          // [table_rows][rotary]
  const float* sin;
  const void* q_norm;        // weights of the vectors' type, or null
  const void* k_norm;
  uint64_t table_rows;
  uint32_t tokens, q_heads, rotary;
  float eps;
};

struct PagedDecodeArgs {
  PagedPool pool[2];
  PagedLayout layout;
  PagedVectors out[2];       // data null: not read back
  const int32_t* tables;     // [sequences][table_width] page numbers
  const int32_t* row_starts; // [sequences + 1]
  const int32_t* first_tokens;  // [sequences] or null
  uint32_t table_width, sequences, rows;
};

struct PagedAttnArgs {
  PagedPool k, v;
  PagedLayout layout;
  PagedVectors q, out;       // token = sequence
  const int32_t* tables;
  const int32_t* lengths;    // [sequences] cached tokens
  const float* slopes;       // [query heads] or null
  float* lse;                // [sequences][query heads] or null
  float* ws;
  uint32_t table_width, sequences, nq, window;
  uint32_t most_tokens;      // table_width * page_size
  float qscale;              // what the rotated queries are multiplied by
  float cap, cap_r;          // scores x are cap * tanh(x * cap_r) when cap is positive (log2 units), else x
  float slope_scale;         // log2(e): slopes to log2 units
  float oscale;              // 1 / sqrt(dim) of the value decode
  float kfactor, vfactor;    // the tables' factors and their reciprocals (set by the launcher)
  float kinv, vinv;
  uint32_t groups;           // workgroups
  uint32_t groups_r, page_r; // floor((2^32 - 1) / d) of groups and of page_size / 16 (set by the launcher, as the next two)
  uint32_t tile_cols, tile_rest;  // 64 tokens as pages and the rest
  uint32_t whole;            // workgroups take whole pairs of sequence and KV head: no join
  uint32_t kpage, vpage, khead, vhead, kslot, vslot;  // bytes of codes from page to page, head to head, slot to slot
};

#define PITCH_DECLARE_PAGED(D, IO)                                                     \
  hipError_t launch_paged_append_d##D##_io##IO(const PagedAppendArgs& a, hipStream_t s); \
  hipError_t launch_paged_decode_d##D##_io##IO(const PagedDecodeArgs& a, hipStream_t s);
PITCH_DECLARE_PAGED(64, 0)
PITCH_DECLARE_PAGED(64, 1)
PITCH_DECLARE_PAGED(64, 2)
PITCH_DECLARE_PAGED(128, 0)
PITCH_DECLARE_PAGED(128, 1)
PITCH_DECLARE_PAGED(128, 2)
#undef PITCH_DECLARE_PAGED

// Attention: most sequences of a call (32 per lane of a wave), waves of a workgroup, floats of a partial result (maxima and sums
// of eight heads, accumulators of nh heads), floats of workspace of a call (four words and two slots per workgroup, one slot per
// wave; the same whatever the sequences are).
constexpr uint32_t kPagedMostSequences = 2048;
constexpr uint32_t kPagedAttnWaves = 8;
constexpr uint32_t paged_slot_floats(uint32_t dim, uint32_t nh) { return 16 + dim * nh; }
constexpr uint64_t paged_attention_workspace_floats(uint32_t dim, uint32_t nq, uint32_t groups) {
  return groups * (4ull + (2ull + kPagedAttnWaves) * paged_slot_floats(dim, nq <= 4 ? 4 : 8));
}
#define PITCH_DECLARE_PAGED_ATTN(K)                                                             \
  hipError_t launch_paged_attention_d64_k##K(const PagedAttnArgs& a, uint32_t io, hipStream_t s); \
  hipError_t launch_paged_attention_d128_k##K(const PagedAttnArgs& a, uint32_t io, hipStream_t s);
PITCH_DECLARE_PAGED_ATTN(0)
PITCH_DECLARE_PAGED_ATTN(2)
PITCH_DECLARE_PAGED_ATTN(3)
PITCH_DECLARE_PAGED_ATTN(4)
#undef PITCH_DECLARE_PAGED_ATTN

}  // namespace pitch
