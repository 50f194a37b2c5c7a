// Arguments and launches of attention over whole prompts (pitch_prompt.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pitch_paged.h"

namespace pitch {

struct PromptArgs {
  PagedVectors q, k, v, out;  // of the call's 16-bit type
  const int32_t* row_starts;  // [sequences + 1]: queries of each sequence
  const int32_t* key_starts;  // [sequences + 1]: keys of each sequence
  const float* slopes;        // [query heads] or null
  float* lse;                 // [rows][query heads] or null
  float* ws;                  // partial results of a call whose keys are split
  uint32_t rows, keys;        // tokens that the queries' and the keys' buffers hold
  uint32_t sequences, kv_heads, nq;
  uint32_t causal, window;    // window 0: all
  uint32_t negate;            // 1: a negative scale, whose sign the queries take
  float c;                    // |scale| log2(e): scores to log2 units (1 with a cap or slopes, which give such units)
  float pre;                  // with a cap or slopes: what a product is multiplied by first
  float cap, cap_r;           // scores x are cap * tanh(x * cap_r) when cap is positive (log2 units), else x
  uint32_t tiles;             // an upper bound of the query tiles of a KV head (set by the launcher, as splits)
  uint32_t splits;            // parts of a tile's keys
};

// Rows of (token, query head of a KV head) in a tile; tiles and parts of the keys; floats of workspace.
constexpr uint32_t kPromptRows = 128;
struct PromptPlan {
  uint32_t tiles, splits;
  uint64_t ws_floats;
};
inline PromptPlan prompt_plan(uint32_t rows, uint32_t keys, uint32_t sequences, uint32_t kv_heads, uint32_t nq, uint32_t dim,
                              uint32_t cus) {
  PromptPlan p{};
  p.tiles = (uint32_t)((uint64_t)rows * nq / kPromptRows) + (sequences < rows ? sequences : rows);
  const uint64_t groups = (uint64_t)p.tiles * kv_heads, slots = 2ull * cus;
  uint64_t splits = 1;
  if (groups < slots) {
    // parts of 256 keys or more, of a sequence of twice the average length
    const uint64_t most = 2ull * keys / sequences / 256;
    splits = (4 * slots + groups - 1) / groups;
    splits = splits < most ? splits : most;
    splits = splits < 1 ? 1 : splits > 64 ? 64 : splits;
  }
  p.splits = (uint32_t)splits;
  if (splits > 1) p.ws_floats = splits * rows * kv_heads * nq * (dim + 2ull);
  return p;
}

#define PITCH_DECLARE_PROMPT(D)                                                             \
  hipError_t launch_prompt_d##D##_io1(const PromptArgs& a, hipStream_t s);                   \
  hipError_t launch_prompt_d##D##_io2(const PromptArgs& a, hipStream_t s);
PITCH_DECLARE_PROMPT(64)
PITCH_DECLARE_PROMPT(128)
#undef PITCH_DECLARE_PROMPT

}  // namespace pitch
