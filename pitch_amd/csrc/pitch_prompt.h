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
  float* ws;                  // with places: 5 words per sequence and 2 more, parts of results from parts_at on
  uint32_t rows, keys;        // tokens that the queries' and the keys' buffers hold
  uint32_t sequences, kv_heads, nq;
  uint32_t causal, window;    // window 0: all
  uint32_t negate;            // 1: a negative scale, whose sign the queries take
  float c;                    // |scale| log2(e): scores to log2 units (1 with a cap or slopes, which give such units)
  float pre;                  // with a cap or slopes: what a product is multiplied by first
  float cap, cap_k, cap_r;    // with a positive cap, products s give cap * tanh(x), x = s * cap_k, e^2x = 2^(s * cap_r), in log2 units
  float cap_small, cap_p[3];  // for |s| below cap_small (0: never) that is s (pre + cap_p[0] t + cap_p[1] t^2 + cap_p[2] t^3), t = s^2
  uint32_t tiles;             // an upper bound of the query tiles of a KV head
  uint32_t by_height;         // 1: the tiles of all sequences in the order of the keys that they see, not sequence by sequence
  uint32_t places;            // workgroups of a KV head that run at once, where keys may be cut into parts; 0: they are not
  uint32_t most_items;        // parts of a KV head's tiles that the workspace has room for, where any are cut
  uint64_t parts_at;
};

// Rows of (token, query head of a KV head) in a query tile; the most sequences of a call whose keys may be cut into parts, and the
// keys from which that is looked at; what writing and joining a part of 128 rows costs, in tiles of 64 keys.
constexpr uint32_t kPromptRows = 128, kPromptCutSequences = 1024, kPromptCutKeys = 1024, kPromptCut = 7;
struct PromptPlan {
  uint32_t tiles, by_height, places, most_items;
  uint64_t parts_at, ws_floats;
};
// What the host decides. Workgroups take whole query tiles where these are enough for four turns of every workgroup place (two on a
// compute unit), or fill half of the places and belong to whole prompts, whose tiles grow in number as they grow in length. Else, where
// tiles may be long, the lengths decide on the device whether keys are cut: two launches more, about 10 us (eight sequences of five
// drafted tokens behind up to 32,000: 123 us; 500 and more if a workgroup has the longest by itself). From 1,024 keys on: 20 queries over
// 1,500 keys of 8 heads of 128 take 18 us cut and 34 uncut, over 700 keys about 17 either way.
//
// The host knows the keys of all sequences together, not the longest, and errs both ways. A call of short sequences with 1,024 keys and
// more in all is looked at for nothing: seven of 29 queries over 385 keys 21.7 us and 15.0 if it were not, five of 100 over 600
// 26.7 and 19.8 (8 KV and 32 query heads of 128). One long sequence among many tiles is not cut: a chunk of 8,192 tokens and 31
// drafts behind up to 2,000 take 567 us, with one more draft behind 32,000 1,098. The places are those of heads of 128, two workgroups on
// a compute unit; three of heads of 64 run there.
//
// Whole tiles of several sequences come in the order of their keys where a place has fewer than four: the longest do not come last (16
// sequences of 12 heads in a window, one or two tiles a place: 27.8 us, sequence by sequence 30.3). With more, the search for a tile, 0.9
// us each, costs what the shorter end gains (ten tiles a place: 415 us, sequence by sequence 410).
inline PromptPlan prompt_plan(uint32_t rows, uint32_t keys, uint32_t window, uint32_t sequences, uint32_t kv_heads, uint32_t nq,
                              uint32_t dim, uint32_t cus) {
  PromptPlan p{};
  p.tiles = (uint32_t)((uint64_t)rows * nq / kPromptRows) + (sequences < rows ? sequences : rows);
  const uint32_t places = 2 * cus, seen = window && window < keys ? window : keys;
  const uint64_t tiles = (uint64_t)p.tiles * kv_heads;
  p.by_height = sequences > 1 && tiles < 4ull * places;
  if (tiles >= 4ull * places || (tiles >= places / 2 && keys < 2ull * rows)) return p;
  if (sequences > kPromptCutSequences || seen < kPromptCutKeys || kv_heads > places) return p;
  p.places = places / kv_heads;
  p.most_items = 4 * p.places;
  p.parts_at = (sequences * 5 + 2 + 3) / 4 * 4;
  p.ws_floats = p.parts_at + (uint64_t)p.most_items * kv_heads * kPromptRows * (dim + 2);
  return p;
}

#define PITCH_DECLARE_PROMPT(D)                                                             \
  hipError_t launch_prompt_d##D##_io1(const PromptArgs& a, hipStream_t s);                   \
  hipError_t launch_prompt_d##D##_io2(const PromptArgs& a, hipStream_t s);
PITCH_DECLARE_PROMPT(64)
PITCH_DECLARE_PROMPT(128)
#undef PITCH_DECLARE_PROMPT

}  // namespace pitch
