// Arguments and launches of the pages' bookkeeping (pitch_pages.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace pitch {

// Page tables of sequences over a pool, and where the kernels of a call leave what the next one reads (all in the workspace).
struct PagesTables {
  int32_t* tables;      // [sequences][width]
  int32_t* lengths;     // [sequences] tokens
  int32_t* references;  // [pages]; a page is free where it is not positive
  int32_t* missing;     // or null
  uint32_t width, sequences, pages, page_size;
  uint32_t most_tokens;            // width * page_size
  uint32_t segments, segment;      // the pool in segments of as many pages, which a workgroup counts
  uint32_t* counts;                // [segments] pages found in each
  uint32_t* plan;                  // eight words and five arrays of `sequences`, as each operator says
  uint32_t* room;                  // the operators' long arrays
};

// Words of the workspace: counts, plan, room (fork: the tables as they were; compact: three arrays of `pages`).
constexpr uint32_t kPagesMostSegments = 4096, kPagesLeastSegment = 256;
constexpr uint32_t pages_segment(uint64_t pages) {
  const uint64_t each = (pages + kPagesMostSegments - 1) / kPagesMostSegments;
  return (uint32_t)((each + kPagesLeastSegment - 1) / kPagesLeastSegment * kPagesLeastSegment);
}
constexpr uint64_t pages_plan_words(uint64_t sequences) { return 8 + 5 * sequences; }
constexpr uint64_t pages_workspace_words(uint64_t pages, uint64_t sequences, uint64_t width) {
  return kPagesMostSegments + pages_plan_words(sequences) + (sequences * width > 3 * pages ? sequences * width : 3 * pages);
}

struct PagesReserveArgs {
  PagesTables t;
  const int32_t* new_tokens;  // [sequences]
  int64_t* slots;             // [capacity]
  int64_t* positions;         // [capacity] or null
  uint32_t capacity;
};

struct PagesTrimArgs {
  PagesTables t;
  const int32_t* keep;  // [sequences]
};

// A layer's pool for the copies: keys' codes and scales, values' codes and scales.
struct PagesLayer {
  uint8_t* base[4];
  uint32_t page_stride;    // vectors from page to page
  uint32_t kv_heads;
  uint32_t row_bytes[2];   // bytes of codes of a vector, keys and values
  uint32_t head_major;
};
constexpr uint32_t kPagesLayers = 48;  // of a launch: its arguments hold them
// Bytes of a layer's page that a workgroup copies at a time. One index over all pieces of a page instead, divided for each: 642 us where
// slices of buffers take 408 to 470 (1.1 GB). Four pieces read before one is written, or four times as many workgroups: no change to 2
// %.
constexpr uint32_t kPagesSlice = 1u << 16;
struct PagesCopyArgs {
  const uint32_t* count;   // pages to copy
  const uint32_t* source;  // page numbers
  const uint32_t* target;
  const uint32_t* tokens;  // of each page, or null: all of the page
  uint32_t backwards;      // 1: sources in descending order of the targets' index (source[count - 1 - i])
  uint32_t page_size, layers, slices, most;  // slices of a layer's page; the most pages there can be
  uint32_t parts;          // 4: a unit of work is one of a layer's four buffers (set by the launcher)
  PagesLayer layer[kPagesLayers];
};

struct PagesForkArgs {
  PagesTables t;
  const int32_t* parents;  // [sequences]
};

struct PagesCompactArgs {
  PagesTables t;
  int32_t* mapping;  // [pages] or null
  int32_t* used;     // or null
};

hipError_t launch_pages_reserve(const PagesReserveArgs& a, hipStream_t s);
hipError_t launch_pages_trim(const PagesTrimArgs& a, hipStream_t s);
// The bookkeeping; the copies are launched behind it, layer by layer, with what these calls leave in the workspace.
hipError_t launch_pages_fork(const PagesForkArgs& a, PagesCopyArgs* copies, hipStream_t s);
hipError_t launch_pages_compact(const PagesCompactArgs& a, PagesCopyArgs* copies, hipStream_t s);
hipError_t launch_pages_copy(const PagesCopyArgs& a, uint32_t cus, hipStream_t s);

}  // namespace pitch
