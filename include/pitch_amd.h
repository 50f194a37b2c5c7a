/*
 * pitch_amd.h - C ABI of the MI355X (gfx950) KV-cache codec library libpitch_amd.so.
 *
 * Drop-in boundary for the codec path of SwiftCham/PITCH. Each entry point below replaces one operator of
 * the reference's Swift surface (file:line in /root/reference) with the same argument meaning, the same
 * validation and the same error categories. Buffers are device pointers owned by the caller; every offset
 * is in bytes and must be a non-negative multiple of 4; every length is the byte size of the whole buffer
 * starting at the pointer, so the library can perform the reference's "needs N bytes after offset" check.
 * The enqueue functions validate, launch on the given HIP stream and return without waiting, as the
 * reference's enqueue* calls encode into the caller's command buffer (Sources/PITCH/PITCH.swift:136-165).
 *
 * Deviation: counts and offsets are 64-bit, so a single call may cover count * dim >= 2^32 elements,
 * which the reference rejects (Sources/PITCH/Core/Codec.swift:30-32). Per-channel calls require
 * count < 2^32 tokens.
 */
#ifndef PITCH_AMD_H
#define PITCH_AMD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Return codes, mirroring PITCHError (Sources/PITCH/Core/PITCHError.swift:10-19). */
#define PITCH_OK 0
#define PITCH_ERR_INVALID_INPUT (-1)          /* PITCHError.invalidInput */
#define PITCH_ERR_INVALID_BIT_WIDTH (-2)      /* PITCHError.invalidBitWidth */
#define PITCH_ERR_INVALID_DIMENSION (-3)      /* PITCHError.invalidDimension */
#define PITCH_ERR_CONFIGURATION_MISMATCH (-4) /* PITCHError.configurationMismatch */
#define PITCH_ERR_ENCODING_FAILED (-5)        /* PITCHError.encodingFailed */
#define PITCH_ERR_DECODING_FAILED (-6)        /* PITCHError.decodingFailed */
#define PITCH_ERR_DEVICE_UNAVAILABLE (-7)     /* PITCHError.metalNotSupported (no usable GPU) */

/* QuantMethod (Sources/PITCH/Models/QuantMethod.swift:8-11). */
#define PITCH_METHOD_TURBO 0u
#define PITCH_METHOD_POLAR 1u

/* Element type of the uncompressed vectors of the *_io entry points: what encode reads and decode writes.
 * The reference's codec is float32 only ("Inputs and outputs are float32; models that keep caches in fp16 or
 * bf16 need a conversion", README.md:97). 16-bit inputs are widened to float32 exactly and encoded as the
 * float32 entry point encodes them; decoded values are the float32 entry point's results rounded to nearest
 * even (overflow to infinity). Codes, scales and ranges are the same bytes for every element type. */
#define PITCH_IO_F32 0u
#define PITCH_IO_F16 1u
#define PITCH_IO_BF16 2u

/* Default rotation seed, PITCH.defaultSeed = 0x50495443 (Sources/PITCH/PITCH.swift:18). */
#define PITCH_DEFAULT_SEED 0x50495443u

/* QuantConfig (Sources/PITCH/Models/QuantConfig.swift:11-60); same 16-byte layout as BatchParams minus
 * count (Sources/PITCH/Core/Codec.swift:12-17). */
typedef struct pitch_config {
  uint32_t method; /* PITCH_METHOD_TURBO or PITCH_METHOD_POLAR */
  uint32_t dim;    /* power of two, 2..1024 */
  uint32_t bits;   /* 2..8 */
  uint32_t seed;   /* rotation seed */
} pitch_config_t;

/* ChannelQuantConfig (Sources/PITCH/PerChannel.swift:15-70). */
typedef struct pitch_channel_config {
  uint32_t dim;        /* channels per token, 1..1024 (any value) */
  uint32_t bits;       /* 2..8 */
  uint32_t group_size; /* tokens per group, 1..65536 */
  uint32_t reserved;   /* 0 */
} pitch_channel_config_t;

/* Library version as 0xMMmmpp. */
uint32_t pitch_version(void);

/* Message of the last failed call on this thread ("" if none). */
const char* pitch_last_error(void);

/* Validates and fills a QuantConfig; *code_stride = ceil(dim * bits / 32) * 4 bytes.
 * Replaces PITCH.config(method:dim:bits:) / QuantConfig.init (Sources/PITCH/PITCH.swift:53-55,
 * Sources/PITCH/Models/QuantConfig.swift:24-35,47). code_stride may be NULL. */
int pitch_config(uint32_t method, uint32_t dim, uint32_t bits, uint32_t seed, pitch_config_t* out,
                 uint32_t* code_stride);

/* Validates and fills a ChannelQuantConfig; *code_stride = ceil(dim * bits / 32) * 4 bytes and
 * *range_stride = 4 * dim bytes (fp16 minima then maxima per group).
 * Replaces PITCH.channelConfig(dim:bits:groupSize:) / ChannelQuantConfig.init
 * (Sources/PITCH/PerChannel.swift:184-187,30-43,55,58). Either output stride may be NULL. */
int pitch_channel_config(uint32_t dim, uint32_t bits, uint32_t group_size, pitch_channel_config_t* out,
                         uint32_t* code_stride, uint32_t* range_stride);

/* Encodes count contiguous fp32 vectors: writes count * code_stride bytes of packed codes and count fp32
 * scales (the norm for TurboQuant, the largest pair radius for PolarQuant).
 * Replaces PITCH.enqueueEncode(input:inputOffset:codes:codesOffset:scales:scalesOffset:count:config:
 * commandBuffer:) (Sources/PITCH/PITCH.swift:144-153 -> Sources/PITCH/Core/Codec.swift:70-103). */
int pitch_enqueue_encode(const pitch_config_t* config, const void* input, uint64_t input_bytes,
                         uint64_t input_offset, void* codes, uint64_t codes_bytes, uint64_t codes_offset,
                         void* scales, uint64_t scales_bytes, uint64_t scales_offset, uint64_t count,
                         void* stream /* hipStream_t; NULL = default stream */);

/* pitch_enqueue_encode with input elements of type io_type (PITCH_IO_*): the input buffer needs
 * count * dim * element-size bytes after its offset. Extends PITCH.enqueueEncode (Sources/PITCH/PITCH.swift:
 * 144-153) past its float32-only input (README.md:97). */
int pitch_enqueue_encode_io(const pitch_config_t* config, uint32_t io_type, const void* input,
                            uint64_t input_bytes, uint64_t input_offset, void* codes, uint64_t codes_bytes,
                            uint64_t codes_offset, void* scales, uint64_t scales_bytes, uint64_t scales_offset,
                            uint64_t count, void* stream);

/* One segment of a batched encode: count vectors of the batch's element type from input + input_offset, their
 * codes to codes + codes_offset and their scales to scales + scales_offset (byte offsets and sizes as in
 * pitch_enqueue_encode_io). */
typedef struct pitch_encode_item {
  const void* input;
  uint64_t input_bytes, input_offset;
  void* codes;
  uint64_t codes_bytes, codes_offset;
  void* scales;
  uint64_t scales_bytes, scales_offset;
  uint64_t count;
} pitch_encode_item_t;

/* Encodes n_items independent segments with one configuration and element type io_type (PITCH_IO_*) in as few
 * launches as it can (one per 32 segments), with the same codes and scales as one pitch_enqueue_encode_io per
 * segment. Every segment is validated as that call validates it, before anything is launched. For the
 * decode-phase append of a token's vectors across many layers: README.md:65-71 issues one
 * PITCH.enqueueEncode (Sources/PITCH/PITCH.swift:144-153) per cache, and a launch costs several microseconds
 * of host time here, so appending to 32 layers' caches through one call takes a fraction of 32 calls' time. */
int pitch_enqueue_encode_batch(const pitch_config_t* config, uint32_t io_type, const pitch_encode_item_t* items,
                               uint32_t n_items, void* stream);

/* Decodes count vectors into count * dim fp32 values. A vector's decoded bytes do not depend on the call: any count,
 * offset or batch that contains it writes the same bytes (every decode kernel runs the same arithmetic in the same
 * order; only the grid differs with the call's size).
 * Replaces PITCH.enqueueDecode(codes:codesOffset:scales:scalesOffset:output:outputOffset:count:config:
 * commandBuffer:) (Sources/PITCH/PITCH.swift:156-165 -> Sources/PITCH/Core/Codec.swift:107-140). */
int pitch_enqueue_decode(const pitch_config_t* config, const void* codes, uint64_t codes_bytes,
                         uint64_t codes_offset, const void* scales, uint64_t scales_bytes,
                         uint64_t scales_offset, void* output, uint64_t output_bytes, uint64_t output_offset,
                         uint64_t count, void* stream);

/* pitch_enqueue_decode writing elements of type io_type (PITCH_IO_*). Extends PITCH.enqueueDecode
 * (Sources/PITCH/PITCH.swift:156-165) past its float32-only output (README.md:97). */
int pitch_enqueue_decode_io(const pitch_config_t* config, uint32_t io_type, const void* codes,
                            uint64_t codes_bytes, uint64_t codes_offset, const void* scales, uint64_t scales_bytes,
                            uint64_t scales_offset, void* output, uint64_t output_bytes, uint64_t output_offset,
                            uint64_t count, void* stream);

/* One segment of a batched decode: count vectors' codes from codes + codes_offset and scales from scales +
 * scales_offset, decoded to output + output_offset (byte offsets and sizes as in pitch_enqueue_decode_io). */
typedef struct pitch_decode_item {
  const void* codes;
  uint64_t codes_bytes, codes_offset;
  const void* scales;
  uint64_t scales_bytes, scales_offset;
  void* output;
  uint64_t output_bytes, output_offset;
  uint64_t count;
} pitch_decode_item_t;

/* Decodes n_items independent segments with one configuration and output element type io_type (PITCH_IO_*) in as
 * few launches as it can (one per 32 segments of fewer than 2^18 vectors; a longer segment gets the launch of a
 * single call), writing the same bytes as one pitch_enqueue_decode_io per segment.
 * Every segment is validated as that call validates it, before anything is launched. For a model's per-layer
 * decodes (README.md:65-76 decodes each layer's cache with its own PITCH.enqueueDecode, Sources/PITCH/PITCH.swift:
 * 156-165): a layer of one decode step is a few tens of thousands of vectors, too few to fill the GPU alone, and
 * one call over every layer's cache runs at the rate of a bulk decode. */
int pitch_enqueue_decode_batch(const pitch_config_t* config, uint32_t io_type, const pitch_decode_item_t* items,
                               uint32_t n_items, void* stream);

/* Key-projection bias removal for the per-vector methods (reference/mechanism_eval.py:88-97,113-116: a model
 * whose key projection adds a bias b before RoPE has keys k = R_t W x + R_t b; compressing k - R_t b and adding
 * R_t b back restores the per-vector methods, README.md:28; "not yet built into the kernels", README.md:100).
 * Vector v of a call is token first_position + v / heads of head v % heads (a token-major [t][h] cache) and
 * carries o = b_h * cos_t + rotate_half(b_h) * sin_t, rotate_half(x) = (-x[dim/2:], x[:dim/2]), in float32 with
 * each product and the sum rounded once. All three tables are fp32 device memory. */
typedef struct pitch_key_bias {
  const void* bias;        /* [heads][dim]: the key projection's bias per KV head, before RoPE */
  uint64_t bias_bytes;
  const void* cos;         /* [positions][dim]: the model's RoPE cosines (rotate_half layout) */
  const void* sin;         /* [positions][dim]: the model's RoPE sines */
  uint64_t table_bytes;    /* bytes of cos and of sin each; positions = table_bytes / (4 * dim) */
  uint64_t first_position; /* position of the call's first token */
  uint32_t heads;          /* KV heads per token */
  uint32_t reserved;       /* 0 */
} pitch_key_bias_t;

/* pitch_enqueue_encode of x - o (fp32 input): the scales are the norms (or rmax) of the debiased keys. */
int pitch_enqueue_encode_key_bias(const pitch_config_t* config, const pitch_key_bias_t* key_bias, const void* input,
                                  uint64_t input_bytes, uint64_t input_offset, void* codes, uint64_t codes_bytes,
                                  uint64_t codes_offset, void* scales, uint64_t scales_bytes, uint64_t scales_offset,
                                  uint64_t count, void* stream);

/* pitch_enqueue_decode followed by + o (fp32 output). */
int pitch_enqueue_decode_key_bias(const pitch_config_t* config, const pitch_key_bias_t* key_bias, const void* codes,
                                  uint64_t codes_bytes, uint64_t codes_offset, const void* scales,
                                  uint64_t scales_bytes, uint64_t scales_offset, void* output, uint64_t output_bytes,
                                  uint64_t output_offset, uint64_t count, void* stream);

/* Encodes count tokens of one head's keys (token-major, dim channels) per channel over groups of
 * group_size tokens: writes count * code_stride bytes of codes and ceil(count / group_size) * range_stride
 * bytes of fp16 ranges laid out [group][min row of dim][max row of dim].
 * Replaces PITCH.enqueuePerChannelEncode(input:inputOffset:codes:codesOffset:ranges:rangesOffset:count:
 * config:commandBuffer:) (Sources/PITCH/PerChannel.swift:251-260 -> :338-363). */
int pitch_enqueue_channel_encode(const pitch_channel_config_t* config, const void* input,
                                 uint64_t input_bytes, uint64_t input_offset, void* codes,
                                 uint64_t codes_bytes, uint64_t codes_offset, void* ranges,
                                 uint64_t ranges_bytes, uint64_t ranges_offset, uint64_t count,
                                 void* stream);

/* pitch_enqueue_channel_encode with key elements of type io_type (PITCH_IO_*). Extends
 * PITCH.enqueuePerChannelEncode (Sources/PITCH/PerChannel.swift:251-260) past float32-only input
 * (README.md:97). */
int pitch_enqueue_channel_encode_io(const pitch_channel_config_t* config, uint32_t io_type, const void* input,
                                    uint64_t input_bytes, uint64_t input_offset, void* codes,
                                    uint64_t codes_bytes, uint64_t codes_offset, void* ranges,
                                    uint64_t ranges_bytes, uint64_t ranges_offset, uint64_t count,
                                    void* stream);

/* Decodes count per-channel tokens into count * dim fp32 values.
 * Replaces PITCH.enqueuePerChannelDecode(codes:codesOffset:ranges:rangesOffset:output:outputOffset:count:
 * config:commandBuffer:) (Sources/PITCH/PerChannel.swift:261-270 -> :365-389). */
int pitch_enqueue_channel_decode(const pitch_channel_config_t* config, const void* codes,
                                 uint64_t codes_bytes, uint64_t codes_offset, const void* ranges,
                                 uint64_t ranges_bytes, uint64_t ranges_offset, void* output,
                                 uint64_t output_bytes, uint64_t output_offset, uint64_t count,
                                 void* stream);

/* pitch_enqueue_channel_decode writing elements of type io_type (PITCH_IO_*). Extends
 * PITCH.enqueuePerChannelDecode (Sources/PITCH/PerChannel.swift:261-270) past float32-only output
 * (README.md:97). */
int pitch_enqueue_channel_decode_io(const pitch_channel_config_t* config, uint32_t io_type, const void* codes,
                                    uint64_t codes_bytes, uint64_t codes_offset, const void* ranges,
                                    uint64_t ranges_bytes, uint64_t ranges_offset, void* output,
                                    uint64_t output_bytes, uint64_t output_offset, uint64_t count,
                                    void* stream);

/* Appends new_tokens tokens to one head's per-channel cache that already holds total_tokens - new_tokens of
 * them, re-encoding every group the new tokens touch: a partial last group is encoded again over all of its
 * tokens, so its fp16 ranges always cover the tokens it holds ("the newest, partial group can be kept in full
 * precision or re-encoded as it grows", README.md:85; the reference's ChannelCompressedBlock.append refuses
 * to append after a partial group, Sources/PITCH/PerChannel.swift:120-130). input holds the head's keys of
 * tokens [0, total_tokens) in the element type io_type (only the touched groups are read); codes and ranges
 * are the head's whole cache buffers, laid out as pitch_enqueue_channel_encode writes them. The result is
 * byte for byte that of one pitch_enqueue_channel_encode_io over all total_tokens tokens. */
int pitch_enqueue_channel_append(const pitch_channel_config_t* config, uint32_t io_type, const void* input,
                                 uint64_t input_bytes, uint64_t input_offset, void* codes, uint64_t codes_bytes,
                                 uint64_t codes_offset, void* ranges, uint64_t ranges_bytes, uint64_t ranges_offset,
                                 uint64_t total_tokens, uint64_t new_tokens, void* stream);

/* Decode-phase attention over compressed caches (no counterpart in the reference: it evaluates attention on
 * decoded caches, reference/attention_extra.py:70-74, and names decoding inside attention as its next step,
 * README.md:96). For each of kv_heads KV heads and each of its q_per_kv query heads:
 *   out = softmax(scale * q . K^T) V,  lse = log sum exp(scale * q . K^T)  (natural log)
 * where K and V are the decodes of the per-vector codes (TurboQuant or PolarQuant, any bit width 2..8, key and
 * value configs may differ in method, bits and seed but not in dimension, which must be 64 or 128). The codes
 * are read as stored; no decoded vector is written. Queries and outputs are fp32 [kv_heads][q_per_kv][dim].
 * The cache vector of (KV head h, token t) is t * token_stride + h * head_stride, in units of vectors, for
 * both the codes (code_stride bytes each) and the scales (4 bytes each): a token-major [t][h] cache has
 * token_stride = number of heads and head_stride = 1; a head-major [h][t] one has token_stride = 1. */
typedef struct pitch_attention_desc {
  uint32_t q_per_kv;     /* query heads per KV head (grouped-query attention), 1..8 */
  uint32_t kv_heads;     /* KV heads in the call, 1..65535 */
  uint64_t tokens;       /* cached tokens per KV head, >= 1 */
  uint64_t token_stride; /* vectors between consecutive tokens of one head */
  uint64_t head_stride;  /* vectors between consecutive KV heads */
  float scale;           /* softmax scale applied to q . k, e.g. 1 / sqrt(dim) */
  uint32_t reserved;     /* 0 */
} pitch_attention_desc_t;

/* Bytes of device workspace pitch_enqueue_attention_decode needs for these arguments. */
int pitch_attention_workspace_size(const pitch_config_t* key_config, const pitch_config_t* value_config,
                                   const pitch_attention_desc_t* desc, uint64_t* bytes);

/* Enqueues the attention described above on the stream. lse may be NULL. The workspace (at least
 * pitch_attention_workspace_size bytes of device memory) must not be used by another call until this one has
 * completed on the stream. */
int pitch_enqueue_attention_decode(const pitch_config_t* key_config, const pitch_config_t* value_config,
                                   const pitch_attention_desc_t* desc, const void* q, uint64_t q_bytes,
                                   uint64_t q_offset, const void* key_codes, uint64_t key_codes_bytes,
                                   uint64_t key_codes_offset, const void* key_scales, uint64_t key_scales_bytes,
                                   uint64_t key_scales_offset, const void* value_codes, uint64_t value_codes_bytes,
                                   uint64_t value_codes_offset, const void* value_scales,
                                   uint64_t value_scales_bytes, uint64_t value_scales_offset, void* output,
                                   uint64_t output_bytes, uint64_t output_offset, void* lse, uint64_t lse_bytes,
                                   uint64_t lse_offset, void* workspace, uint64_t workspace_bytes, void* stream);

/* pitch_enqueue_attention_decode over a key cache encoded with key-bias removal (pitch_enqueue_encode_key_bias):
 * the scores are q . (decode(k) + o_t) with o_t = b_h cos_t + rotate_half(b_h) sin_t, the cache's k - o_t
 * restored as pitch_enqueue_decode_key_bias restores it (reference/mechanism_eval.py:113-116: the keys are
 * compress(k - R_t b) + R_t b). key_bias->heads must equal desc->kv_heads (row h of the bias is KV head h) and
 * token t of the cache is at position key_bias->first_position + t, so the tables need first_position + tokens
 * rows. Per-vector keys only (per-channel keys need no bias removal). Extends the fused attention, which the
 * reference does not have (README.md:96, 100). */
int pitch_enqueue_attention_decode_key_bias(
    const pitch_config_t* key_config, const pitch_config_t* value_config, const pitch_attention_desc_t* desc,
    const pitch_key_bias_t* key_bias, const void* q, uint64_t q_bytes, uint64_t q_offset, const void* key_codes,
    uint64_t key_codes_bytes, uint64_t key_codes_offset, const void* key_scales, uint64_t key_scales_bytes,
    uint64_t key_scales_offset, const void* value_codes, uint64_t value_codes_bytes, uint64_t value_codes_offset,
    const void* value_scales, uint64_t value_scales_bytes, uint64_t value_scales_offset, void* output,
    uint64_t output_bytes, uint64_t output_offset, void* lse, uint64_t lse_bytes, uint64_t lse_offset,
    void* workspace, uint64_t workspace_bytes, void* stream);

/* Largest workspace pitch_enqueue_attention_decode_noalloc can serve, in bytes (32 MiB: e.g. 8 KV heads x 4 query
 * heads x 131072 tokens at dim 128 needs 18.9 MB). */
#define PITCH_NOALLOC_SCRATCH_BYTES (32ull << 20)

/* pitch_enqueue_attention_decode without a workspace argument, for callers that cannot allocate device memory
 * (code under HIP graph capture, tight serving loops, harnesses that forbid hipMalloc). It has no counterpart in
 * the reference. The workspace is a scratch array compiled into the library, one per device, held until the process
 * ends; the call allocates nothing. Calls whose workspace (pitch_attention_workspace_size) exceeds
 * PITCH_NOALLOC_SCRATCH_BYTES fail with PITCH_ERR_INVALID_INPUT before any work is issued. Every call on a device
 * shares that device's array: calls that overlap on one device (on different streams, or from different threads
 * without ordering) race and must not be issued; calls ordered on one stream are safe. Results are otherwise those
 * of pitch_enqueue_attention_decode on the same arguments. The array's device address is looked up (one
 * hipGetSymbolAddress, no allocation) by the first call of any pitch_enqueue_* entry point on the device, so a caller
 * that captures a HIP graph makes that lookup outside the capture by issuing any one call on the device first. */
int pitch_enqueue_attention_decode_noalloc(const pitch_config_t* key_config, const pitch_config_t* value_config,
                                           const pitch_attention_desc_t* desc, const void* q, uint64_t q_bytes,
                                           uint64_t q_offset, const void* key_codes, uint64_t key_codes_bytes,
                                           uint64_t key_codes_offset, const void* key_scales,
                                           uint64_t key_scales_bytes, uint64_t key_scales_offset,
                                           const void* value_codes, uint64_t value_codes_bytes,
                                           uint64_t value_codes_offset, const void* value_scales,
                                           uint64_t value_scales_bytes, uint64_t value_scales_offset, void* output,
                                           uint64_t output_bytes, uint64_t output_offset, void* lse,
                                           uint64_t lse_bytes, uint64_t lse_offset, void* stream);

/* pitch_enqueue_attention_decode with per-channel (KIVI) keys and per-vector values: the configuration the
 * reference recommends for models whose key projection has a bias (README.md:30) and evaluates as
 * "kivi_K{b}_turboV{b}" (reference/attention_extra.py:57-59). Keys decode as f32(c) * step + lo per group and
 * channel (reference/pitch_reference.py:165-174). The key cache is head-major, as per-head
 * pitch_enqueue_channel_encode calls write it: codes of (head h, token t) at row h * head_stride + t, fp16 ranges
 * of (h, group g) at group h * head_stride / group_size + g; desc->token_stride must be 1 and, with more than one
 * KV head, head_stride a multiple of the group size holding the tokens (one head: head_stride is ignored). The
 * values use the same rows. The group size must be a multiple of 64. */
int pitch_attention_channel_keys_workspace_size(const pitch_channel_config_t* key_config,
                                                const pitch_config_t* value_config, const pitch_attention_desc_t* desc,
                                                uint64_t* bytes);
int pitch_enqueue_attention_decode_channel_keys(
    const pitch_channel_config_t* key_config, const pitch_config_t* value_config, const pitch_attention_desc_t* desc,
    const void* q, uint64_t q_bytes, uint64_t q_offset, const void* key_codes, uint64_t key_codes_bytes,
    uint64_t key_codes_offset, const void* key_ranges, uint64_t key_ranges_bytes, uint64_t key_ranges_offset,
    const void* value_codes, uint64_t value_codes_bytes, uint64_t value_codes_offset, const void* value_scales,
    uint64_t value_scales_bytes, uint64_t value_scales_offset, void* output, uint64_t output_bytes,
    uint64_t output_offset, void* lse, uint64_t lse_bytes, uint64_t lse_offset, void* workspace,
    uint64_t workspace_bytes, void* stream);

/* ------------------------------------------------------------------------------------------------------------------
 * Paged caches. The reference keeps one sequence's cache in contiguous buffers (README.md:65-76); a program that serves
 * many sequences keeps their keys and values in the pages of one pool and a table of pages per sequence. The pages hold
 * per-vector codes and scales as pitch_enqueue_encode_io writes them. A pool has `pages` pages of page_size token slots
 * for each of kv_heads KV heads. The vector of (page p, head h, slot s), for codes (code_stride bytes each) and scales
 * (4 bytes each) alike, is p * page_stride + h * page_size + s (PITCH_PAGES_HEAD_MAJOR) or p * page_stride +
 * s * kv_heads + h (PITCH_PAGES_TOKEN_MAJOR). The three operators below are captured into graphs like the others: they
 * launch kernels only. What lies in device memory (slots, positions, page tables, lengths) cannot be checked before the
 * launch; the kernels check every value against the pool and the tables and take none on trust. */
#define PITCH_PAGES_HEAD_MAJOR 0u
#define PITCH_PAGES_TOKEN_MAJOR 1u

typedef struct pitch_paged_cache {
  pitch_config_t key_config, value_config; /* one dimension, 64 or 128; methods, bit widths and seeds may differ */
  void* key_codes;
  uint64_t key_codes_bytes;
  void* key_scales;
  uint64_t key_scales_bytes;
  void* value_codes;
  uint64_t value_codes_bytes;
  void* value_scales;
  uint64_t value_scales_bytes;
  uint64_t pages;       /* pages * page_size < 2^32 */
  uint64_t page_stride; /* vectors from page to page, at least kv_heads * page_size, below 2^25 */
  uint32_t page_size;   /* token slots of a page: a multiple of 16, at most 65536 */
  uint32_t kv_heads;    /* 1..65535 */
  uint32_t layout;      /* PITCH_PAGES_* */
  uint32_t reserved;    /* 0 */
} pitch_paged_cache_t;

/* The vectors of a paged call: coordinate i of (token t, head h) is element t * token_stride + h * head_stride + i of
 * data, of the call's io_type. For 16-bit types data and both strides are multiples of 4 bytes. bytes is what the buffer
 * holds from data on. */
typedef struct pitch_paged_vectors {
  void* data;
  uint64_t bytes;
  uint64_t token_stride, head_stride; /* elements */
} pitch_paged_vectors_t;

/* Writes tokens to the cache. Token t's keys and values [kv_heads][dim] are encoded into slot slots[t] = page * page_size
 * + slot; a token whose slot lies outside the pool (-1 for the padding of a batch) is not written. Two tokens of a call
 * must not have the same slot (what such a slot holds afterwards is undefined).
 * With key_norm, a key is x / sqrt(mean(x^2) + eps) times the weights (dim elements of io_type); with positions, its first
 * rotary_dim coordinates are then rotated: x * cos[p] + rotate_half(x) * sin[p], rotate_half over these coordinates
 * (-x[rotary_dim / 2:], x[:rotary_dim / 2]), p = positions[t], cos and sin [rows][rotary_dim] fp32. A key is not rounded
 * between these steps and its codes. Queries (q_heads per token, 0 for none) are normed with query_norm and rotated alike,
 * in float32, and written to queries_out in io_type; they may be written in place (queries_out the same vectors), and else
 * queries_out must not overlap what the call reads. A token whose position lies outside the tables is not written, nor are
 * its queries. Without norm and positions the codes and scales are those of
 * pitch_enqueue_encode_io, up to values within 1e-11 of an edge between two codes (relative to the vector's norm). A vector
 * with an element that is not finite gets a scale that is not finite.
 * For a decode step's or a prompt's write (README.md:65-71 appends with one PITCH.enqueueEncode per cache). */
typedef struct pitch_paged_append {
  uint32_t io_type; /* PITCH_IO_*: keys, values, queries, norm weights */
  uint32_t q_heads;
  uint64_t tokens;  /* at least 1; tokens * heads < 2^31 */
  pitch_paged_vectors_t keys, values, queries, queries_out;
  const void* slots;     /* int64 [tokens] */
  uint64_t slots_bytes;
  const void* positions; /* int64 [tokens], or null: no rotation */
  uint64_t positions_bytes;
  const void* cos;
  const void* sin;
  uint64_t table_bytes;  /* bytes of cos and of sin each */
  const void* query_norm; /* or null */
  uint64_t query_norm_bytes;
  const void* key_norm;   /* or null */
  uint64_t key_norm_bytes;
  uint32_t rotary_dim;    /* a multiple of 16, at most dim; 0 without positions */
  float eps;              /* at least 0 */
} pitch_paged_append_t;
int pitch_enqueue_paged_append(const pitch_paged_cache_t* cache, const pitch_paged_append_t* call, void* stream);

/* Reads tokens back. Row r of the outputs, row_starts[b] <= r < row_starts[b + 1], is token first_tokens[b] + r -
 * row_starts[b] of sequence b, found in page block_tables[b][token / page_size]; it is decoded as pitch_enqueue_decode_io
 * decodes it. row_starts does not decrease. Rows outside the sequences' ranges, and rows whose page lies outside the pool or
 * the table, are left as they were. keys or values may have null data (not read back); their token strides are at most 2^22
 * elements, and they share no element. */
typedef struct pitch_paged_decode {
  uint32_t io_type;   /* PITCH_IO_* of the outputs */
  uint32_t sequences; /* at least 1 */
  uint64_t rows;      /* rows of the outputs, at least 1; rows * ceil(kv_heads / 4) <= 2^28 */
  const void* block_tables; /* int32 [sequences][table_width] */
  uint64_t block_tables_bytes;
  uint64_t table_width; /* at least 1 */
  const void* row_starts; /* int32 [sequences + 1] */
  uint64_t row_starts_bytes;
  const void* first_tokens; /* int32 [sequences], or null: 0 */
  uint64_t first_tokens_bytes;
  pitch_paged_vectors_t keys, values;
} pitch_paged_decode_t;
int pitch_enqueue_paged_decode(const pitch_paged_cache_t* cache, const pitch_paged_decode_t* call, void* stream);

/* Attention of one new token of every sequence over its pages. Sequence b has lengths[b] = L cached tokens, the new one
 * among them; query head h of its q_per_kv * kv_heads heads reads KV head h / q_per_kv:
 *   out = softmax(z) V,  lse = log sum exp(z),  z_t = cap(scale * q . k_t) + slopes[h] * (t - (L - 1))
 * over the tokens t of [0, L), of [L - window, L) with a window; cap(x) = softcap * tanh(x / softcap), x itself with
 * softcap 0. Queries and outputs are float16 or bfloat16: the products run on the 16-bit matrix cores. With float16 every operand
 * has two float16 parts and the outputs are the exact result's rounding; with bfloat16 the vectors that the codes stand for
 * have one (11 bits, PolarQuant of 5 to 8 bits about 10), which moves an lse by up to 2e-3. A length of 0 or
 * less gives zeros and an lse of minus infinity; lengths are cut to table_width * page_size tokens; tokens of pages
 * outside the pool (-1) take no part, nor do scores of minus infinity; a query, a visible token's scale or a score of plus
 * infinity that is no number gives NaN to the heads that it reaches. Page tables need be right only up to the sequences'
 * lengths. Extends
 * pitch_enqueue_attention_decode, which the reference does not have (README.md:96). */
typedef struct pitch_paged_attention {
  uint32_t io_type;   /* PITCH_IO_F16 or PITCH_IO_BF16 */
  uint32_t sequences; /* 1..2048 */
  uint32_t q_per_kv;  /* 1..8 */
  uint32_t window;    /* tokens; 0: all */
  /* token = sequence, head = query head; the output may be the queries' own vectors, else the two share no element */
  pitch_paged_vectors_t queries, output;
  const void* block_tables; /* int32 [sequences][table_width] */
  uint64_t block_tables_bytes;
  uint64_t table_width; /* at least 1; (table_width * page_size / 64 + 2) * sequences * kv_heads < 2^31 */
  const void* lengths; /* int32 [sequences] */
  uint64_t lengths_bytes;
  const void* slopes; /* fp32 [q_per_kv * kv_heads], or null */
  uint64_t slopes_bytes;
  void* lse; /* fp32 [sequences][q_per_kv * kv_heads], or null */
  uint64_t lse_bytes;
  float scale;
  float softcap; /* 0: none */
  void* workspace; /* pitch_paged_attention_workspace_size bytes; not used by another call until this one has completed */
  uint64_t workspace_bytes;
} pitch_paged_attention_t;
/* Bytes of device workspace pitch_enqueue_paged_attention needs on the current device for these arguments (call needs
 * sequences and q_per_kv only). */
int pitch_paged_attention_workspace_size(const pitch_paged_cache_t* cache, const pitch_paged_attention_t* call,
                                         uint64_t* bytes);
int pitch_enqueue_paged_attention(const pitch_paged_cache_t* cache, const pitch_paged_attention_t* call, void* stream);

/* Attention over whole prompts, or chunks of them, packed one behind the other: the step between the append of a prompt's
 * tokens and the first new token's pitch_enqueue_paged_attention (no counterpart in the reference, whose next step is attention,
 * README.md:96). Sequence b has the queries row_starts[b] <= r < row_starts[b + 1] and the keys and values key_starts[b] <= r <
 * key_starts[b + 1]; its nq queries are the last of its nk tokens: query i is at position p = nk - nq + i. Query head h of
 * q_heads reads KV head h / (q_heads / kv_heads):
 *   out = softmax(z) V,  lse = log sum exp(z),  z_j = cap(scale * q . k_j) + slopes[h] * (j - p)
 * over the sequence's keys j, with causal those j <= p, with a window those j > p - window; cap(x) = softcap * tanh(x / softcap), x
 * itself with softcap 0. Keys and values may be the projection's (slices of one buffer), or rows that pitch_enqueue_paged_decode read
 * back: with its row_starts as key_starts a chunk attends to all of its cached tokens. Products run on the 16-bit matrix cores and are
 * summed in float32; the softmax's weights are rounded to the vectors' type. A query that sees no key (more queries than keys) gives
 * zeros and an lse of minus infinity; scores of minus infinity take no part; what is hidden from a query has no effect on it, also
 * where it is not finite; a visible value that is not finite gives what its sum is, a score that is NaN or plus infinity gives NaN to
 * its query. (Sums of weighted values are held in float32 before they are divided by the weights': bfloat16 values beyond 2^89
 * may overflow there.) Rows of no sequence are left as they were. row_starts and key_starts do not decrease; they lie in device
 * memory, are cut to the buffers' rows and taken on trust no further. Kernels only: captured into graphs like the others. */
typedef struct pitch_prompt_attention {
  uint32_t io_type;   /* PITCH_IO_F16 or PITCH_IO_BF16 */
  uint32_t dim;       /* 64 or 128 */
  uint32_t sequences; /* at least 1; (rows * q_heads / 128 / kv_heads + sequences) * kv_heads < 2^24 */
  uint32_t q_heads, kv_heads; /* q_heads a multiple of kv_heads, both at least 1 */
  uint32_t causal;    /* 0 or 1 */
  uint32_t window;    /* tokens, below 2^31; 0: all. Needs causal, as slopes do */
  uint32_t reserved;  /* 0 */
  uint64_t rows;      /* tokens of queries and output, at least 1; rows * q_heads < 2^31 */
  uint64_t key_rows;  /* tokens of keys and values: 1..2^31 - 1025 */
  /* data and strides are multiples of 16 bytes; the token strides of keys and values are at most 2^22 elements. The output may be
   * the queries' own vectors, and else shares no element with what the call reads */
  pitch_paged_vectors_t queries, keys, values, output;
  const void* row_starts; /* int32 [sequences + 1] */
  uint64_t row_starts_bytes;
  const void* key_starts; /* int32 [sequences + 1] */
  uint64_t key_starts_bytes;
  const void* slopes; /* fp32 [q_heads], or null */
  uint64_t slopes_bytes;
  void* lse; /* fp32 [rows][q_heads], or null */
  uint64_t lse_bytes;
  float scale;
  float softcap; /* 0: none */
  void* workspace; /* pitch_prompt_attention_workspace_size bytes (null for none); not used by another call until this one has completed */
  uint64_t workspace_bytes;
} pitch_prompt_attention_t;
/* Bytes of device workspace pitch_enqueue_prompt_attention needs on the current device (0 for many tiles or few keys; else up to 136 MB
 * with vectors of 128 and 69 MB with vectors of 64 on 256 compute units) for these dim, sequences, heads, rows, key_rows and window.
 * Calls that run one after the other, a step's layers, may share one. */
int pitch_prompt_attention_workspace_size(const pitch_prompt_attention_t* call, uint64_t* bytes);
int pitch_enqueue_prompt_attention(const pitch_prompt_attention_t* call, void* stream);

/* ------------------------------------------------------------------------------------------------------------------
 * Page tables in device memory: handing out a pool's pages, giving them back, sharing them between sequences and compacting them, for
 * a program whose steps are captured into graphs (no counterpart in the reference, whose caches are one sequence's buffers,
 * README.md:65-76). Sequence b holds the pages block_tables[b][0 .. ceil(lengths[b] / page_size) - 1]; references[p] counts the
 * rows' entries that hold page p (a program may add its own, for a prefix that it keeps), and a page whose count is not positive is
 * free. The tables serve all layers: their caches have pools of as many pages of the same size. Lengths are cut to
 * 0 .. table_width * page_size; entries outside the pool are no pages; entries behind a row's length are left as they are. Where free
 * pages are handed out, the lowest number goes first, in the order of the sequences and their tokens; where they run out, a row ends
 * with its last token that has a page, and *missing is the number of pages that were lacking (0 where none were).
 * Calls that share tables, pools or a workspace run one after the other: the caller orders those on different streams. */
typedef struct pitch_paged_tables {
  void* block_tables; /* int32 [sequences][table_width] */
  uint64_t block_tables_bytes;
  uint64_t table_width; /* at least 1; table_width * page_size < 2^31 */
  void* lengths; /* int32 [sequences] */
  uint64_t lengths_bytes;
  void* references; /* int32 [pages] */
  uint64_t references_bytes;
  void* missing; /* int32 [1], or null; written by reserve and fork */
  uint64_t missing_bytes;
  uint64_t pages;     /* pages * page_size < 2^32 */
  uint32_t page_size; /* a multiple of 16, at most 65536 */
  uint32_t sequences; /* 1..2048 */
  void* workspace;    /* pitch_paged_tables_workspace_size bytes */
  uint64_t workspace_bytes;
} pitch_paged_tables_t;
/* Bytes of device workspace that the calls on these tables need (sequences, table_width, pages and page_size are looked at). */
int pitch_paged_tables_workspace_size(const pitch_paged_tables_t* tables, uint64_t* bytes);

/* Takes new_tokens[b] (int32; 0 or less: none) further tokens into every sequence b: pages are handed out where the held ones do not
 * suffice, and lengths grow. The call's tokens are packed in the order of the sequences, as a batch of prompts or a decode step has
 * them: token t's slot (page * page_size + slot, for pitch_enqueue_paged_append) goes to slots[t] and its position in its sequence to
 * positions[t] (or null). A token without a page or a place in its row has -1 in both, one whose entry of the table is no page has
 * slot -1; the entries behind the last token have -1 in both. Tokens beyond `capacity` are not taken. */
typedef struct pitch_paged_reserve {
  const void* new_tokens; /* int32 [sequences] */
  uint64_t new_tokens_bytes;
  uint64_t capacity; /* entries of slots and positions: 1..2^31 - 1 */
  void* slots; /* int64 [capacity] */
  uint64_t slots_bytes;
  void* positions; /* int64 [capacity], or null */
  uint64_t positions_bytes;
} pitch_paged_reserve_t;
int pitch_enqueue_paged_reserve(const pitch_paged_tables_t* tables, const pitch_paged_reserve_t* call, void* stream);

/* Cuts every sequence b to at most keep[b] tokens (int32; 0 or less: the whole sequence is given back): the pages behind lose a
 * reference. The tokens that remain are untouched: drafted tokens that were rejected, sequences that have ended. A row that is cut below
 * the length that it had in the last fork, as parent or as child, may end within a page that another row holds as well; it shares that
 * page from then on partly filled, and reserve, which does not look at who else holds a page, would have its next tokens written over the other's. Such
 * a row is first forked into an empty one, which gets that page as a copy, and given back behind that. A program that cannot know
 * which rows these are (a captured step) keeps n empty rows behind its n, and forks with the parents 0 .. n - 1, 0 .. n - 1, then n .. 2 n - 1
 * and n times -1: every row's partly filled last page is then its own, for a free page and a copy a row. (*missing above 0 behind the
 * first of these forks: rows have lost their last tokens.) */
int pitch_enqueue_paged_trim(const pitch_paged_tables_t* tables, const void* keep, uint64_t keep_bytes, void* stream);

/* Makes every row b a copy of row parents[b] (int32) as it was before the call: b itself leaves the row alone, a number outside the
 * rows empties it. Whole pages are shared and counted. A last page that is partly filled goes to one row (the parent's own if that
 * stays, else its first child); the others get a page of their own, into which its tokens are copied in all n_caches caches. Pages that lose their last
 * reference are handed out again in the same call. */
int pitch_enqueue_paged_fork(const pitch_paged_tables_t* tables, const pitch_paged_cache_t* caches, uint32_t n_caches,
                             const void* parents, uint64_t parents_bytes, void* stream);

/* Moves the pages in use to the lowest numbers: with U pages in use, those at U and above go into the free ones below U, the k-th to the
 * k-th, in all n_caches caches; tables and references follow. mapping (int32 [pages], or null) receives each page's new number, -1
 * for a free page; used (int32 [1], or null) receives U. The moved pages' old places keep their contents. */
int pitch_enqueue_paged_compact(const pitch_paged_tables_t* tables, const pitch_paged_cache_t* caches, uint32_t n_caches,
                                void* mapping, uint64_t mapping_bytes, void* used, uint64_t used_bytes, void* stream);

/* Packs count rows of dim unpacked codes (one uint8 per code, each < 2^bits) into count * code_stride
 * bytes, code i at bits [i * bits, i * bits + bits) of the row's little-endian 32-bit words.
 * Replaces pack_codes (reference/pitch_reference.py:68-78). */
int pitch_enqueue_pack_codes(uint32_t dim, uint32_t bits, const void* unpacked, uint64_t unpacked_bytes,
                             uint64_t unpacked_offset, void* packed, uint64_t packed_bytes,
                             uint64_t packed_offset, uint64_t count, void* stream);

/* Inverse of pitch_enqueue_pack_codes. Replaces unpack_codes (reference/pitch_reference.py:80-90). */
int pitch_enqueue_unpack_codes(uint32_t dim, uint32_t bits, const void* packed, uint64_t packed_bytes,
                               uint64_t packed_offset, void* unpacked, uint64_t unpacked_bytes,
                               uint64_t unpacked_offset, uint64_t count, void* stream);

/* Self-test of a hardware property the per-channel encoder relies on; no counterpart in the reference. The
 * encoder forms the correctly rounded reciprocal of each channel's step as v_rcp_f32 plus one Newton step,
 * which on gfx950 equals the correctly rounded 1 / x for every positive normal float below 2^126. This call
 * checks all of them on the current device (synchronously, allocating 4 MB of device memory) and writes
 * the number that differ (0 expected) to *mismatches. For tests and bring-up on new hardware. */
int pitch_selftest_reciprocal(uint64_t* mismatches);

/* Self-test of the work split of attention over codes of 2-4 bits, without a device; no counterpart in the
 * reference. For a call of kv_heads heads x tokens with one query head per KV head on a device of compute_units, writes
 * the tokens per workgroup, the workgroups per KV head (each leaves 2 + dim floats of partial results in the workspace
 * when there are several), the waves per workgroup and the floats of the workspace that
 * pitch_attention_workspace_size asks for (workspace_chunk 0; otherwise of one sized with chunks of that many tokens). */
int pitch_selftest_attention_split(uint32_t dim, uint64_t tokens, uint32_t kv_heads, uint32_t key_bias,
                                   uint32_t head_major, uint32_t compute_units, uint32_t workspace_chunk, uint64_t split[4]);

/* Self-test of the choice of kernels for attention over per-vector caches without the key-bias term, without a device; no
 * counterpart in the reference. Writes 1 if a call of kv_heads heads x tokens with q_per_kv query heads per KV head on a
 * device of compute_units runs the kernels for codes of 2-4 bits, 0 if it runs the others. head_major is 1 for caches in
 * which the rows of a KV head's tokens follow each other. */
int pitch_selftest_attention_route(uint32_t dim, uint64_t tokens, uint32_t kv_heads, uint32_t q_per_kv, uint32_t key_bits,
                                   uint32_t value_bits, uint32_t head_major, uint32_t compute_units, uint32_t* codes);

#ifdef __cplusplus
}
#endif

#endif /* PITCH_AMD_H */
