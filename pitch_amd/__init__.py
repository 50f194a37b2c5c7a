"""pitch_amd: the MI355X (gfx950) KV-cache codec of SwiftCham/PITCH, as hand-written HIP kernels behind a C ABI.

The operator surface mirrors the reference: ``PITCH`` (config / encode / decode / enqueueEncode /
enqueueDecode and the per-channel forms), ``QuantConfig``, ``ChannelQuantConfig``, ``CompressedBatch``,
``ChannelCompressedBlock``, the ``PITCHError`` family, and function-level mirrors of
reference/pitch_reference.py (``turbo_encode``, ``polar_decode``, ``channel_encode``, ``pack_codes``, ...)
that run on device tensors. ``PITCH.enqueueEncodeBatch`` / ``EncodeBatch`` encode many caches' segments (a
token's append to every layer) in one call, and ``PITCH.enqueueDecodeBatch`` / ``DecodeBatch`` decode them. ``attention_decode`` / ``PITCH.enqueueAttentionDecode`` compute decode-step
attention directly over the compressed caches. ``PagedCache`` keeps many sequences' keys and values as codes in the pages of
one pool, written by ``PagedAppend``, read back by ``PagedDecode`` and attended over by ``PagedAttention``; ``PagedTables`` hands the
pages out and takes them back on the device (``PagedReserve``, ``PagedTrim``, ``PagedFork``, ``PagedCompact``). ``PromptAttention`` /
``PITCH.enqueuePromptAttention`` compute attention over whole prompts, or chunks of them behind a cached prefix.
"""
from .api import (  # noqa: F401
    CHANNEL_DEFAULT_GROUP, DECODERS, DEFAULT_SEED, ENCODERS, FP16_MAX, PITCH, SUPPORTED_BITS, SUPPORTED_DIMS,
    ChannelCompressedBlock, ChannelQuantConfig, CompressedBatch, ConfigurationMismatch, DecodeBatch, DecodingFailed,
    DeviceUnavailable, EncodeBatch, EncodingFailed, InvalidBitWidth, InvalidDimension, InvalidInput, KeyBias, PITCHError,
    QuantConfig, QuantMethod, attention_decode, attention_decode_channel_keys, attention_workspace_bytes, bits_per_coordinate, channel_bits_per_coordinate, channel_decode, channel_encode,
    channel_group_count, code_stride_bytes, half_to_float, pack_codes, polar_decode, polar_encode, rand_signs,
    turbo_decode, turbo_encode, unpack_codes,
)
from .paged import PagedAppend, PagedAttention, PagedCache, PagedDecode  # noqa: F401
from .pages import PagedCompact, PagedFork, PagedReserve, PagedTables, PagedTrim  # noqa: F401
from .prompt import PromptAttention  # noqa: F401

__version__ = "0.1.0"
