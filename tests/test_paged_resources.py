"""What the compiler gave the paged caches' kernels, read from the built library: none spills a vector register, and the append and
the read-back have no scratch memory. A scratch access in a tile's loop waits for all of the tile's loads."""
import pytest

from pitch_amd import _lib
from test_kernel_resources import _code_objects, _kernels


@pytest.mark.parametrize("name,count", [
    ("paged_attn", 2 * 4 * 4 * 2 * 2),   # dimensions, widths of keys and of values, four or eight heads, element types
    ("paged_append", 2 * 3 * 3),         # dimensions, element types, heads at once and PolarQuant
    ("paged_decode", 2 * 3 * 2),         # dimensions, element types, heads at once
])
def test_paged_kernels_spill_nothing(name, count):
    pytest.importorskip("msgpack")
    if not _lib.LIB_PATH.exists():
        pytest.skip("HIP library not built")
    found = [k for elf in _code_objects(_lib.LIB_PATH.read_bytes()) for k in _kernels(elf) if name in k[".name"]]
    assert len(found) == count
    for k in found:
        assert k[".vgpr_spill_count"] == 0, k[".name"]
        if name != "paged_attn":   # (whose scalar registers may want a slot)
            assert k[".private_segment_fixed_size"] == 0, k[".name"]
