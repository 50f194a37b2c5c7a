"""What the compiler gave the kernels of prompt attention and of the page tables, read from the built library: none spills or has
scratch memory, and the attention's registers let as many workgroups run on a compute unit as its shared memory does."""
import pytest

from pitch_amd import _lib
from test_kernel_resources import _code_objects, _kernels


def _found(name):
    pytest.importorskip("msgpack")
    if not _lib.LIB_PATH.exists():
        pytest.skip("HIP library not built")
    return [k for elf in _code_objects(_lib.LIB_PATH.read_bytes()) for k in _kernels(elf) if name in k[".name"]]


@pytest.mark.parametrize("name,count", [
    ("prompt_attention", 2 * 2 * 2 * 2),   # dimensions, types, plain scores or not, keys cut or not
    ("prompt_cut", 4), ("prompt_join", 4), ("pages_", 13)])
def test_kernels_spill_nothing(name, count):
    found = _found(name)
    assert len(found) == count
    for k in found:
        assert [k[".private_segment_fixed_size"], k[".vgpr_spill_count"], k[".sgpr_spill_count"]] == [0, 0, 0], k[".name"]


def test_registers_of_prompt_attention():
    registers = sorted(k[".vgpr_count"] for k in _found("prompt_attention"))
    assert registers[7] <= 168 and registers[-1] <= 256     # heads of 64: three waves a SIMD; of 128: two
