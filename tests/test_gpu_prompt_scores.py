"""Prompt attention whose scores are NaN or infinite, in whole query tiles and in keys that are cut into parts (one part holds them):
such a score gives NaN to its query and to no other."""
import math

import pytest
import torch

import pitch_amd as P
from prompt_scores import definition, spoiled, strict

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]
WHOLE, CUT = [(70, 70), (200, 200), (5, 130)], [(3, 3000), (5, 2500)]


def _i32(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _run(pitch, q, k, v, rs, ks, **more):
    q, k, v = (t.cuda() for t in (q, k, v))
    if more.get("slopes") is not None:
        more["slopes"] = more["slopes"].cuda()
    out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device="cuda")
    call = P.PromptAttention(pitch, q, k, v, _i32(rs), out, keyStarts=_i32(ks), lse=lse, **more)
    call.enqueue()
    torch.cuda.synchronize()
    assert bool((out[rs[-1]:] == 7).all()) and bool((lse[rs[-1]:] == 7).all())
    return out, lse, call


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lengths", [WHOLE, CUT])
@pytest.mark.parametrize("values", [False, True])
@pytest.mark.parametrize("more", [dict(), dict(softcap=10.0), dict(softcap=0.2), dict(window=40), dict(causal=False), dict(scale=-0.2)])
def test_scores_that_are_not_finite(q, dtype, dim, lengths, values, more):
    args = spoiled(lengths, 4, 2, dim, dtype, 3, values=values)
    out, lse, call = _run(q, *args, **more)
    assert (call.workspaceBytes > 0) == (lengths is CUT and not more.get("window"))
    assert strict(out, lse, definition(*args, **more)) > 0


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [WHOLE, CUT])
@pytest.mark.parametrize("softcap", [0.0, 10.0])
def test_with_slopes(q, dtype, lengths, softcap):
    args = spoiled(lengths, 6, 2, 64, dtype, 4, values=True)
    slopes = 2.0 ** -torch.arange(1, 7, dtype=torch.float32)
    out, lse, _ = _run(q, *args, slopes=slopes, softcap=softcap)
    assert strict(out, lse, definition(*args, slopes=slopes, softcap=softcap)) > 0


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("at", [0, 63, 64, 1499, 2936, 2999])
@pytest.mark.parametrize("what", ["nan", "inf"])
@pytest.mark.parametrize("softcap", [0.0, 10.0])
def test_one_key_of_a_cut_sequence(q, dim, at, what, softcap):
    """The part that holds the key, first, last or between, makes the joined rows NaN; the other KV head's rows are as without it."""
    qq, k, v = torch.ones(4, 4, dim), torch.full((3000, 2, dim), 0.01), torch.ones(3000, 2, dim)
    k[at, 0, 9] = math.nan if what == "nan" else math.inf
    args = [t.to(torch.bfloat16) for t in (qq, k, v)] + [[0, 4], [0, 3000]]
    out, lse, call = _run(q, *args, softcap=softcap)
    assert call.workspaceBytes > 0
    sees = torch.arange(2996, 3000) >= at
    for h in range(4):
        bad = sees & (h < 2) & (what == "nan" or softcap == 0)
        assert torch.equal(torch.isnan(out[:, h].cpu()).all(1), bad) and torch.equal(torch.isnan(out[:, h].cpu()).any(1), bad)
        assert torch.equal(torch.isnan(lse[:, h].cpu()), bad)
        assert bool((out[:, h].cpu()[~bad] == 1).all())
    strict(out, lse, definition(*args, softcap=softcap))


@pytest.mark.parametrize("dtype", TYPES)
def test_all_scores_of_a_row_are_nan(q, dtype):
    """Also where its values are not finite: the plain sum of nothing else would be finite or infinite there."""
    args = spoiled([(40, 40), (4, 2800)], 2, 1, 128, dtype, 5)
    args[0][:] = math.nan
    args[2][3, 0, 3], args[2][50, 0, 4] = math.inf, -math.inf
    out, lse, _ = _run(q, *args)
    assert bool(torch.isnan(out[:44]).all()) and bool(torch.isnan(lse[:44]).all())
