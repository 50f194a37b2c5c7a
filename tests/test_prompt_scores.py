"""The comparison of attention results whose scores are not finite finds what it is there to find: mistakes are planted in results that
the definition gives."""
import math

import pytest
import torch

from prompt_scores import definition, spoiled, strict

LENGTHS = [(20, 20), (3, 50), (1, 9)]
MORE = [dict(), dict(softcap=10.0), dict(causal=False), dict(window=6)]


def _right(more, values, dtype=torch.bfloat16):
    q, k, v, rs, ks = spoiled(LENGTHS, 4, 2, 64, dtype, 1, values=values)
    want = definition(q, k, v, rs, ks, **more)
    return want, want["out"].to(dtype), want["lse"].float()


@pytest.mark.parametrize("more", MORE)
@pytest.mark.parametrize("values", [False, True])
def test_right_results_pass(more, values):
    want, out, lse = _right(more, values)
    assert 0 < strict(out, lse, want) < int(want["inside"].sum()) * 4
    assert bool(torch.isfinite(want["out"][want["inside"][:, None] & ~want["bad"]]).any())


@pytest.mark.parametrize("more", MORE)
@pytest.mark.parametrize("values", [False, True])
@pytest.mark.parametrize("wrong", [0.0, 5.0, math.inf])
def test_rows_that_should_be_nan_and_are_not(more, values, wrong):
    want, out, lse = _right(more, values)
    row, head = (int(x) for x in want["bad"].nonzero()[0])
    for spoil in (lambda o, s: o[row, head].fill_(wrong), lambda o, s: o[row, head, 9:10].fill_(wrong), lambda o, s: s[row, head:head + 1].fill_(wrong)):
        o, s = out.clone(), lse.clone()
        spoil(o, s)
        with pytest.raises(AssertionError, match="not NaN"):
            strict(o, s, want)


@pytest.mark.parametrize("more", MORE)
@pytest.mark.parametrize("values", [False, True])
def test_rows_that_are_wrong_beside_them(more, values):
    want, out, lse = _right(more, values)
    fine = (want["inside"][:, None] & ~want["bad"]).nonzero()
    for row, head in (tuple(int(x) for x in fine[i]) for i in (0, len(fine) // 2, -1)):
        for spoil in (lambda o, s: o[row, head, 20:21].add_(0.5), lambda o, s: o[row, head, 20:21].fill_(math.nan), lambda o, s: s[row, head:head + 1].add_(0.1)):
            o, s = out.clone(), lse.clone()
            spoil(o, s)
            with pytest.raises(AssertionError):
                strict(o, s, want)
