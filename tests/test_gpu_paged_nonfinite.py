"""Vectors that are not finite, appended to a paged cache: their scales are not finite, and no other vector notices."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

WHERE = [[(3, "nan")], [(3, "inf")], [(70, "-inf")], [(3, "inf"), (4, "-inf")], [(0, "inf"), (63, "inf")], [(5, "nan"), (6, "inf")]]


@pytest.mark.parametrize("normed", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "float16", "bfloat16"])
@pytest.mark.parametrize("method,bits", [("turboQuant", 4), ("polarQuant", 4), ("polarQuant", 2), ("turboQuant", 8)])
def test_append_of_what_is_not_finite(q, method, bits, dtype, normed):
    import torch
    import pitch_amd as P
    dev, d, kv, page = q.device, 128, 5, 16     # (long calls: four heads a team)
    dt, cfg = getattr(torch, dtype), q.config(method, d, bits)
    for n in (12, 9000):
        g = torch.Generator(device=dev).manual_seed(n)
        x = torch.randn(n, kv, d, device=dev, generator=g).to(dt)
        pages = -(-n // page)
        more = dict(keyNorm=torch.ones(d, device=dev, dtype=dt)) if normed else {}
        good, bad = (P.PagedCache(q, cfg, cfg, pages=pages, pageSize=page, kvHeads=kv) for _ in range(2))
        good.enqueueAppend(x, x, torch.arange(n, device=dev), **more)
        y, hit = x.clone(), np.zeros((n, kv), bool)
        for i, what in enumerate(WHERE):
            for at, value in what:
                y[2 * i, i % kv, at] = float(value)
            hit[2 * i, i % kv] = True
        bad.enqueueAppend(y, y, torch.arange(n, device=dev), **more)
        torch.cuda.synchronize()
        for name in ("key", "value"):
            s, s0 = (getattr(c, name + "Scales").transpose(1, 2).reshape(-1, kv)[:n].cpu().numpy() for c in (bad, good))
            c, c0 = (getattr(c, name + "Codes").transpose(1, 2).reshape(pages * page, kv, -1)[:n].cpu().numpy() for c in (bad, good))
            assert not np.isfinite(s[hit]).any(), (name, s[hit])
            assert np.array_equal(s[~hit], s0[~hit]) and np.array_equal(c[~hit], c0[~hit])


def test_attention_over_it(q):
    """The sequence that holds such a vector gives NaN, others what they give without it."""
    import torch
    import pitch_amd as P
    dev, d, page = q.device, 64, 16
    for method in ("turboQuant", "polarQuant"):
        cfg = q.config(method, d, 3)
        cache = P.PagedCache(q, cfg, cfg, pages=8, pageSize=page)
        x = torch.randn(8 * page, 1, d, device=dev).to(torch.float16)
        x[5, 0, 9] = float("nan")
        cache.enqueueAppend(x, x, torch.arange(8 * page, device=dev))
        queries = torch.randn(2, 2, d, device=dev).to(torch.float16)
        out = torch.zeros_like(queries)
        table = torch.arange(8, dtype=torch.int32, device=dev).view(2, 4)
        cache.enqueueAttention(queries, table, torch.tensor([60, 60], dtype=torch.int32, device=dev), out)
        torch.cuda.synchronize()
        assert out[0].isnan().all() and out[1].isfinite().all() and out[1].abs().sum() > 0, method
