"""Paged attention at shapes drawn at random, at the longest tables, over pages far apart, and several paged calls at once."""
import math
import threading

import numpy as np
import pytest

import paged_reference as R
from test_gpu_paged_values import _attend, _pool, _typed

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(40))
def test_random_shapes(q, seed):
    """Any widths, methods, heads, pages, layouts, lengths (none, one, edges of tiles), windows, caps and slopes."""
    rng = np.random.default_rng(1000 + seed)
    pick = lambda *x: x[int(rng.integers(len(x)))]  # noqa: E731
    d, kv, nq, page, dtype = pick(64, 128), pick(1, 1, 2, 3, 5), int(rng.integers(1, 9)), pick(16, 32, 48, 64, 80, 128), pick("float16", "bfloat16")
    keys, values = [(pick("turboQuant", "turboQuant", "polarQuant"), int(rng.integers(2, 9))) for _ in range(2)]
    B = pick(1, 2, 5, 30, 70, 150)
    most = pick(70, 600, 600, 2500) if B < 70 else pick(70, 300)
    edges = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, most]
    lengths = [int(pick(*edges)) if rng.random() < 0.4 else int(rng.integers(0, most + 1)) for _ in range(B)]
    lengths = [min(n, most) for n in lengths]
    window, softcap, sloped = pick(0, 0, 1, 16, 33, 200), pick(0.0, 0.0, 20.0, 1e5), bool(rng.random() < 0.3)
    print(d, kv, nq, page, dtype, keys, values, B, most, window, softcap, sloped, flush=True)
    tables, pages = R.tables_of(rng, lengths, page)
    pool = _pool(rng, d, kv, keys, values, page, pages)
    slopes = (0.05 * 2.0 ** -rng.random(kv * nq)).astype(np.float32) if sloped else None
    scale = float(np.float32(0.9 / math.sqrt(d)))
    Q = _typed(R.queries_of(rng, pool, tables, lengths, kv * nq, scale, window, softcap=softcap, slopes=slopes), dtype)
    ref = R.reference(pool, tables, lengths, Q, dtype, scale, softcap, window, None if slopes is None else slopes.astype(np.float64))
    out, lse = _attend(q, pool, pick("head", "token"), tables, lengths, Q, dtype, scale=scale, softcap=softcap, window=window, slopes=slopes)
    bad = R.wrong(out, lse, ref)
    assert not len(bad), (bad[:5], [(np.linalg.norm(out[b, h] - ref["out"][b, h]), ref["bar"][b, h], lse[b, h] - ref["lse"][b, h],
                                     ref["lse_bar"][b, h]) for b, h in bad[:5]])


@pytest.mark.parametrize("sloped", [False, True])
def test_the_longest_table(q, sloped):
    """A table of nearly 2^31 tokens, all pages but the last outside the pool: what lies in the last page is attended over."""
    rng = np.random.default_rng(3)
    d, page, width = 64, 65536, 32767
    pool = _pool(rng, d, 1, ("turboQuant", 4), ("turboQuant", 3), page, 1)
    length = width * page - 65000
    tables = np.full((1, width), -1, np.int32)
    tables[0, -1] = 0
    slopes = np.array([0.03, 0.01], np.float32) if sloped else None
    Q = _typed(rng.normal(size=(1, 2, d)) * 0.7, "float16")
    scale = float(np.float32(0.1))

    short = R.reference(pool, np.zeros((1, 1), np.int32), [length - (width - 1) * page], Q, "float16", scale, slopes=None if slopes is None else slopes.astype(np.float64))
    out, lse = _attend(q, pool, "head", tables, [length], Q, "float16", scale=scale, slopes=slopes)
    assert not len(R.wrong(out, lse, short))


def test_pages_far_apart(q):
    """Pages 2^24 vectors apart, more than 2^32 bytes from the first to the last: the same as a small pool."""
    import torch
    import pitch_amd as P
    dev, d, kv, page, pages, far = q.device, 64, 2, 32, 18, 1 << 24
    cfg = q.config("turboQuant", d, 2)
    made = []
    for _ in range(2):
        codes = torch.empty(((pages - 1) * far + kv * page) * cfg.codeStride, dtype=torch.uint8, device=dev)
        scales = torch.empty((pages - 1) * far + kv * page, dtype=torch.float32, device=dev)
        made += [codes.as_strided((pages, kv, page, cfg.codeStride), (far * cfg.codeStride, page * cfg.codeStride, cfg.codeStride, 1)),
                 scales.as_strided((pages, kv, page), (far, page, 1))]
    assert far * cfg.codeStride * (pages - 1) > 2 ** 32
    caches = [P.PagedCache(q, cfg, cfg, pages=pages, pageSize=page, kvHeads=kv),
              P.PagedCache(q, cfg, cfg, pages=pages, pageSize=page, kvHeads=kv, keyCodes=made[0], keyScales=made[1], valueCodes=made[2],
                           valueScales=made[3])]
    n = pages * page
    x = torch.randn(2, n, kv, d, device=dev).to(torch.float16)
    queries = torch.randn(1, 3 * kv, d, device=dev).to(torch.float16)
    table = torch.randperm(pages, device=dev).to(torch.int32)[None]
    got = []
    for c in caches:
        c.enqueueAppend(x[0], x[1], torch.arange(n, device=dev))
        back = [torch.zeros(n, kv, d, device=dev, dtype=torch.float16) for _ in range(2)]
        c.enqueueDecode(table, torch.tensor([0, n], dtype=torch.int32, device=dev), keysOut=back[0], valuesOut=back[1])
        out = torch.zeros_like(queries)
        c.enqueueAttention(queries, table, torch.tensor([n], dtype=torch.int32, device=dev), out)
        got.append(back + [out, c.keyCodes, c.keyScales, c.valueCodes, c.valueScales])
    torch.cuda.synchronize()
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert got[0][2].abs().sum() > 0


def test_calls_of_several_threads(q):
    """Attention of different kernels, appends and read-backs from threads with streams and workspaces of their own: each
    writes what it writes alone."""
    import torch
    import pitch_amd as P
    dev = q.device

    def side(d, kv, nq, bits, dtype, lengths):
        torch.manual_seed(d + nq)
        cfg, page = q.config("turboQuant", d, bits), 16
        width = -(-max(lengths) // page)
        cache = P.PagedCache(q, cfg, cfg, pages=width, pageSize=page, kvHeads=kv)
        x = torch.randn(width * page, kv, d, device=dev).to(dtype)
        queries = torch.randn(len(lengths), kv * nq, d, device=dev).to(dtype)
        table = torch.arange(width, dtype=torch.int32, device=dev)[None].repeat(len(lengths), 1).contiguous()
        L = torch.tensor(lengths, dtype=torch.int32, device=dev)
        slots, starts = torch.arange(width * page, device=dev), torch.tensor([0, width * page], dtype=torch.int32, device=dev)
        ws = torch.empty(cache.attentionWorkspaceBytes(len(lengths), nq), dtype=torch.uint8, device=dev)
        out, back = torch.zeros_like(queries), torch.zeros_like(x)
        calls = [P.PagedAppend(cache, x, x, slots), P.PagedAttention(cache, queries, table, L, out, workspace=ws),
                 P.PagedDecode(cache, table[:1].contiguous(), starts, keysOut=back)]
        for c in calls:
            c.enqueue()
        torch.cuda.synchronize()
        return calls, out, back, out.clone(), back.clone()

    sides = [side(128, 2, 4, 4, torch.bfloat16, [900, 30]), side(64, 1, 8, 8, torch.float16, [2000]),
             side(64, 3, 1, 3, torch.bfloat16, [100] * 90), side(128, 1, 6, 2, torch.float16, [400, 1])]
    failed = []

    def work(calls, out, back, out_ref, back_ref):
        try:
            stream = torch.cuda.Stream()
            for _ in range(100):
                with torch.cuda.stream(stream):
                    out.zero_()
                    back.zero_()
                for c in calls:
                    c.enqueue(stream)
                stream.synchronize()
                assert torch.equal(out, out_ref) and torch.equal(back, back_ref)
        except Exception as e:  # noqa: BLE001 (reported by the main thread)
            failed.append(repr(e))

    threads = [threading.Thread(target=work, args=s) for s in sides]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
