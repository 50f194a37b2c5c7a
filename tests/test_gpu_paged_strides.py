"""Paged caches whose pages lie apart, and attention's outputs of any stride: the same bits as contiguous buffers, and nothing
written beside them."""
import pytest

pytestmark = pytest.mark.gpu

LAYERS, LAYER = 3, 1


def _pools(q, kcfg, vcfg, pages, page, kv, layout):
    """(a contiguous cache, one that is a layer's part of buffers [page][layer][...], those buffers)."""
    import torch
    import pitch_amd as P
    kw = dict(pages=pages, pageSize=page, kvHeads=kv, layout=layout)
    whole = P.PagedCache(q, kcfg, vcfg, **kw)
    names = ("keyCodes", "keyScales", "valueCodes", "valueScales")
    wide = {n: torch.full((pages, LAYERS) + tuple(getattr(whole, n).shape[1:]), 0x5A, dtype=getattr(whole, n).dtype, device=q.device) for n in names}
    for n in names:
        getattr(whole, n).fill_(0x5A)
    return whole, P.PagedCache(q, kcfg, vcfg, **kw, **{n: t[:, LAYER] for n, t in wide.items()}), wide


@pytest.mark.parametrize("d,kv,nq,page,layout,methods,dtype", [
    (128, 2, 4, 16, "head", ("turboQuant", 4, "turboQuant", 3), "bfloat16"),
    (64, 3, 2, 48, "token", ("polarQuant", 3, "turboQuant", 2), "float16"),
    (128, 1, 8, 64, "token", ("turboQuant", 5, "polarQuant", 6), "float16"),
    (64, 4, 1, 32, "head", ("turboQuant", 8, "turboQuant", 4), "bfloat16"),
])
def test_pages_that_lie_apart(q, d, kv, nq, page, layout, methods, dtype):
    import torch
    dev, dt, pages, n = q.device, getattr(torch, dtype), 40, 700
    kcfg, vcfg = q.config(methods[0], d, methods[1]), q.config(methods[2], d, methods[3])
    whole, part, wide = _pools(q, kcfg, vcfg, pages, page, kv, layout)
    g = torch.Generator(device=dev).manual_seed(d + kv)
    n = min(n, pages * page - 5)
    x = torch.randn(n, 2 * kv, d, device=dev, generator=g).to(dt)
    order = torch.randperm(pages, device=dev, generator=g)
    used = -(-n // page)
    slots = order[torch.arange(n, device=dev) // page] * page + torch.arange(n, device=dev) % page
    tables = order[:used][None].to(torch.int32).repeat(3, 1).contiguous()
    lengths = torch.tensor([n, 65, 0], dtype=torch.int32, device=dev)
    queries = torch.randn(3, kv * nq, d, device=dev, generator=g).to(dt)
    results = []
    for cache in (whole, part):
        cache.enqueueAppend(x[:, :kv], x[:, kv:], slots)
        back = [torch.full((n + 1, kv, d), -5.0, dtype=dt, device=dev) for _ in range(2)]
        cache.enqueueDecode(tables[:1], torch.tensor([0, n], dtype=torch.int32, device=dev), keysOut=back[0], valuesOut=back[1])
        out, lse = torch.zeros_like(queries), torch.zeros(3, kv * nq, device=dev)
        cache.enqueueAttention(queries, tables, lengths, out, lse=lse)
        results.append(back + [out, lse])
    torch.cuda.synchronize()
    for a, b in zip(*results):
        assert torch.equal(a, b) and a.abs().sum() > 0
    for name, t in wide.items():
        assert torch.equal(t[:, LAYER], getattr(whole, name)), name
        for other in set(range(LAYERS)) - {LAYER}:
            assert (t[:, other] == 0x5A).all(), name


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("d,kv,nq,lengths", [(128, 2, 3, [300, 0, 20]), (64, 1, 8, [9000, 70, 0]), (64, 4, 1, [130] * 90)])
def test_outputs_of_any_stride(q, d, kv, nq, lengths, dtype):
    """A slice of a wider buffer, [head][sequence] order, the queries' own buffer."""
    import torch
    dev, dt, page, B, H = q.device, getattr(torch, dtype), 16, len(lengths), kv * nq
    cfg = q.config("turboQuant", d, 4)
    import pitch_amd as P
    width = -(-max(lengths) // page)
    cache = P.PagedCache(q, cfg, cfg, pages=width, pageSize=page, kvHeads=kv)
    g = torch.Generator(device=dev).manual_seed(d)
    x = torch.randn(width * page, kv, d, device=dev, generator=g).to(dt)
    cache.enqueueAppend(x, x.flip(0).contiguous(), torch.arange(width * page, device=dev))
    tables = torch.arange(width, dtype=torch.int32, device=dev)[None].repeat(B, 1).contiguous()
    L = torch.tensor(lengths, dtype=torch.int32, device=dev)
    queries = torch.randn(B, H, d, device=dev, generator=g).to(dt)
    ref = torch.zeros_like(queries)
    cache.enqueueAttention(queries, tables, L, ref)
    wide = torch.full((B, H + 3, d + 6), -9.0, dtype=dt, device=dev)
    cache.enqueueAttention(queries, tables, L, wide[:, 2:H + 2, 4:d + 4])
    turned = torch.full((H, B + 1, d), -9.0, dtype=dt, device=dev)
    cache.enqueueAttention(queries, tables, L, turned[:, :B].transpose(0, 1))
    same = queries.clone()
    cache.enqueueAttention(same, tables, L, same)
    torch.cuda.synchronize()
    assert ref.abs().sum() > 0 and torch.equal(wide[:, 2:H + 2, 4:d + 4], ref) and torch.equal(turned[:, :B].transpose(0, 1), ref)
    assert torch.equal(same, ref)
    wide[:, 2:H + 2, 4:d + 4] = -9.0
    assert (wide == -9.0).all() and (turned[:, B] == -9.0).all()
