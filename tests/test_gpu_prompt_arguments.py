"""Arguments of PromptAttention and of the page tables' classes that do not fit: InvalidInput, before anything is launched."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def _prompt(q, torch):
    dev = q.device
    x = torch.zeros(20, 4, 64, device=dev, dtype=torch.bfloat16)
    k = torch.zeros(30, 2, 64, device=dev, dtype=torch.bfloat16)
    return x, k, torch.tensor([0, 20], dtype=torch.int32, device=dev), torch.zeros_like(x)


def test_prompt_arguments_that_are_no_tensors(q):
    import torch
    import pitch_amd as P
    x, k, starts, out = _prompt(q, torch)
    for t in ([0.0] * 4, np.zeros((20, 4, 64), np.float32), 3, "x"):
        for args in ((t, k, k, starts, out), (x, t, k, starts, out), (x, k, t, starts, out), (x, k, k, t, out), (x, k, k, starts, t)):
            with pytest.raises(P.InvalidInput):
                q.enqueuePromptAttention(*args)
        for more in (dict(keyStarts=t), dict(slopes=t), dict(lse=t)):
            with pytest.raises(P.InvalidInput):
                q.enqueuePromptAttention(x, k, k, starts, out, **more)


def test_prompt_arguments_that_do_not_fit(q):
    import torch
    import pitch_amd as P
    x, k, starts, out = _prompt(q, torch)
    f32, i64 = x.float(), starts.long()
    cases = [((f32, k, k, starts, out), {}), ((x, k.half(), k, starts, out), {}), ((x, k, k.half(), starts, out), {}), ((x, k, k, i64, out), {}),
             ((x, k, k, starts, out.half()), {}), ((x[:, :3], k, k, starts, out[:, :3]), {}), ((x, k, k[:29], starts, out), {}),
             ((x, k, k, starts, out[:19]), {}), ((x, k, k, starts[:1], out), {}), ((x[..., :32], k[..., :32], k[..., :32], starts, out[..., :32]), {}),
             ((x.transpose(1, 2), k, k, starts, out), {}), ((x[:0], k, k, starts, out[:0]), {}), ((x, k[:0], k[:0], starts, out), {}),
             ((x, k, k, starts, out), dict(window=-1)), ((x, k, k, starts, out), dict(window=1.5)), ((x, k, k, starts, out), dict(window=2 ** 31)),
             ((x, k, k, starts, out), dict(window=2 ** 40)), ((x, k, k, starts, out), dict(causal=1)), ((x, k, k, starts, out), dict(causal=False, window=4)),
             ((x, k, k, starts, out), dict(softcap=-1.0)), ((x, k, k, starts, out), dict(softcap="x")), ((x, k, k, starts, out), dict(scale=float("nan"))),
             ((x, k, k, starts, out), dict(scale="x")), ((x, k, k, starts, out), dict(slopes=torch.zeros(3, device=q.device))),
             ((x, k, k, starts, out), dict(lse=torch.zeros(79, device=q.device))), ((x, k, k, starts, out), dict(keyStarts=starts[:1])),
             ((x, k, k, starts, k.new_zeros(1, 1, 1).expand(20, 4, 64)), {}), ((x, x[:, :2], x[:, 2:], starts, x), {})]
    for args, more in cases:
        with pytest.raises((P.InvalidInput, P.InvalidDimension)):
            q.enqueuePromptAttention(*args, **more)
    wide = torch.zeros(20, 4, 68, device=q.device, dtype=torch.bfloat16)[..., :64]
    with pytest.raises(P.InvalidInput, match="16 bytes"):
        q.enqueuePromptAttention(wide, k, k, starts, out)
    few = (x[:1], torch.zeros(4000, 2, 64, device=q.device, dtype=torch.bfloat16))
    with pytest.raises(P.InvalidInput, match="workspace"):
        q.enqueuePromptAttention(few[0], few[1], few[1].clone(), starts, out[:1], workspace=torch.zeros(64, dtype=torch.uint8, device=q.device))


def test_tables_arguments(q):
    import torch
    import pitch_amd as P
    dev = q.device
    cfg = q.config("turboQuant", 64, 4)
    cache = P.PagedCache(q, cfg, cfg, pages=6, pageSize=16)
    i32 = lambda *n: torch.zeros(*n, dtype=torch.int32, device=dev)  # noqa: E731
    tables = P.PagedTables(cache, sequences=3, width=2)
    assert tables.blockTables.tolist() == [[-1, -1]] * 3 and tables.lengths.tolist() == [0] * 3 and tables.references.tolist() == [0] * 6
    other = P.PagedCache(q, cfg, cfg, pages=7, pageSize=16)
    for make in (lambda: P.PagedTables(5, sequences=1, width=1), lambda: P.PagedTables([], sequences=1, width=1), lambda: P.PagedTables([cache, 3], sequences=1, width=1),
                 lambda: P.PagedTables([cache, other], sequences=1, width=1), lambda: P.PagedTables(cache), lambda: P.PagedTables(cache, sequences=1),
                 lambda: P.PagedTables(cache, sequences=0, width=1), lambda: P.PagedTables(cache, sequences=2049, width=1),
                 lambda: P.PagedTables(cache, sequences=1, width=2 ** 30), lambda: P.PagedTables(cache, sequences=1, width=1, blockTables=i32(1, 1)),
                 lambda: P.PagedTables(cache, blockTables=i32(3)), lambda: P.PagedTables(cache, blockTables=i32(3, 2).long()),
                 lambda: P.PagedTables(cache, blockTables=i32(3, 2), lengths=i32(2)), lambda: P.PagedTables(cache, blockTables=i32(3, 2), references=i32(5)),
                 lambda: P.PagedTables(cache, blockTables=i32(3, 2), missing=i32(2)), lambda: P.PagedTables(cache, blockTables=i32(4, 3)[:, :2])):
        with pytest.raises(P.InvalidInput):
            make()
    slots = torch.zeros(4, dtype=torch.int64, device=dev)
    for t in ([0, 0, 0], np.zeros(3, np.int32), 3, "x", i32(2), i32(3).long()):
        for call in (lambda: tables.enqueueReserve(t, slots), lambda: tables.enqueueTrim(t), lambda: tables.enqueueFork(t),
                     lambda: tables.enqueueCompact(mapping=t), lambda: tables.enqueueCompact(used=t)):
            with pytest.raises(P.InvalidInput):
                call()
    for call in (lambda: tables.enqueueReserve(None, slots), lambda: tables.enqueueTrim(None), lambda: tables.enqueueFork(None),
                 lambda: tables.enqueueReserve(i32(3), None), lambda: tables.enqueueReserve(i32(3), i32(4)), lambda: tables.enqueueReserve(i32(3), slots[:0]),
                 lambda: tables.enqueueReserve(i32(3), slots, positions=slots[:3]), lambda: tables.enqueueReserve(i32(3), slots, positions=slots),
                 lambda: P.PagedTrim(cache, i32(3)), lambda: tables.enqueueTrim(tables.lengths), lambda: tables.enqueueFork(tables.lengths),
                 lambda: tables.enqueueReserve(tables.lengths, slots), lambda: tables.enqueueCompact(mapping=tables.references)):
        with pytest.raises(P.InvalidInput):
            call()
    # tables in a pool of theirs, or over each other
    inside = cache.keyScales.view(torch.int32).flatten()
    with pytest.raises(P.InvalidInput, match="overlap"):
        P.PagedTables(cache, blockTables=inside[:6].view(3, 2)).enqueueCompact()
    both = i32(8)
    with pytest.raises(P.InvalidInput, match="overlap"):
        P.PagedTables(cache, blockTables=both[:6].view(3, 2), lengths=both[5:8]).enqueueTrim(i32(3))
    torch.cuda.synchronize()
    assert tables.lengths.tolist() == [0] * 3
