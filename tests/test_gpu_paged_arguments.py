"""Arguments of the paged classes that are no tensors, or no numbers: InvalidInput, as for tensors of the wrong kind."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu


def test_arguments_that_are_no_tensors(q):
    import torch
    import pitch_amd as P
    dev, d, kv = q.device, 64, 2
    cfg = q.config("turboQuant", d, 4)
    cache = P.PagedCache(q, cfg, cfg, pages=4, pageSize=16, kvHeads=kv)
    x = torch.zeros(5, kv, d, device=dev, dtype=torch.bfloat16)
    slots, table = torch.arange(5, device=dev), torch.zeros(5, 2, dtype=torch.int32, device=dev)
    lengths, starts = torch.ones(5, dtype=torch.int32, device=dev), torch.zeros(6, dtype=torch.int32, device=dev)
    cos = torch.zeros(8, d, device=dev)
    lists = [[0.0] * 4, np.zeros((5, kv, d), np.float32), 3, "x"]
    for t in lists:
        for call in (
            lambda: cache.enqueueAppend(t, x, slots),
            lambda: cache.enqueueAppend(x, t, slots),
            lambda: cache.enqueueAppend(x, x, t),
            lambda: cache.enqueueAppend(x, x, slots, queries=t, queriesOut=x.clone()),
            lambda: cache.enqueueAppend(x, x, slots, queries=x, queriesOut=t),
            lambda: cache.enqueueAppend(x, x, slots, keyNorm=t),
            lambda: cache.enqueueAppend(x, x, slots, cos=t, sin=cos, positions=slots),
            lambda: cache.enqueueAppend(x, x, slots, cos=cos, sin=t, positions=slots),
            lambda: cache.enqueueAppend(x, x, slots, cos=cos, sin=cos, positions=t),
            lambda: cache.enqueueDecode(t, starts, keysOut=x),
            lambda: cache.enqueueDecode(table, t, keysOut=x),
            lambda: cache.enqueueDecode(table, starts, keysOut=t),
            lambda: cache.enqueueDecode(table, starts, keysOut=x, firstTokens=t),
            lambda: cache.enqueueAttention(t, table, lengths, x),
            lambda: cache.enqueueAttention(x, t, lengths, x),
            lambda: cache.enqueueAttention(x, table, t, x),
            lambda: cache.enqueueAttention(x, table, lengths, t),
            lambda: cache.enqueueAttention(x, table, lengths, x, slopes=t),
            lambda: cache.enqueueAttention(x, table, lengths, x, workspace=t),
            lambda: P.PagedCache(q, cfg, cfg, pages=4, pageSize=16, kvHeads=kv, keyCodes=t, keyScales=cache.keyScales,
                                 valueCodes=cache.valueCodes, valueScales=cache.valueScales),
        ):
            with pytest.raises(P.InvalidInput):
                call()


@pytest.mark.parametrize("value", [None, "x", [1.0]])
def test_numbers_that_are_none(q, value):
    import torch
    import pitch_amd as P
    dev, d = q.device, 64
    cfg = q.config("turboQuant", d, 4)
    cache = P.PagedCache(q, cfg, cfg, pages=4, pageSize=16)
    x, table = torch.zeros(5, 1, d, device=dev, dtype=torch.bfloat16), torch.zeros(5, 2, dtype=torch.int32, device=dev)
    lengths = torch.ones(5, dtype=torch.int32, device=dev)
    with pytest.raises(P.InvalidInput, match="eps"):
        cache.enqueueAppend(x, x, torch.arange(5, device=dev), eps=value)
    with pytest.raises(P.InvalidInput, match="softcap"):
        cache.enqueueAttention(x, table, lengths, x, softcap=value)
    if value is not None:      # (the default scale)
        with pytest.raises(P.InvalidInput, match="scale"):
            cache.enqueueAttention(x, table, lengths, x, scale=value)
