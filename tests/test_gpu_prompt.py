"""Attention over whole prompts against its definition in 64 bits: packed sequences of every kind of length, both types and
dimensions, grouped heads, masks, strides, values that are not finite, split keys, streams and graphs."""
import math

import numpy as np
import pytest
import torch

import pitch_amd as P
from prompt_reference import compare, reference, starts

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16]


def _inputs(lengths, heads, kv, dim, dtype, seed=0, prefixed=False, extra=3):
    """q, k, v on the device (rows behind the last sequence included) and the starts."""
    rng = torch.Generator().manual_seed(seed)
    new, keys = [n for n, _ in lengths], [n for _, n in lengths]
    rows, cached = sum(new) + extra, sum(keys) + extra
    q = torch.randn((rows, heads, dim), generator=rng) * 1.3
    k = (torch.randn((cached, kv, dim), generator=rng) + 0.4) * torch.exp(0.4 * torch.randn((kv, dim), generator=rng))
    v = torch.randn((cached, kv, dim), generator=rng) * torch.exp(torch.randn((cached, kv, 1), generator=rng) * 0.5)
    return [t.to(dtype).cuda() for t in (q, k, v)] + [starts(new), starts(keys)]


def _dev(a):
    return torch.tensor(a, dtype=torch.int32, device="cuda")


def _run(pitch, q, k, v, rs, ks, out=None, **more):
    out = torch.full_like(q, 7.0) if out is None else out
    lse = torch.full(q.shape[:2], 7.0, device="cuda")
    P.PromptAttention(pitch, q, k, v, _dev(rs), out, keyStarts=_dev(ks), lse=lse, **more).enqueue()
    torch.cuda.synchronize()
    return out, lse


def _check(pitch, lengths, heads, kv, dim, dtype, seed=0, **more):
    q, k, v, rs, ks = _inputs(lengths, heads, kv, dim, dtype, seed)
    out, lse = _run(pitch, q, k, v, rs, ks, **more)
    compare(out, lse, reference(q, k, v, rs, ks, **more))
    assert bool((out[rs[-1]:] == 7).all()) and bool((lse[rs[-1]:] == 7).all())


MIXED = [(1, 1), (0, 0), (77, 77), (2, 2), (64, 64), (65, 65), (0, 5), (128, 128), (130, 300), (1, 200), (33, 64), (5, 3), (3, 0)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("kv,group", [(1, 1), (2, 6), (3, 4), (1, 8), (2, 13)])
def test_packed_sequences(q, dtype, dim, kv, group):
    _check(q, MIXED, kv * group, kv, dim, dtype)


@pytest.mark.parametrize("kv,group,lengths", [(1, 200, [(3, 70), (130, 140)]), (600, 1, [(2, 2100), (3, 3)]), (1, 64, [(2, 2500)])])
def test_many_heads(q, kv, group, lengths):
    """A token that fills more than a query tile, and more KV heads than the device has places for workgroups."""
    _check(q, lengths, kv * group, kv, 64, torch.float16, seed=38)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("more", [
    dict(causal=False), dict(window=1), dict(window=7), dict(window=64), dict(window=100), dict(window=2 ** 31 - 1), dict(softcap=5.0),
    dict(softcap=50.0, window=30), dict(scale=0.0), dict(scale=-0.2), dict(scale=1.0), dict(softcap=3.0, scale=-0.3), dict(causal=False, softcap=9.0)])
def test_masks_and_scores(q, dim, more):
    for dtype in TYPES:
        _check(q, MIXED, 6, 2, dim, dtype, seed=1, **more)


@pytest.mark.parametrize("softcap", [1e-30, 1e-3, 0.1, 1.0, 100.0, 1e4, 1e20, 3e38])
def test_soft_caps_of_any_size(q, softcap):
    """A cap far above the scores leaves them as they are, one far below makes them signs."""
    for dtype in TYPES:
        _check(q, [(1, 1), (40, 90), (3, 3)], 4, 2, 64, dtype, seed=34, softcap=softcap)
        _check(q, [(70, 70)], 2, 1, 128, dtype, seed=35, softcap=softcap, scale=-0.4)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("window,softcap", [(0, 0.0), (50, 0.0), (0, 20.0)])
def test_slopes(q, dim, window, softcap):
    lengths = MIXED
    qq, k, v, rs, ks = _inputs(lengths, 8, 2, dim, torch.float16, 2)
    slopes = 2.0 ** (-torch.arange(1, 9, device="cuda", dtype=torch.float32))
    out, lse = _run(q, qq, k, v, rs, ks, slopes=slopes, window=window, softcap=softcap)
    compare(out, lse, reference(qq, k, v, rs, ks, slopes=slopes.cpu(), window=window, softcap=softcap))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[(700, 700)], [(1, 1500)], [(4, 3000), (1, 17), (0, 900)], [(100, 2100)], [(300, 301), (1, 900)]])
def test_long_sequences(q, dtype, lengths):
    _check(q, lengths, 8, 2, 128, dtype, seed=3)
    _check(q, lengths, 4, 2, 64, dtype, seed=4, window=400)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("more", [dict(), dict(causal=False), dict(window=2100), dict(softcap=8.0)])
def test_tiles_that_are_cut(q, dtype, more):
    """Few query tiles of very different lengths: workgroups share them, beginning and ending within a tile."""
    _check(q, [(500, 4500), (130, 2500), (0, 100), (1, 5000), (33, 40), (20, 3), (64, 700)], 8, 2, 128, dtype, seed=30, **more)
    _check(q, [(7, 9000)], 3, 1, 64, dtype, seed=31, **more)
    _check(q, [(900, 2300), (300, 2900)], 2, 1, 64, dtype, seed=32, **more)


def test_many_sequences_over_long_keys(q):
    """A thousand sequences and more, most of a token, some of them long."""
    for n in (700, 1024, 1025):
        rng = np.random.default_rng(n)
        lengths = [(int(a), int(a + b)) for a, b in zip(rng.integers(0, 3, n), rng.integers(0, 9, n))]
        lengths[n // 2] = (40, 3000)
        lengths[-1] = (1, 2500)
        _check(q, lengths, 2, 1, 64, torch.bfloat16, seed=33)


@pytest.mark.parametrize("dim,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_parts_of_many_rows(q, dim, dtype):
    """A long sequence among short ones: its tiles are cut, and joined by workgroups that take rows one after the other."""
    _check(q, [(500, 560), (600, 5000), (1, 1), (500, 520), (590, 600)], 32, 8, dim, dtype, seed=34)


@pytest.mark.parametrize("heads", [(4, 2), (8, 8)])
def test_orders_of_tiles(q, heads):
    """Uneven sequences, with and without keys before their queries, some empty: few tiles and many (which come in another order)."""
    rng = np.random.default_rng(35)
    lengths = [(int(n), int(n + p * (p % 3 == 0))) for n, p in zip(rng.integers(0, 300, 290), rng.integers(0, 400, 290))]
    lengths[7] = lengths[100] = (0, 0)
    _check(q, lengths, *heads, 64, torch.bfloat16, seed=35)
    _check(q, lengths[:50], *heads, 64, torch.float16, seed=36)


def test_more_sequences_than_a_wave_has_lanes(q):
    rng = np.random.default_rng(5)
    lengths = [(int(n), int(n + p)) for n, p in zip(rng.integers(0, 9, 333), rng.integers(0, 30, 333))]
    _check(q, lengths, 4, 2, 64, torch.bfloat16, seed=5)


def test_scores_that_grow_from_tile_to_tile(q):
    """The largest score comes late, early or in between, by far more than the maximum in use may lag behind."""
    for order in (1, -1):
        qq, k, v, rs, ks = _inputs([(600, 600)], 2, 1, 64, torch.bfloat16, 6)
        grow = torch.linspace(0, 9, 603, device="cuda")
        k = (k * (grow if order > 0 else grow.flip(0))[:, None, None]).to(torch.bfloat16)
        out, lse = _run(q, qq, k, v, rs, ks)
        compare(out, lse, reference(qq, k, v, rs, ks))


@pytest.mark.parametrize("dtype", TYPES)
def test_slices_transposed_and_broadcast_views(q, dtype):
    lengths, kv, group, dim = MIXED, 2, 3, 64
    lengths = [(n, n) for n, _ in lengths]
    rows = sum(n for n, _ in lengths) + 3
    qkv = torch.randn((rows, kv * group + 2 * kv, dim), generator=torch.Generator().manual_seed(7)).to(dtype).cuda()
    a, b, c = qkv[:, :kv * group], qkv[:, kv * group:kv * group + kv], qkv[:, kv * group + kv:]
    rs = starts([n for n, _ in lengths])
    want = reference(a, b, c, rs, rs)
    out, lse = _run(q, a, b, c, rs, rs)
    compare(out, lse, want)
    # head-major memory, the output too
    turned = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (a, b, c)]
    out2, lse2 = _run(q, *turned, rs, rs, out=torch.full_like(turned[0].transpose(0, 1).contiguous(), 7.0).transpose(0, 1))
    assert torch.equal(out, out2) and torch.equal(lse, lse2)
    # in place, in the projection's own buffer
    _run(q, a, b, c, rs, rs, out=a)
    assert torch.equal(out[:rs[-1]], a[:rs[-1]])
    # one key and value vector for all heads and tokens
    one = b[:1, :1].expand(rows, kv, dim)
    out, lse = _run(q, turned[0], one, one, rs, rs)
    compare(out, lse, reference(turned[0], one, one, rs, rs))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dim", [64, 128])
def test_what_is_hidden_has_no_effect(q, dtype, dim):
    """NaN and infinities in later tokens, in other sequences, behind the window and behind the last sequence."""
    bad = [math.nan, math.inf, -math.inf]
    lengths = [(50, 50), (130, 130), (40, 200)]
    qq, k, v, rs, ks = _inputs(lengths, 4, 2, dim, dtype, 8)
    for i, at in enumerate((49, ks[1] + 100, ks[1] + 129, ks[2] + 3, ks[-1])):
        k[at], v[at] = bad[i % 3], bad[(i + 1) % 3]
    qq[rs[1] + 5, 1] = math.nan
    for more in (dict(), dict(window=20), dict(softcap=10.0)):
        out, lse = _run(q, qq, k, v, rs, ks, **more)
        compare(out, lse, reference(qq, k, v, rs, ks, **more))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths", [[(70, 70), (200, 200)], [(3, 3000)]])   # (the second's keys are cut into parts)
def test_values_that_are_not_finite(q, dtype, lengths):
    """Each coordinate of each row gets NaN, an infinity or its sum, by what its visible values hold."""
    qq, k, v, rs, ks = _inputs(lengths, 4, 2, 64, dtype, 9)
    at = ks[-1] - 1
    v[at - 60, 0, 3], v[at - 20, 0, 3] = math.inf, -math.inf
    v[at - 50, 0, 4], v[at - 40, 1, 63], v[at - 30, 1, 7] = math.inf, -math.inf, math.nan
    v[at, 1, 9], v[ks[1] - 2, 0, 0] = math.nan, math.inf
    out, lse = _run(q, qq, k, v, rs, ks)
    compare(out, lse, reference(qq, k, v, rs, ks))


@pytest.mark.parametrize("dim", [64, 128])
def test_values_that_are_not_finite_in_other_parts(q, dim):
    """What one part holds reaches the joined row, also where that part's weight has become zero (e^-106
    and less against the others' scores)."""
    qq, k, v, rs, ks = _inputs([(3, 3000), (5, 2500)], 4, 2, dim, torch.bfloat16, 37)
    qq[:, :, 0] = 4.0
    k[:, :, 0] = torch.where(torch.arange(len(k), device="cuda") % 2600 < 200, -300.0, 0.0)[:, None]
    v[20, 0, 3], v[30, 0, 3], v[40, 0, 4], v[50, 1, 5], v[3100, 1, 6] = math.inf, -math.inf, math.inf, math.nan, -math.inf
    v[2900, 1, 7], v[5300, 0, 8], v[5310, 1, 9] = math.inf, math.nan, math.inf
    out, lse = _run(q, qq, k, v, rs, ks)
    compare(out, lse, reference(qq, k, v, rs, ks))
    assert bool(torch.isnan(out[:3, :2, 3]).all()) and bool((out[:3, :2, 4] == math.inf).all())


def test_scores_of_minus_infinity_take_no_part(q):
    qq, k, v, rs, ks = _inputs([(90, 90)], 2, 1, 64, torch.float16, 10)
    qq[:, :, 0] = 1.0
    k[10:20, :, 0] = -math.inf
    k[0, :, 0] = -math.inf      # the first query sees nothing else
    v[12] = math.nan            # and its value does not matter then
    out, lse = _run(q, qq, k, v, rs, ks)
    assert bool((out[0] == 0).all()) and bool((lse[0] == -math.inf).all())
    keep = [i for i in range(90) if i not in (0, *range(10, 20))]
    for i in (5, 15, 89):
        sub = [j for j in keep if j <= i]
        want = reference(qq[i:i + 1], k[sub], v[sub], [0, 1], [0, len(sub)])
        compare(out[i:i + 1], lse[i:i + 1], want)


def test_starts_that_leave_the_buffers(q):
    """Starts are cut to the buffers; a sequence that would begin behind its end is empty."""
    qq, k, v, rs, ks = _inputs([(40, 40)], 2, 1, 64, torch.bfloat16, 11, extra=0)
    want, want_lse = _run(q, qq, k, v, [0, 40], [0, 40])
    for bad in ([-7, 4000], [-2 ** 31, 2 ** 31 - 1]):
        out, lse = _run(q, qq, k, v, bad, bad)
        assert torch.equal(out, want) and torch.equal(lse, want_lse)
    out, lse = _run(q, qq, k, v, [30, 10], [0, 40])
    assert bool((out == 7).all())


def test_a_call_is_the_same_whatever_else_it_holds(q):
    """A sequence's rows are the same bits alone and among others, in unsplit calls."""
    qq, k, v, rs, ks = _inputs([(200, 200)] * 40, 8, 2, 128, torch.bfloat16, 12, extra=0)
    whole, lse = _run(q, qq, k, v, rs, ks)
    again, lse2 = _run(q, qq, k, v, rs, ks)
    assert torch.equal(whole, again) and torch.equal(lse, lse2)
    some, _ = _run(q, qq[:7800], k[:7800], v[:7800], rs[:40], ks[:40])
    assert torch.equal(whole[:7800], some)


def test_graph_and_streams(q):
    """A captured call is replayed over changing contents and starts; calls on several streams have workspaces of their own."""
    qq, k, v, rs, ks = _inputs([(3, 2400), (2, 700)], 8, 2, 128, torch.bfloat16, 13)
    drs, dks = _dev(rs), _dev(ks)
    out, lse = torch.full_like(qq, 7.0), torch.full(qq.shape[:2], 7.0, device="cuda")
    call = P.PromptAttention(q, qq, k, v, drs, out, keyStarts=dks, lse=lse)
    assert call.workspaceBytes > 0
    call.enqueue()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call.enqueue()
    for i in range(4):
        qq.copy_(torch.randn_like(qq))
        new, keys = [(3, 2), (1, 4), (5, 0), (0, 5)][i], [(1200, 700), (900, 1000), (1900, 0), (100, 1800)][i]
        drs.copy_(_dev(starts(new)))
        dks.copy_(_dev(starts(keys)))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        compare(out, lse, reference(qq, k, v, starts(new), starts(keys)))
    streams = [torch.cuda.Stream() for _ in range(3)]
    sets = [_inputs([(2, 2500)], 8, 2, 128, torch.float16, 20 + i) for i in range(3)]
    outs = [torch.zeros_like(s[0]) for s in sets]
    calls = [P.PromptAttention(q, *s[:3], _dev(s[3]), o, keyStarts=_dev(s[4])) for s, o in zip(sets, outs)]
    torch.cuda.synchronize()
    for _ in range(3):
        for c, s in zip(calls, streams):
            c.enqueue(s)
    torch.cuda.synchronize()
    for s, o in zip(sets, outs):
        want, _ = _run(q, *s)
        assert torch.equal(o[:2], want[:2])


def test_enqueue_of_the_codec(q):
    qq, k, v, rs, ks = _inputs([(20, 20)], 2, 1, 64, torch.float16, 14, extra=0)
    out = torch.zeros_like(qq)
    q.enqueuePromptAttention(qq, k, v, _dev(rs), out)
    want, _ = _run(q, qq, k, v, rs, ks)
    assert torch.equal(out, want)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    out.zero_()
    s.wait_stream(torch.cuda.current_stream())
    q.enqueuePromptAttention(qq, k, v, _dev(rs), out, stream=s)      # (no workspace is needed)
    s.synchronize()
    assert torch.equal(out, want)
    long = _inputs([(1, 3000)], 2, 1, 64, torch.float16, 15, extra=0)
    with pytest.raises(P.InvalidInput, match="workspace of its own"):
        q.enqueuePromptAttention(*long[:3], _dev(long[3]), torch.zeros_like(long[0]), keyStarts=_dev(long[4]), stream=s)


def test_keys_far_apart(q):
    """Keys whose rows and heads lie far apart: offsets pass 32 bits."""
    rows, kv, dim = 1100, 2, 64
    room = torch.empty(rows * (1 << 21) + (1 << 24), dtype=torch.float16, device="cuda")
    k = room.as_strided((rows, kv, dim), (1 << 21, 1 << 20, 1))
    v = room.as_strided((rows, kv, dim), (1 << 21, 1 << 20, 1), storage_offset=1 << 12)
    qq, a, b, rs, ks = _inputs([(rows, rows)], 4, kv, dim, torch.float16, 16, extra=0)
    k.copy_(a)
    v.copy_(b)
    out, lse = _run(q, qq, k, v, rs, ks)
    want, want_lse = _run(q, qq, a, b, rs, ks)
    assert torch.equal(out, want) and torch.equal(lse, want_lse)
