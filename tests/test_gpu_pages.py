"""The pages' bookkeeping on the device against the same in numpy, entry by entry: every table, count, slot and byte of the pools."""
import numpy as np
import pytest
import torch

import pitch_amd as P
from pages_reference import Tables

pytestmark = pytest.mark.gpu


def _i32(a):
    return torch.tensor(np.array(a).copy(), dtype=torch.int32, device="cuda")


def _caches(q, pages, page, layers, seed=0):
    """Caches of random bytes; layers: (kv heads, dim, key bits, value bits, layout)."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    made = []
    for kv, dim, kb, vb, layout in layers:
        c = P.PagedCache(q, q.config("turboQuant", dim, kb), q.config("polarQuant", dim, vb), pages=pages, pageSize=page, kvHeads=kv,
                         layout=layout)
        for t in (c.keyCodes, c.valueCodes):
            t.copy_(torch.randint(0, 256, t.shape, generator=gen, device="cuda", dtype=torch.uint8))
        for t in (c.keyScales, c.valueScales):
            t.copy_(torch.rand(t.shape, generator=gen, device="cuda"))
        made.append(c)
    return made


def _buffers(c):
    return (c.keyCodes, c.keyScales, c.valueCodes, c.valueScales)


def _state(rng, sequences, width, page, pages, share=0.6):
    """Random tables: lengths, pages in no order, some shared by two rows."""
    lengths = [int(x) for x in rng.integers(0, width * page + 1, sequences)]
    lengths[0] = 0
    ids = list(rng.permutation(pages))
    tables, references = np.full((sequences, width), -1), np.zeros(pages, dtype=np.int64)
    for b in range(sequences):
        n = -(-lengths[b] // page)
        if n > len(ids) * share:
            lengths[b] = n = 0
        tables[b, :n] = [ids.pop() for _ in range(n)]
        references[tables[b, :n]] += 1
    return tables, lengths, references


def _both(q, rng, sequences, width, page, pages, layers=((2, 64, 4, 3, "head"),), share=0.6):
    caches = _caches(q, pages, page, layers, seed=int(rng.integers(1 << 30)))
    tables, lengths, references = _state(rng, sequences, width, page, pages, share)
    t = P.PagedTables(caches, blockTables=_i32(tables), lengths=_i32(lengths), references=_i32(references))
    pools = [(b.cpu().numpy(), 2 if c.layout == "head" else 1) for c in caches for b in _buffers(c)]
    return t, Tables(tables, lengths, references, page, pools)


def _same(t, ref, what=""):
    torch.cuda.synchronize()
    for name, got, want in (("tables", t.blockTables, ref.tables), ("lengths", t.lengths, ref.lengths),
                            ("references", t.references, ref.references)):
        assert np.array_equal(got.cpu().numpy(), want), f"{what}: {name}"
    assert int(t.missing[0]) == ref.missing, f"{what}: missing"
    for i, (got, (want, _)) in enumerate(zip([b for c in t.caches for b in _buffers(c)], ref.pools)):
        assert np.array_equal(got.cpu().numpy(), want), f"{what}: pool {i}"


def _reserve(t, ref, new, capacity, what=""):
    slots, positions = (torch.full((capacity,), 77, dtype=torch.int64, device="cuda") for _ in range(2))
    t.enqueueReserve(_i32(new), slots, positions=positions)
    want = ref.reserve(new, capacity)
    torch.cuda.synchronize()
    assert np.array_equal(slots.cpu().numpy(), want[0]) and np.array_equal(positions.cpu().numpy(), want[1]), what
    _same(t, ref, what)


SHAPES = [(1, 1, 16, 3), (5, 7, 16, 60), (9, 30, 32, 500), (70, 5, 48, 300), (300, 3, 16, 2000), (2048, 2, 16, 5000), (3, 400, 16, 1300)]


@pytest.mark.parametrize("sequences,width,page,pages", SHAPES)
def test_reserve(q, sequences, width, page, pages):
    rng = np.random.default_rng(sequences + pages)
    for new, room in ((rng.integers(0, 4, sequences), 10), (rng.integers(-3, 3 * page, sequences), 0), (np.full(sequences, 1), -1),
                      (np.full(sequences, 2 ** 31 - 1), None), (np.zeros(sequences), 5)):
        t, ref = _both(q, rng, sequences, width, page, pages)
        total = int(np.maximum(new, 0).sum())
        _reserve(t, ref, new, 3000 if room is None else max(1, total + room), (sequences, new[:4]))


def test_reserve_until_nothing_is_left(q):
    rng = np.random.default_rng(3)
    t, ref = _both(q, rng, 6, 40, 16, 50, share=0.3)
    for _ in range(30):
        new = rng.integers(0, 23, 6)
        _reserve(t, ref, new, int(new.sum()) + 2)
    assert ref.missing > 0


@pytest.mark.parametrize("sequences,width,page,pages", SHAPES)
def test_trim(q, sequences, width, page, pages):
    rng = np.random.default_rng(sequences)
    t, ref = _both(q, rng, sequences, width, page, pages)
    for keep in (np.full(sequences, 2 ** 31 - 1), rng.integers(-5, width * page + 9, sequences), ref.lengths - 1, np.full(sequences, -2 ** 31)):
        t.enqueueTrim(_i32(keep))
        ref.trim(keep)
        _same(t, ref)


LAYERS = [((2, 64, 4, 3, "head"),), ((1, 128, 3, 8, "token"), (3, 64, 2, 5, "head")), ((8, 128, 4, 4, "head"), (2, 128, 7, 2, "token"))]


@pytest.mark.parametrize("layers", LAYERS)
@pytest.mark.parametrize("sequences,width,page,pages", SHAPES)
def test_fork(q, sequences, width, page, pages, layers):
    rng = np.random.default_rng(sequences * 7 + len(layers))
    t, ref = _both(q, rng, sequences, width, page, pages, layers)
    identity = np.arange(sequences)
    for parents in (identity, rng.integers(0, sequences, sequences), np.where(rng.random(sequences) < 0.5, identity, rng.integers(-2, sequences + 2, sequences)),
                    identity[::-1], np.full(sequences, sequences // 2), np.full(sequences, -1)):
        t.enqueueFork(_i32(parents))
        ref.fork(parents)
        _same(t, ref, parents[:5])


def test_fork_without_free_pages(q):
    """Children whose last page cannot be copied end with their parent's whole pages; pages that a row gives up are handed out again."""
    for pages, first in ((4, [33, 0, 0, 0, 0]), (7, [50, 20, 0, 40, 0])):
        caches = _caches(q, pages, 16, [(2, 64, 4, 4, "head")])
        tables, at = np.full((5, 6), -1), 0
        for b, n in enumerate(first):
            k = -(-n // 16)
            tables[b, :min(k, pages - at)] = range(at, min(at + k, pages))
            first[b], at = min(n, (pages - at) * 16), min(at + k, pages)
        references = np.bincount(tables[tables >= 0], minlength=pages)
        for parents in ([0, 0, 0, 0, 0], [0, 1, 0, 3, 1], [3, 3, 3, 3, 0], [1, 0, 3, 2, 4]):
            t = P.PagedTables(caches, blockTables=_i32(tables), lengths=_i32(first), references=_i32(references))
            ref = Tables(tables, first, references, 16, [(b.cpu().numpy(), 2) for b in _buffers(caches[0])])
            t.enqueueFork(_i32(parents))
            ref.fork(parents)
            _same(t, ref, parents)


@pytest.mark.parametrize("layers", LAYERS)
@pytest.mark.parametrize("sequences,width,page,pages", SHAPES)
def test_compact(q, sequences, width, page, pages, layers):
    for share in (0.05, 0.6, 1.0):
        rng = np.random.default_rng(pages)
        t, ref = _both(q, rng, sequences, width, page, pages, layers, share)
        extra = int(rng.integers(pages))          # a page that the program keeps for itself
        t.references[extra] += 1
        ref.references[extra] += 1
        mapping, used = _i32(np.full(pages, 9)), _i32([0])
        t.enqueueCompact(mapping=mapping, used=used)
        want, n = ref.compact()
        _same(t, ref)
        assert np.array_equal(mapping.cpu().numpy(), want) and int(used[0]) == n
        assert (ref.references[:n] > 0).all() and (ref.references[n:] <= 0).all()
        t.enqueueCompact()                        # a second one moves nothing
        ref.compact()
        _same(t, ref)


@pytest.mark.parametrize("full", [False, True])
def test_compact_of_empty_and_full_pools(q, full):
    caches = _caches(q, 20, 16, [(1, 64, 4, 4, "head")])
    tables = np.arange(20).reshape(2, 10)[:, ::-1] if full else np.full((2, 10), -1)
    lengths, references = ([160, 145], np.ones(20)) if full else ([0, 0], np.zeros(20))
    t = P.PagedTables(caches, blockTables=_i32(tables.copy()), lengths=_i32(lengths), references=_i32(references))
    ref = Tables(tables, lengths, references, 16, [(b.cpu().numpy(), 2) for b in _buffers(caches[0])])
    mapping, used = _i32(np.full(20, 9)), _i32([5])
    t.enqueueCompact(mapping=mapping, used=used)
    want, n = ref.compact()
    _same(t, ref)
    assert np.array_equal(mapping.cpu().numpy(), want) and int(used[0]) == n == (20 if full else 0)


def test_state_that_is_not_right(q):
    """Lengths and entries out of range, counts below zero: cut, left alone or taken as free, never followed out of the pool."""
    rng = np.random.default_rng(8)
    for op in ("reserve", "trim", "fork", "compact"):
        caches = _caches(q, 40, 16, [(2, 64, 4, 4, "head")])
        tables = rng.integers(-3, 45, (6, 5))
        tables[0, 1], tables[1, 0] = 2 ** 31 - 1, -2 ** 31
        lengths = [2 ** 31 - 1, 70, -2 ** 31, 33, -1, 80]
        references = np.zeros(40, dtype=np.int64)
        for b in range(6):
            row = tables[b, :-(-min(max(lengths[b], 0), 80) // 16)]
            np.add.at(references, row[(row >= 0) & (row < 40)], 1)
        references[rng.integers(0, 40, 5)] -= 2
        t = P.PagedTables(caches, blockTables=_i32(tables), lengths=_i32(lengths), references=_i32(references))
        ref = Tables(tables, lengths, references, 16, [(b.cpu().numpy(), 2) for b in _buffers(caches[0])])
        if op == "reserve":
            _reserve(t, ref, [3, 20, 40, 0, 7, 2], 80)
        elif op == "trim":
            t.enqueueTrim(_i32([40, 2, 5, 1, 0, 70]))
            ref.trim([40, 2, 5, 1, 0, 70])
            _same(t, ref)
        elif op == "fork":
            t.enqueueFork(_i32([2, 1, 3, 3, 5, -1]))
            ref.fork([2, 1, 3, 3, 5, -1])
            for name, got, want in (("tables", t.blockTables, ref.tables), ("lengths", t.lengths, ref.lengths),
                                    ("references", t.references, ref.references)):
                assert np.array_equal(got.cpu().numpy(), want), name
        else:
            t.enqueueCompact()
            ref.compact()
            for name, got, want in (("tables", t.blockTables, ref.tables), ("references", t.references, ref.references)):
                assert np.array_equal(got.cpu().numpy(), want), name


def test_layers_that_lie_between_each_other(q):
    """Layers' parts of one buffer [page][layer][head][slot], more layers than one launch's arguments hold."""
    rng = np.random.default_rng(9)
    pages, page, layers, kv = 30, 16, 53, 2
    kc, vc = q.config("turboQuant", 64, 3), q.config("turboQuant", 64, 4)
    made = []
    for c in (kc, vc):
        made += [torch.randint(0, 256, (pages, layers, kv, page, c.codeStride), device="cuda", dtype=torch.uint8),
                 torch.rand((pages, layers, kv, page), device="cuda")]
    caches = [P.PagedCache(q, kc, vc, pages=pages, pageSize=page, kvHeads=kv, keyCodes=made[0][:, i], keyScales=made[1][:, i],
                           valueCodes=made[2][:, i], valueScales=made[3][:, i]) for i in range(layers)]
    tables, lengths, references = _state(rng, 4, 6, page, pages)
    lengths[1] = 37
    lengths[2] = lengths[3] = 0
    tables[1, :3] = [29, 5, 11]
    references = np.bincount(np.concatenate([tables[b, :-(-lengths[b] // page)] for b in range(4)]), minlength=pages)
    t = P.PagedTables(caches, blockTables=_i32(tables), lengths=_i32(lengths), references=_i32(references))
    ref = Tables(tables, lengths, references, page, [(b.cpu().numpy(), 2) for c in caches for b in _buffers(c)])
    t.enqueueFork(_i32([0, 1, 1, 1]))
    ref.fork([0, 1, 1, 1])
    _same(t, ref)
    t.enqueueCompact()
    ref.compact()
    _same(t, ref)


def test_large_pages_and_a_large_pool(q):
    """Pages of several slices, and a pool of more segments than a workgroup has threads."""
    rng = np.random.default_rng(10)
    t, ref = _both(q, rng, 3, 2, 4096, 7, [(5, 128, 8, 5, "head"), (4, 64, 3, 2, "token")], share=1.0)
    for parents in ([1, 1, 2], [2, 1, 1]):
        t.enqueueFork(_i32(parents))
        ref.fork(parents)
        _same(t, ref)
    t.enqueueCompact()
    ref.compact()
    _same(t, ref)
    pages = 1_500_000
    cache = P.PagedCache(q, q.config("turboQuant", 64, 2), pages=pages, pageSize=16, kvHeads=1)
    references = np.ones(pages, dtype=np.int64)
    holes = np.sort(rng.choice(pages, 700, replace=False))
    references[holes] = 0
    t = P.PagedTables(cache, blockTables=_i32(np.full((4, 300), -1)), lengths=_i32([0, 5, 0, 0]), references=_i32(references))
    slots = torch.zeros(5000, dtype=torch.int64, device="cuda")
    t.enqueueReserve(_i32([1000, 11, 2000, 16 * 90]), slots)
    torch.cuda.synchronize()
    got = t.blockTables.cpu().numpy()
    assert np.array_equal(got[0, :63], holes[:63]) and np.array_equal(got[2, :125], holes[63:188])
    assert np.array_equal(got[3, :90], holes[188:278]) and int(t.lengths[1]) == 16
    mapping, used = _i32(np.zeros(pages)), _i32([0])
    t.enqueueCompact(mapping=mapping, used=used)
    want = np.arange(pages)
    free = holes[278:]
    n = pages - len(free)
    low = free[free < n]
    want[free] = -1
    want[np.array([p for p in range(n, pages) if want[p] >= 0], dtype=np.int64)] = low
    assert int(used[0]) == n and np.array_equal(mapping.cpu().numpy(), want)


def test_a_random_program(q):
    """All four calls in turn, many times."""
    rng = np.random.default_rng(11)
    t, ref = _both(q, rng, 12, 9, 16, 90, [(2, 64, 4, 3, "head"), (1, 128, 2, 6, "token")], share=0.4)
    for step in range(60):
        what = rng.integers(4)
        if what == 0:
            new = rng.integers(0, 30, 12)
            _reserve(t, ref, new, int(new.sum()) + 1, step)
        elif what == 1:
            keep = np.where(rng.random(12) < 0.6, 10 ** 6, ref.lengths - rng.integers(0, 40, 12))
            t.enqueueTrim(_i32(keep))
            ref.trim(keep)
        elif what == 2:
            parents = np.where(rng.random(12) < 0.6, np.arange(12), rng.integers(-1, 12, 12))
            t.enqueueFork(_i32(parents))
            ref.fork(parents)
        else:
            t.enqueueCompact()
            ref.compact()
        _same(t, ref, step)


def test_graph(q):
    """A captured reserve, trim and fork serve every step: what they read and change lies on the device."""
    rng = np.random.default_rng(12)
    t, ref = _both(q, rng, 8, 12, 16, 160, share=0.3)
    new, keep, parents = _i32(np.zeros(8)), _i32(np.full(8, 10 ** 6)), _i32(np.arange(8))
    slots, positions = (torch.zeros(40, dtype=torch.int64, device="cuda") for _ in range(2))
    calls = [P.PagedFork(t, parents), P.PagedTrim(t, keep), P.PagedReserve(t, new, slots, positions=positions), P.PagedCompact(t)]
    for c in calls:
        c.enqueue()
    ref.fork(np.arange(8))
    ref.trim(np.full(8, 10 ** 6))
    ref.reserve(np.zeros(8), 40)
    ref.compact()
    _same(t, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in calls:
            c.enqueue()
    for step in range(6):
        n, k, p = rng.integers(0, 5, 8), ref.lengths - rng.integers(-3, 9, 8), np.where(rng.random(8) < 0.6, np.arange(8), rng.integers(0, 8, 8))
        new.copy_(_i32(n))
        keep.copy_(_i32(k))
        parents.copy_(_i32(p))
        graph.replay()
        ref.fork(p)
        ref.trim(k)
        want = ref.reserve(n, 40)
        ref.compact()
        _same(t, ref, step)
        assert np.array_equal(slots.cpu().numpy(), want[0]) and np.array_equal(positions.cpu().numpy(), want[1])


def test_calls_on_another_stream(q):
    rng = np.random.default_rng(13)
    t, ref = _both(q, rng, 8, 12, 16, 160)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    parents = _i32([1, 1, 2, 3, 3, 3, 0, 7])
    torch.cuda.synchronize()
    t.enqueueFork(parents, stream=s)
    t.enqueueCompact(stream=s.cuda_stream)
    s.synchronize()
    ref.fork([1, 1, 2, 3, 3, 3, 0, 7])
    ref.compact()
    _same(t, ref)
