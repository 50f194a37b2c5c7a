"""Rows that are cut into pages which other rows hold as well: what goes wrong if they take tokens as they are, and the two forks that
give every row a last page of its own, which need nothing that only the device knows. On the CPU with the definition of the operators,
and on the GPU in a captured step."""
import numpy as np
import pytest

from pages_reference import Tables

ROWS, WIDTH, PAGE, PAGES = 5, 8, 16, 200
OUT, BACK = np.concatenate([np.arange(ROWS), np.arange(ROWS)]), np.concatenate([np.arange(ROWS, 2 * ROWS), np.full(ROWS, -1)])


class Plan:
    """Steps of a program: beams of `parents`, sequences cut to `keep`, `new` tokens; and the tokens (numbers) that each row then holds."""

    def __init__(self, seed):
        self.rng, self.rows, self.next = np.random.default_rng(seed), [[] for _ in range(ROWS)], 1

    def step(self):
        parents = np.where(self.rng.random(ROWS) < 0.5, np.arange(ROWS), self.rng.integers(0, ROWS, ROWS))
        rows = [list(self.rows[p]) for p in parents]
        keep = np.array([max(0, len(r) - int(self.rng.integers(0, 40))) for r in rows])
        new = self.rng.integers(0, 30, ROWS)
        new = np.minimum(new, WIDTH * PAGE - keep)
        ids = np.arange(self.next, self.next + new.sum())
        self.next += int(new.sum())
        at = np.concatenate([[0], np.cumsum(new)])
        self.rows = [r[:k] + list(ids[at[b]:at[b + 1]]) for b, (r, k) in enumerate(zip(rows, keep))]
        tail = np.full(ROWS, -1)
        return np.concatenate([parents, tail]), np.concatenate([keep, 0 * keep]), np.concatenate([new, 0 * new]), ids


def _held(tables, lengths, pool):
    return [[pool[tables[b, i // PAGE], 0, i % PAGE] for i in range(lengths[b])] for b in range(ROWS)]


def _on_the_cpu(seed, apart):
    """Whether all rows of twelve steps hold the tokens that they were given."""
    plan, ref = Plan(seed), Tables(np.full((2 * ROWS, WIDTH), -1), np.zeros(2 * ROWS), np.zeros(PAGES), PAGE, [(np.zeros((PAGES, 1, PAGE)), 2)])
    for _ in range(12):
        parents, keep, new, ids = plan.step()
        ref.fork(parents)
        ref.trim(keep)
        if apart:
            ref.fork(OUT)
            assert ref.missing == 0
            ref.fork(BACK)
            assert (ref.lengths[ROWS:] == 0).all()
            for b in range(ROWS):     # the last page is the row's own
                assert ref.lengths[b] % PAGE == 0 or ref.references[ref.held(b)[-1]] == 1
        slots, _ = ref.reserve(new, len(ids) + 1)
        pool = ref.pools[0][0]
        pool[slots[:len(ids)] // PAGE, 0, slots[:len(ids)] % PAGE] = ids
        held = np.bincount([p for b in range(2 * ROWS) for p in ref.held(b)], minlength=PAGES)
        assert np.array_equal(held, ref.references)
        if _held(ref.tables, ref.lengths, pool) != plan.rows:
            return False
    return True


def test_tokens_are_written_over_without_the_forks():
    assert not all(_on_the_cpu(seed, False) for seed in range(5))


def test_no_token_is_written_over_with_them():
    assert all(_on_the_cpu(seed, True) for seed in range(5))


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["head", "token"])
def test_in_a_captured_step(q, layout):
    """Cut, part and hand out in one graph: nothing is read back, and every row keeps its tokens in every cache."""
    import torch
    import pitch_amd as P
    caches = [P.PagedCache(q, q.config("turboQuant", 64, 4), pages=PAGES, pageSize=PAGE, layout=layout) for _ in range(2)]
    tables = P.PagedTables(caches, sequences=2 * ROWS, width=WIDTH)
    i32 = lambda a: torch.tensor(np.array(a), dtype=torch.int32, device="cuda")  # noqa: E731
    parents, keep, new = (i32(np.zeros(2 * ROWS)) for _ in range(3))
    slots = torch.zeros(ROWS * 30, dtype=torch.int64, device="cuda")
    calls = [P.PagedFork(tables, parents), P.PagedTrim(tables, keep), P.PagedFork(tables, i32(OUT)), P.PagedFork(tables, i32(BACK)),
             P.PagedReserve(tables, new, slots)]
    for c in calls:
        c.enqueue()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in calls:
            c.enqueue()
    plan = Plan(7)
    for _ in range(12):
        *step, ids = plan.step()
        for t, a in zip((parents, keep, new), step):
            t.copy_(i32(a))
        graph.replay()
        torch.cuda.synchronize()
        assert int(tables.missing[0]) == 0
        got, where = tables.lengths.cpu().numpy(), tables.blockTables.cpu().numpy()
        assert (slots[:len(ids)] >= 0).all() and (slots[len(ids):] == -1).all()
        for i, c in enumerate(caches):
            c.keyScales.view(-1)[slots[:len(ids)]] = torch.tensor(ids, device="cuda").float() + i
            c.valueScales.view(-1)[slots[:len(ids)]] = -torch.tensor(ids, device="cuda").float() - i
            for scales, sign in ((c.keyScales, 1), (c.valueScales, -1)):
                pool = scales.view(PAGES, 1, PAGE).cpu().numpy() * sign - i
                assert _held(where, got, pool) == plan.rows
