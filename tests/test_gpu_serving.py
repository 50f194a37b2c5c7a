"""The operators of a serving program in the order in which it runs them: prompts and drafted tokens get slots, are appended, read
back and attended to; beams fork; sequences end; the pool is compacted. Each step's attention is compared with the definition over the
vectors that the reference pool's codes stand for."""
import math

import numpy as np
import pytest
import torch

import pitch_amd as P
from prompt_reference import compare, reference, starts

pytestmark = pytest.mark.gpu
KV, GROUP, DIM, PAGE = 2, 3, 64, 16


def _i32(a):
    return torch.tensor(np.array(a).copy(), dtype=torch.int32, device="cuda")


class Program:
    """Two layers' caches, page tables, and the decoded vectors of every sequence's tokens, as they were when they were appended."""

    def __init__(self, q, sequences, width, pages):
        cfg = q.config("turboQuant", DIM, 4)
        self.q, self.n = q, sequences
        self.caches = [P.PagedCache(q, cfg, cfg, pages=pages, pageSize=PAGE, kvHeads=KV, layout=layout) for layout in ("head", "token")]
        self.tables = P.PagedTables(self.caches, sequences=sequences, width=width)
        self.rows = [[torch.zeros((0, 2, KV, DIM)) for _ in range(sequences)] for _ in self.caches]
        angle = torch.arange(500, dtype=torch.float64)[:, None] / 1e4 ** (torch.arange(0, DIM, 2) / DIM)
        self.cos, self.sin = (torch.cat([f(angle)] * 2, 1).float().cuda() for f in (torch.cos, torch.sin))
        self.seed = 0

    def tokens(self, new, padding=0):
        """New tokens of every sequence: slots, the append in every layer, and what attention makes of them."""
        new = list(new)
        total = sum(new) + padding
        slots, positions = (torch.zeros(total, dtype=torch.int64, device="cuda") for _ in range(2))
        before = self.tables.lengths.cpu().tolist()
        self.tables.enqueueReserve(_i32(new), slots, positions=positions)
        at = starts(new)
        for layer, cache in enumerate(self.caches):
            self.seed += 1
            gen = torch.Generator(device="cuda").manual_seed(self.seed)
            qkv = torch.randn((total, KV * GROUP + 2 * KV, DIM), generator=gen, device="cuda").to(torch.float16)
            qq, k, v = qkv[:, :KV * GROUP], qkv[:, KV * GROUP:-KV], qkv[:, -KV:]
            cache.enqueueAppend(k, v, slots, queries=qq, queriesOut=qq, cos=self.cos, sin=self.sin, positions=positions)
            lengths = [b + n for b, n in zip(before, new)]
            held = starts(lengths)
            keys, values = (torch.zeros((max(1, held[-1]), KV, DIM), dtype=torch.float16, device="cuda") for _ in range(2))
            cache.enqueueDecode(self.tables.blockTables, _i32(held), keysOut=keys, valuesOut=values)
            out, lse = torch.zeros((total, KV * GROUP, DIM), dtype=torch.float16, device="cuda"), torch.zeros((total, KV * GROUP), device="cuda")
            self.q.enqueuePromptAttention(qq, keys, values, _i32(at), out, keyStarts=_i32(held), lse=lse)
            torch.cuda.synchronize()
            assert self.tables.lengths.cpu().tolist() == lengths
            # the older tokens are still what they were
            for b in range(self.n):
                got = torch.stack([keys[held[b]:held[b + 1]], values[held[b]:held[b + 1]]], 1).cpu()
                assert torch.equal(got[:before[b]], self.rows[layer][b]), f"layer {layer}, sequence {b}"
                self.rows[layer][b] = got
            compare(out, lse, reference(qq, keys, values, at, held), f"layer {layer}")
            if max(new) == 1 and all(new):     # single tokens: the paged attention over codes says the same
                step = torch.zeros_like(out[:self.n])
                cache.enqueueAttention(qq[:self.n], self.tables.blockTables, self.tables.lengths, step)
                torch.cuda.synchronize()
                err = (step.float() - out[:self.n].float()).norm() / out[:self.n].float().norm()
                assert float(err) < 2e-3       # (keys and values rounded to float16 on the one side)

    def fork(self, parents):
        self.tables.enqueueFork(_i32(parents))
        self.rows = [[rows[p] if 0 <= p < self.n else rows[0][:0] for p in parents] for rows in self.rows]

    def trim(self, keep):
        self.tables.enqueueTrim(_i32(keep))
        self.rows = [[r[:max(0, k)] for r, k in zip(rows, keep)] for rows in self.rows]

    def check_pages(self):
        torch.cuda.synchronize()
        lengths, tables = self.tables.lengths.cpu().numpy(), self.tables.blockTables.cpu().numpy()
        held = np.concatenate([tables[b, :-(-lengths[b] // PAGE)] for b in range(self.n)] + [np.zeros(0, dtype=int)]).astype(int)
        assert np.array_equal(np.bincount(held, minlength=len(self.tables.references)), self.tables.references.cpu().numpy())
        assert int(self.tables.missing[0]) == 0


def test_a_program(q):
    p = Program(q, 4, 12, 60)
    p.tokens([37, 0, 100, 5], padding=3)          # prompts
    p.check_pages()
    p.tokens([1, 20, 1, 1])                       # a decode step beside a new prompt
    for _ in range(2):
        p.tokens([1, 1, 1, 1])
    p.fork([0, 0, 2, 0])                          # beams
    p.check_pages()
    for _ in range(3):
        p.tokens([1, 1, 1, 1])
    lengths = p.tables.lengths.cpu().tolist()
    p.tokens([5, 4, 0, 3])                        # drafts, some of them rejected
    p.trim([lengths[0] + 2, lengths[1], 10 ** 6, lengths[3] + 3])
    p.check_pages()
    p.tokens([1, 1, 1, 1])
    p.fork([3, 1, -1, 0])                         # two rows change places, one sequence ends
    p.tables.enqueueCompact()
    p.check_pages()
    assert bool((p.tables.references.cpu()[int((p.tables.references > 0).sum()):] == 0).all())
    p.tokens([2, 1, 50, 1])
    p.trim([0, 0, 0, 0])
    p.check_pages()
    assert not bool(p.tables.references.any())


def test_a_row_that_is_cut_into_a_shared_page(q):
    """What the documentation says of such a row: forked into an empty one it gets a page of its own, and the others keep their tokens."""
    p = Program(q, 4, 12, 60)
    p.tokens([50, 0, 0, 7])
    p.fork([0, 0, 0, 3])                          # rows 0, 1 and 2 share three pages of 16
    p.tokens([3, 1, 1, 0])
    p.trim([60, 21, 40, 60])                      # rows 1 and 2 end inside of the second and the third
    p.trim([60, 60, 60, 0])
    p.fork([0, 1, 2, 1])
    p.trim([60, 0, 60, 60])
    p.fork([0, 2, 2, 3])
    p.trim([60, 60, 0, 60])
    p.check_pages()
    for _ in range(2):
        p.tokens([2, 13, 20, 9])                  # (the older tokens of all rows are compared here)
        p.check_pages()


def test_a_captured_decode_step(q):
    """Reserve, append and attend of one step in a graph, replayed over changing tables."""
    p = Program(q, 4, 12, 60)
    p.tokens([37, 1, 90, 15])
    new, slots, positions = _i32([1, 1, 1, 1]), *(torch.zeros(4, dtype=torch.int64, device="cuda") for _ in range(2))
    qkv = torch.zeros((4, KV * GROUP + 2 * KV, DIM), device="cuda", dtype=torch.float16)
    qq, k, v = qkv[:, :KV * GROUP], qkv[:, KV * GROUP:-KV], qkv[:, -KV:]
    turned, outs = torch.zeros_like(qq), [torch.zeros((4, KV * GROUP, DIM), device="cuda", dtype=torch.float16) for _ in p.caches]
    calls = [P.PagedReserve(p.tables, new, slots, positions=positions)]
    for cache, out in zip(p.caches, outs):
        calls += [P.PagedAppend(cache, k, v, slots, queries=qq, queriesOut=turned, cos=p.cos, sin=p.sin, positions=positions),
                  P.PagedAttention(cache, turned, p.tables.blockTables, p.tables.lengths, out)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for c in calls:
            c.enqueue()
    lengths = p.tables.lengths.cpu().tolist()
    for step in range(5):
        n = [1, 1, 0, 1] if step == 2 else [1, 1, 1, 1]
        new.copy_(_i32(n))
        qkv.copy_(torch.randn_like(qkv))
        graph.replay()
        torch.cuda.synchronize()
        lengths = [a + b for a, b in zip(lengths, n)]
        assert p.tables.lengths.cpu().tolist() == lengths
        rows = [b for b in range(4) if n[b]]
        for cache, out in zip(p.caches, outs):
            held = starts(lengths)
            keys, values = (torch.zeros((held[-1], KV, DIM), device="cuda") for _ in range(2))
            cache.enqueueDecode(p.tables.blockTables, _i32(held), keysOut=keys, valuesOut=values)
            torch.cuda.synchronize()
            for i, b in enumerate(rows):
                kk, vv = (t[held[b]:held[b + 1]].double().repeat_interleave(GROUP, 1) for t in (keys, values))
                z = (kk * turned[i].double()).sum(-1) / math.sqrt(DIM)
                want = (torch.softmax(z, 0)[..., None] * vv).sum(0)
                if rows == list(range(4)):     # (a row without a new token leaves a gap in the packed batch)
                    assert float((out[b].double() - want).norm() / want.norm()) < 1e-3
        if step == 3:
            p.tables.enqueueFork(_i32([1, 1, 2, 2]))
            lengths = [lengths[1], lengths[1], lengths[2], lengths[2]]
