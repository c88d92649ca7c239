"""Page tables on the device against the oracle, and a decoding loop of all of its
operators: steps, attention with a common prefix, verification, acceptance."""

from __future__ import annotations

import random

import numpy as np
import pytest
import torch

import morphottention_amd as ma
from oracle import loop_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"


class Account:
    def __init__(self, B, W, n, P, *, longest, spare, seed, ragged=True, odd=False):
        rng = random.Random(seed)
        self.n, self.P = n, P
        self.lens = [rng.randint(0, longest) for _ in range(B)]
        self.held = [min(W, -(-l // P) + rng.choice([0, 0, 1, 3])) for l in self.lens]
        pool = list(range(sum(self.held) + spare))
        rng.shuffle(pool)
        take = iter(pool)
        self.table = np.array([[next(take) for _ in range(h)] + [-1] * (W - h) for h in self.held], dtype=np.int32)
        self.free = list(take)
        self.count = len(self.free)
        self.free += [-7] * sum(self.held)
        self.news = [rng.choice([0, 1, n, rng.randint(0, n)]) for _ in range(B)] if ragged else None
        if odd:  # lengths and counts outside their range
            for k, v in enumerate((-5, 2 ** 31 - 1, W * P, W * P - 1)):
                self.lens[k % B] = v
            self.held[B // 2], self.held[B - 1] = -3, W + 9
            self.news = None if self.news is None else [-4, n + 100] + self.news[2:]

    def device(self):
        i = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        self.d = {"table": i(self.table), "held": i(self.held), "lens": i(self.lens), "free": i(self.free),
                  "count": i([self.count]), "news": None if self.news is None else i(self.news)}
        return self.d

    def run(self):
        d = self.d
        return ma.morpho_cache_plan(d["table"], d["held"], d["lens"], d["free"], d["count"], self.n, new_lens=d["news"],
                                    page_size=self.P)

    def want(self):
        """The oracle's step; its account becomes this one."""
        got = loop_oracle.plan(self.table, self.held, self.lens, self.free, self.count, self.n, self.news, self.P)
        self.table, self.held, self.free, self.count = got[:4]
        return got[4], got[5]

    def check(self, got):
        granted, slots = self.want()
        assert got[0].tolist() == granted and torch.equal(got[1].cpu(), torch.from_numpy(slots))
        d = self.d
        assert torch.equal(d["table"].cpu(), torch.from_numpy(self.table)) and d["held"].tolist() == self.held
        assert d["free"].tolist() == self.free and d["count"].tolist() == [self.count]


@pytest.mark.parametrize("P", [32, 64, 128, 256])
@pytest.mark.parametrize("B,n", [(1, 1), (3, 70), (64, 12), (200, 40), (1024, 8), (1025, 3), (2500, 1), (5, 3000), (700, 300)])
@pytest.mark.parametrize("spare", [0, 40, 100000])
def test_plans(P, B, n, spare):
    a = Account(B, -(-(400 + n) // P) + 2, n, P, longest=400, spare=spare, seed=B + n + P, ragged=B != 200)
    a.device()
    a.check(a.run())
    # what was kept of it, and more new tokens
    rng = random.Random(B)
    for _ in range(3):
        a.lens = [l + rng.randint(0, 3) for l in a.lens]
        a.news = [rng.randint(0, n) for _ in a.lens]
        a.d["lens"].copy_(torch.tensor(a.lens))
        a.d["news"] = torch.tensor(a.news, dtype=torch.int32, device=DEV)
        a.check(a.run())


@pytest.mark.parametrize("B,n", [(4, 5), (64, 200), (3000, 2)])
def test_plans_out_of_range(B, n):
    """Lengths below 0 and past the table, counts below 0 and past the row: nothing outside the tensors
    is touched, and the others get what they would."""
    a = Account(B, 9, n, 32, longest=64, spare=50, seed=B, odd=True)
    a.table = np.abs(a.table)
    a.device()
    a.check(a.run())


def test_a_stack_without_room_or_pages():
    for count in (-5, 0, 3, 2 ** 31 - 1):
        a = Account(3, 4, 40, 32, longest=60, spare=0, seed=1)
        a.held, a.lens, a.news = [2, 0, 4], [10, 20, 0], [0, 40, 0]
        a.table = np.arange(12, dtype=np.int32).reshape(3, 4)
        a.free, a.count = [20, 21, 22], count
        a.device()
        a.check(a.run())
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    d = a.d
    granted, _ = ma.morpho_cache_plan(d["table"], torch.zeros_like(d["held"]), d["lens"], none, torch.zeros_like(d["count"]), 4)
    assert granted.tolist() == [0, 0, 0]


def test_given_back_and_taken_again_are_the_same_pages():
    a = Account(40, 12, 100, 32, longest=200, spare=200, seed=2, ragged=False)
    a.held = [-(-l // 32) for l in a.lens]
    a.device()
    d, lens = a.d, torch.tensor(a.lens, dtype=torch.int32, device=DEV)
    first = [t.clone() for t in (*a.run(), d["table"], d["held"], d["free"], d["count"])]
    ma.morpho_cache_plan(d["table"], d["held"], lens, d["free"], d["count"], 100, new_lens=torch.zeros_like(lens), page_size=32)
    again = (*a.run(), d["table"], d["held"], d["free"], d["count"])
    for x, y in zip(first, again):
        assert torch.equal(x, y)


@pytest.mark.parametrize("B,n", [(6, 10), (1100, 20)])
def test_a_captured_plan_goes_on(B, n):
    """Replays take up the account where the last one left it, with eager work between them."""
    a = Account(B, 40, n, 32, longest=100, spare=30 * B, seed=4)
    d = a.device()
    keep = {k: v.clone() for k, v in d.items()}
    step = lambda: (a.run(), d["lens"].add_(3))  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = step()[0]
    for k, v in keep.items():
        d[k].copy_(v)
    for _ in range(6):
        graph.replay()
        torch.cuda.synchronize()
        a.check(static)
        a.lens = [l + 3 for l in a.lens]
        assert torch.ones(1000, device=DEV).sum() == 1000


def test_refused_tensors():
    a = Account(3, 4, 5, 32, longest=60, spare=9, seed=1)
    d = a.device()
    names = ("table", "held", "lens", "free", "count", "news")
    for k in names:
        good = d[k]
        for bad in (good.long(), good.cpu(), good[None], torch.cat((good, good))):
            if k == "free" and bad.dtype == torch.int32 and bad.is_cuda and bad.dim() == 1:
                continue
            if k == "count" and bad.dim() == 2:
                continue
            d[k] = bad
            with pytest.raises((RuntimeError, NotImplementedError)):
                a.run()
        d[k] = good
    for n, P in ((0, 32), (-1, 32), (1 << 23, 32), (5, 48)):
        a.n, a.P = n, P
        with pytest.raises(RuntimeError):
            a.run()


# ---------------------------------------------------------------- all of them together
def _model(seed, layers=2, H=2, m=16, dv=32, V=300):
    torch.manual_seed(seed)
    mods = [ma.MorphoAttention(H * dv, H, m, causal=True, dtype=torch.float16, device=DEV) for _ in range(layers)]
    embed = torch.randn(V, H * dv, device=DEV).half()
    head = (torch.randn(H * dv, V, device=DEV) * 0.3).half()
    return mods, [w.pack_cache_weights() for w in mods], embed, head


def _logits(model, cache, step, tokens, tree):
    mods, weights, embed, head = model
    x = embed[tokens]
    for i, (mod, w) in enumerate(zip(mods, weights)):
        x = x + mod.forward_cached(x, w, cache, step, layer=i, tree=tree)
    return x @ head


def _drafts(root, turn, V, n):
    """Tokens of a step: the decided one, and drafts that follow from it and the turn."""
    i = torch.arange(1, n, device=root.device)
    return torch.cat((root[:, None], (root[:, None] * 7 + i * 31 + turn * 13) % V), 1)


PARENTS = [-1, 0, 0, 1, 1, 3]


def _tree(B):
    rows = []
    for i, p in enumerate(PARENTS):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    return torch.tensor(rows, dtype=torch.int64, device=DEV).expand(B, len(rows)).contiguous()


def _prompt(model, cache, length, V):
    a = cache.new()
    g = torch.Generator(device=DEV).manual_seed(length)
    step = cache.step([a], length)
    out = _logits(model, cache, step, torch.randint(0, V, (1, length), generator=g, device=DEV), None)
    cache.commit(step)
    return a, out[:, -1].float().argmax(-1)


@pytest.mark.parametrize("V,length", [(300, 140), (12, 155)])
@pytest.mark.parametrize("captured", [False, True])
def test_a_loop_of_steps(captured, V, length):
    """Answers to one prompt with drafted trees: the loop on the device, eager or as a
    replayed graph, against single calls with the host's account, token by token."""
    B, n, turns = 5, len(PARENTS), 12
    tree = _tree(B)
    g = torch.Generator(device=DEV).manual_seed(11)
    numbers = torch.rand((turns, B, n), generator=g, device=DEV)
    got = []
    with torch.no_grad():
        for on_device in (False, True):
            model = _model(5, V=V)
            cache = ma.MorphoCache(80, 2, 16, 32, num_layers=2, page_size=32, device=DEV)
            a, root = _prompt(model, cache, length, V)
            seqs = [a] + [cache.fork(a) for _ in range(B - 1)]
            root = root.expand(B).contiguous()
            told = [[] for _ in range(B)]

            def tell(tokens, keep, keep_lens, token):
                for b, (row, k) in enumerate(zip(keep.tolist(), keep_lens.tolist())):
                    told[b] += [int(tokens[b, i]) for i in row[:k]]

            if not on_device:
                for turn in range(turns):
                    tokens = _drafts(root, turn, V, n)
                    step = cache.step(seqs, n, shared=True)
                    out = _logits(model, cache, step, tokens, tree)
                    keep, keep_lens, root = ma.morpho_verify_drafts(out, tokens, numbers[turn], tree=tree)
                    cache.accept(step, (keep, keep_lens))
                    tell(tokens, keep, keep_lens, root)
            else:
                with cache.loop(seqs, n, length + turns * n + n, shared=True) as loop:
                    assert loop.shared.pages.tolist() == [4]
                    u = torch.empty((B, n), device=DEV)
                    turn_at = torch.zeros((), dtype=torch.int64, device=DEV)
                    root = root.clone()

                    def one():
                        tokens = _drafts(root, turn_at, V, n)
                        step = loop.step()
                        out = _logits(model, cache, step, tokens, tree)
                        keep, keep_lens, token = ma.morpho_verify_drafts(out, tokens, u, tree=tree, new_lens=step.new_lens)
                        loop.accept(step, keep, keep_lens)
                        root.copy_(token)
                        return tokens, keep, keep_lens, token

                    run = one
                    if captured:
                        state = [t.clone() for t in (loop.table, loop.held, loop.lens, loop.free_pages, loop.free_count, root)]
                        u.copy_(numbers[0])
                        side = torch.cuda.Stream()
                        side.wait_stream(torch.cuda.current_stream())
                        with torch.cuda.stream(side):
                            one()
                        torch.cuda.current_stream().wait_stream(side)
                        graph = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(graph):
                            static = one()
                        for t, v in zip((loop.table, loop.held, loop.lens, loop.free_pages, loop.free_count, root), state):
                            t.copy_(v)

                        def run():
                            graph.replay()
                            return static
                    for turn in range(turns):
                        u.copy_(numbers[turn])
                        turn_at.fill_(turn)
                        tell(*run())
                        torch.cuda.synchronize()
            assert [cache.length(s) for s in seqs] == [length + len(t) for t in told]
            held = sum(len(cache.pages(s)) for s in seqs) - 4 * (B - 1)  # the four common ones count once
            assert cache.free_pages == 80 - held
            got.append(told)
            for s in seqs:
                cache.free(s)
            assert cache.free_pages == 80
    assert got[0] == got[1] and min(len(t) for t in got[0]) >= turns
    if V == 12:  # of few tokens many drafts are kept
        assert sum(len(t) for t in got[0]) > turns * B + 10


def test_a_loop_that_runs_out_of_pages():
    """The sequences that get none stand still, and go on once there are pages again."""
    model = _model(6)
    cache = ma.MorphoCache(12, 2, 16, 32, num_layers=2, page_size=32, device=DEV)
    seqs = [cache.new() for _ in range(3)]
    tokens = torch.arange(60, device=DEV).view(3, 20)
    with torch.no_grad(), cache.loop(seqs, 20, 400, pages=4) as loop:
        for _ in range(6):
            step = loop.step()
            out = _logits(model, cache, step, tokens, None)
            assert out.isfinite().all()
            loop.accept(step)
    # 20 tokens each, 40 of the first (its second page is the fourth), then nobody lacks less than a page
    assert [cache.length(s) for s in seqs] == [60, 20, 20] and cache.free_pages == 8
