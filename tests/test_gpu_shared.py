"""Attention over the cache where sequences have their first pages in common, on the
GPU against its definition in 64 bits: the one and the tolerances of test_gpu_cache
(joining one more piece of a row adds a rounding of 2^-24 to its sums, which the
2^-20 there holds many times over)."""

from __future__ import annotations

import math

import pytest
import torch

import morphottention_amd as ma
from test_gpu_cache import DEV, FLT_MAX, Problem, _check

pytestmark = pytest.mark.gpu


class Shared(Problem):
    """groups: lists of sequences; common: the pages that each has in common. What the
    rows of the table would have had instead is NaN in the pool."""

    def __init__(self, B, n, H, m, dv, lens, groups, common, **kw):
        super().__init__(B, n, H, m, dv, lens, **kw)
        self.groups, self.common = groups, common
        for mine, pages in zip(groups, common):
            first = mine[0]
            for b in mine[1:]:
                t = min(pages * self.P, lens[b], lens[first])
                self.table[b, : t // self.P] = self.table[first, : t // self.P]
                self.k[b][:t] = self.k[first][:t]
                self.v[b][:t] = self.v[first][:t]
        self.codes.fill_(math.nan)
        self.values.fill_(math.nan)
        for b in range(B):
            self.store(b)

    def shared(self, **kw):
        return ma.SharedPrefix.of(self.groups, self.common, self.B, device=DEV, **kw)

    def device(self):
        """With a table so wide that sharing is worth it as far as the host knows (64 MB
        less to read): otherwise the sequences are computed apart."""
        d = super().device()
        spared = max(1, sum(map(len, self.groups)) - len(self.groups)) * self.P * self.H * (self.m + self.dv) * 2
        wide = torch.full((self.B, -(-(64 << 20) // spared)), -1, dtype=torch.int32, device=DEV)
        wide[:, : self.table.shape[1]] = d["table"]
        d["table"] = wide
        return d


def _case(n, H=2, m=16, dv=64, P=64, news=None, seed=0, **kw):
    """Two groups of different prefixes that stand apart in the batch, and one sequence of neither."""
    lens = [5 * P + 3, 2 * P, 5 * P, 70, 2 * P + 31, 5 * P + 64]
    return Shared(6, n, H, m, dv, lens, [[5, 0, 2], [1, 4]], [5, 2], P=P, news=news, seed=seed, **kw)


@pytest.mark.parametrize("m", [16, 32, 64])
@pytest.mark.parametrize("dv", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 7, 20, 64])
def test_shapes(m, dv, n):
    p = _case(n, 3, m, dv, news=[n, max(1, n - 3), 0, n, n, n // 2], seed=m + dv + n)
    _check(p.attend(p.device(), shared=p.shared(max_rest=128 + n)), p.reference())


@pytest.mark.parametrize("P", [32, 64, 128, 256])
@pytest.mark.parametrize("n", [1, 3, 33])
def test_page_sizes(P, n):
    p = _case(n, 2, 32, 32, P=P, seed=P)
    _check(p.attend(p.device(), shared=p.shared()), p.reference())


@pytest.mark.parametrize("n", [2, 16, 17, 64])
@pytest.mark.parametrize("mask,mask_diag", [("causal", False), ("causal", True), ("full", False), ("full", True)])
def test_masks(n, mask, mask_diag):
    p = _case(n, 2, 32, 64, P=32, news=[n, n // 2, 1, 0, n, n], seed=n)
    _check(p.attend(p.device(), causal=mask == "causal", mask_diag=mask_diag, shared=p.shared()),
           p.reference(mask, mask_diag))


@pytest.mark.parametrize("n", [1, 13, 64])
def test_trees(n):
    g = torch.Generator().manual_seed(n)
    p = _case(n, 2, 16, 64, news=[n, max(0, n - 2), n, n, 1, n], seed=n)
    tree = torch.zeros((6, n), dtype=torch.int64)
    for b in range(6):
        for k in range(n):
            parent = int(torch.randint(-1, max(k, 1), (1,), generator=g)) if k else -1
            bits = (int(tree[b, parent]) if parent >= 0 else 0) & (2 ** 64 - 1) | 1 << k
            tree[b, k] = bits - 2 ** 64 if bits >> 63 else bits
    tree[0, n // 2] = 0  # sees no draft, its prefix all the same
    _check(p.attend(p.device(), tree=tree.to(DEV), shared=p.shared()), p.reference(tree=tree))


@pytest.mark.parametrize("B,H,n,L,m,dv", [(3, 1, 1, 4096, 16, 64), (2, 2, 3, 2944, 32, 32), (4, 1, 20, 1536, 64, 128),
                                          (2, 2, 64, 1024, 16, 64), (40, 2, 1, 1088, 32, 64)])
def test_divided_prefixes(B, H, n, L, m, dv):
    """Prefixes of many pieces; the hints may be short or long without changing the result
    (the last two: apart, and as long as the table)."""
    p = Shared(B, n, H, m, dv, [L + 7 * b for b in range(B)], [list(range(B))], [L // 64], seed=L)
    d, want = p.device(), p.reference()
    wide = d["table"].shape[1] * 64
    for hints in ({}, {"max_prefix": wide, "max_rest": 7 * B + n}, {"max_prefix": wide - 64, "max_rest": 1},
                  {"max_prefix": L, "max_rest": 7 * B + n}, {"max_prefix": 2 * wide, "max_rest": 2 * wide}):
        _check(p.attend(d, shared=p.shared(**hints)), want)


@pytest.mark.parametrize("n", [1, 40])
def test_groups_of_any_kind(n):
    """Of one sequence, of no common page, and one whose pages a member has not reached:
    that one has its keys to itself. Rows of many sequences fill several blocks."""
    lens = [130, 200, 64, 320, 330, 340] + [64 + b for b in range(30)]
    p = Shared(36, n, 1, 16, 32, lens, [[0], [1, 2], [3, 4, 5], list(range(6, 36))], [2, 3, 0, 1], seed=3)
    _check(p.attend(p.device(), shared=p.shared()), p.reference())


def test_a_tensor_of_groups_may_say_anything():
    """Groups and members that do not exist have no effect, and no fault."""
    p = _case(2, 1, 16, 32, seed=1)
    d, want = p.device(), p.reference()
    i = lambda *v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    big = 2 ** 31 - 1
    # no sequence's group is one of them
    for group in (i(-1, 7, big, -big, 3, 2),):
        _check(p.attend(d, shared=ma.SharedPrefix(i(0, 1, 2, 3), i(0, 2, 4), group, i(5, 2))), want)
    # groups whose pages no sequence reaches, or fewer than none
    for pages in (i(big, 9), i(-3, -big)):
        _check(p.attend(d, shared=ma.SharedPrefix(i(5, 0, 2, 1, 4), i(0, 3, 5), i(0, 1, 0, -1, 1, 0), pages)), want)
    # members and starts out of range: memory is safe, rows of no group are right
    out, lse = p.attend(d, shared=ma.SharedPrefix(i(9, -4, big, 0, 3), i(-7, big, 2), i(0, 1, 0, -1, 1, 0), i(5, 2)))
    ref = want[0][3]
    assert ((out[3].double().cpu() - ref).abs() <= want[2][3]).all()


@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("P", [32, 64])
def test_pages_that_the_pool_does_not_have(n, P):
    """Their keys are left out for all of the group."""
    lens = [300, 7 * P + 5]
    p = Shared(2, n, 2, 32, 64, lens, [[0, 1]], [3], P=P, seed=5)
    gone = [0, 2]
    for b in range(2):
        p.table[b, 0], p.table[b, 2] = -1, p.codes.shape[0] + 7
    drop = lambda b: [t for t in range(lens[b] + n) if t // P in gone]  # noqa: E731
    _check(p.attend(p.device(), shared=p.shared()), p.reference(drop=drop))


@pytest.mark.parametrize("n", [1, 5, 40])
def test_what_is_not_finite_in_the_prefix(n):
    """An infinite or NaN value of a common key decides its column in every row of the
    group, and in no other."""
    p = _case(n, 2, 16, 64, seed=9)
    for b in p.groups[0]:
        p.v[b][17, 0, 3] = math.inf
        p.v[b][40, 1, 7] = math.nan
        p.v[b][200, 1, 9] = -math.inf
    p.store(p.groups[0][0])
    out = p.attend(p.device(), shared=p.shared())[0].float().cpu().view(6, n, 2, 64)
    bad = torch.zeros_like(out, dtype=torch.bool)
    for b in p.groups[0]:
        bad[b, :, 0, 3] = bad[b, :, 1, 7] = bad[b, :, 1, 9] = True
        assert (out[b, :, 0, 3] == math.inf).all() and out[b, :, 1, 7].isnan().all() and (out[b, :, 1, 9] == -math.inf).all()
    assert torch.equal(~out.isfinite(), bad)


@pytest.mark.parametrize("n", [1, 20])
def test_scores_that_the_prefix_outweighs(n):
    """Large scores: the pieces' references differ by more than the weights' range."""
    p = _case(n, 2, 32, 64, seed=2, scale=40.0)
    _check(p.attend(p.device(), shared=p.shared()), p.reference())


def test_beyond_64_new_tokens_it_is_the_attention_without():
    p = _case(70, 2, 16, 64, seed=4)
    d = p.device()
    for a, b in zip(p.attend(d, shared=p.shared()), p.attend(d)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("n", [1, 20])
def test_a_pool_beyond_32_bits(n):
    """Pages more than 2^32 bytes into a pool: the same results as near its start."""
    far = 34000  # of 128 KiB of values
    p = Shared(3, n, 16, 16, 64, [300, 256, 270], [[0, 1, 2]], [4], seed=3)
    d, shared = p.device(), p.shared()
    want = [t.clone() for t in p.attend(d, shared=shared)]
    for k in ("codes", "values"):
        small, d[k] = d[k], torch.empty((far + d[k].shape[0], *d[k].shape[1:]), dtype=torch.float16, device=DEV)
        d[k][far:] = small
    assert d["values"].numel() * 2 > 2 ** 32
    d["table"] = torch.where(d["table"] >= 0, d["table"] + far, -1)
    for a, b in zip(p.attend(d, shared=shared), want):
        assert torch.equal(a, b)


def test_two_graphs_in_turn():
    """Two captured calls with partial results, replayed in turn: each has its own."""
    ps = [_case(n, seed=n) for n in (1, 30)]
    ds, sharings = [p.device() for p in ps], [p.shared() for p in ps]
    want = [[t.clone() for t in p.attend(d, shared=s)] for p, d, s in zip(ps, ds, sharings)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for p, d, s in zip(ps, ds, sharings):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(p.attend(d, shared=s))
        graphs.append(g)
    for _ in range(3):
        for out, lse in got:
            out.zero_()
            lse.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_repeats_bit_for_bit_and_on_another_stream():
    p = Shared(8, 3, 4, 32, 64, [1024 + b for b in range(8)], [list(range(8))], [16], seed=6)
    d, shared = p.device(), p.shared()
    first = p.attend(d, shared=shared)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [p.attend(d, shared=shared) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for out, lse in got:
        assert torch.equal(out, first[0]) and torch.equal(lse, first[1])


def test_a_captured_call_follows_groups_and_lengths():
    p = _case(2, 2, 16, 32, seed=8)
    q = Shared(6, 2, 2, 16, 32, [130, 70, 129, 200, 128, 3], [[0, 2, 4]], [2], seed=8)
    d, sp = p.device(), p.shared()
    dq, sq = q.device(), q.shared()
    wide = torch.full_like(d["table"], -1)
    call = lambda: p.attend(d, shared=sp)  # noqa: E731
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        static = call()
    before = {k: v.clone() for k, v in d.items() if v is not None}
    groups = {k: getattr(sp, k).clone() for k in ("members", "starts", "group", "pages")}
    pool = max(before["codes"].shape[0], dq["codes"].shape[0])
    assert pool == before["codes"].shape[0]
    for turn in range(4):
        if turn % 2:  # another batch in the same tensors: one group (the other has none), other lengths
            for k in ("codes", "values"):
                d[k][: dq[k].shape[0]] = dq[k]
            wide[:] = -1
            wide[:, : q.table.shape[1]] = dq["table"][:, : q.table.shape[1]]
            d["table"].copy_(wide)
            for k in ("phi", "gq", "gk", "lens"):
                d[k].copy_(dq[k])
            sp.members[:3], sp.starts[:], sp.group[:] = sq.members, torch.tensor([0, 3, 3], device=DEV), sq.group
            sp.pages[:1] = sq.pages
        else:
            for k, v in before.items():
                d[k].copy_(v)
            for k, v in groups.items():
                getattr(sp, k).copy_(v)
        graph.replay()
        torch.cuda.synchronize()
        eager = call()
        assert torch.equal(static[0], eager[0]) and torch.equal(static[1], eager[1])
        _check(static, (q if turn % 2 else p).reference())


def test_refused_tensors():
    p = _case(1, 1, 16, 32)
    d, s = p.device(), p.shared()
    for name in ("members", "starts", "group", "pages"):
        t = getattr(s, name)
        for bad in (t.long(), t.cpu(), torch.stack((t, t), 1)[:, 0], t[None]):
            setattr(s, name, bad)
            with pytest.raises((RuntimeError, NotImplementedError)):
                p.attend(d, shared=s)
        setattr(s, name, t)
    s.group = s.group[:-1]
    with pytest.raises(RuntimeError, match="group must be"):
        p.attend(d, shared=s)
    s = p.shared()
    s.starts = s.starts[:-1]
    with pytest.raises(RuntimeError, match="starts must be"):
        p.attend(d, shared=s)


def test_forks_generate_as_without():
    """A layer on forks of one prompt: each next token with and without sharing."""
    torch.manual_seed(1)
    H, m, dv = 2, 16, 32
    layer = ma.MorphoAttention(H * dv, H, m, causal=True, dtype=torch.float16, device=DEV)
    cache = ma.MorphoCache(60, H, m, dv, page_size=32, device=DEV)
    w = layer.pack_cache_weights()
    a = cache.new()
    with torch.no_grad():
        step = cache.step([a], 200)
        layer.forward_cached(torch.randn(1, 200, H * dv, device=DEV).half(), w, cache, step)
        cache.commit(step)
        seqs = [a] + [cache.fork(a) for _ in range(4)]
        for _ in range(40):
            x = torch.randn(5, 1, H * dv, device=DEV).half()
            step = cache.step(seqs, 1, shared=True)
            assert step.shared.pages.tolist() == [6] and step.shared.members.tolist() == [0, 1, 2, 3, 4]
            y = layer.forward_cached(x, w, cache, step)
            step.shared = None
            z = layer.forward_cached(x, w, cache, step)  # stores the same again
            # fp32 results that differ by 2^-19 or so, rounded to fp16 once
            assert ((y.float() - z.float()).abs() <= 2.0 ** -10 * z.float().abs() + 2.0 ** -18 * z.abs().max()).all()
            cache.commit(step)
    assert (FLT_MAX > 0) and cache.length(seqs[4]) == 240
