"""Verification of drafted tokens on the GPU against the oracle. What comes out are
whole numbers, decided in 64 bits on both sides: a random number lies within rounding
(2^-45 or so) of a border with a chance of 10^-9 a case, so all have to be equal."""

from __future__ import annotations

import math
import random

import numpy as np
import pytest
import torch

import morphottention_amd as ma
from oracle import loop_oracle

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _bits(parents):
    rows = []
    for i, p in enumerate(parents):
        rows.append((rows[p] if p >= 0 else 0) | 1 << i)
    return [r - 2 ** 64 if r >> 63 else r for r in rows]


class Drafts:
    def __init__(self, B, n, V, dtype=torch.float16, *, tree=False, drawn=True, ragged=False, temperature=1.0, seed=0, near=0.5):
        g = torch.Generator().manual_seed(seed)
        rng = random.Random(seed)
        self.temperature = temperature
        base = torch.randn((B, n, V), generator=g) * 2
        self.logits = (base + near * torch.randn((B, n, V), generator=g)).to(dtype)
        draft = (base + near * torch.randn((B, n, V), generator=g)).to(dtype)
        self.draft = draft[:, : n - 1].contiguous() if drawn and n > 1 else None
        self.parents = [[-1] + [rng.randint(max(0, i - 4), i - 1) if tree else i - 1 for i in range(1, n)] for _ in range(B)]
        self.tree = torch.tensor([_bits(p) for p in self.parents], dtype=torch.int64) if tree else None
        self.tokens = torch.randint(0, V, (B, n), generator=g)
        for b in range(B):
            for i in range(1, n):
                q = torch.softmax(draft[b, self.parents[b][i]].float() / (temperature or 1.0), -1)
                self.tokens[b, i] = torch.multinomial(q, 1, generator=g) if drawn else q.argsort(descending=True)[min(i % 3, V - 1)]
        self.uniform = torch.rand((B, n), generator=g)
        self.news = torch.tensor([rng.randint(0, n) for _ in range(B)], dtype=torch.int32) if ragged else None

    def run(self):
        on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
        return ma.morpho_verify_drafts(on(self.logits), on(self.tokens), on(self.uniform), tree=on(self.tree),
                                       new_lens=on(self.news), draft_logits=on(self.draft), temperature=self.temperature)

    def want(self):
        B, n = self.tokens.shape
        out = []
        for b in range(B):
            out.append(loop_oracle.verify(self.logits[b].double().numpy(), self.tokens[b].tolist(),
                                          self.uniform[b].double().tolist(),
                                          tree=None if self.tree is None else self.tree[b].tolist(),
                                          count=None if self.news is None else int(self.news[b]),
                                          draft_logits=None if self.draft is None else self.draft[b].double().numpy(),
                                          temperature=self.temperature))
        keep = [path + [-1] * (n - len(path)) for path, _ in out]
        return keep, [len(path) for path, _ in out], [token for _, token in out]

    def check(self):
        keep, keep_lens, token = self.run()
        assert keep.dtype == keep_lens.dtype == torch.int32 and token.dtype == torch.int64
        want = self.want()
        assert (keep.tolist(), keep_lens.tolist(), token.tolist()) == want
        return want


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [1, 2, 7, 100, 2047, 2050, 8192, 8193, 30011])
@pytest.mark.parametrize("n", [1, 2, 6])
def test_chains(dtype, V, n):
    Drafts(5, n, V, TYPES[dtype], ragged=n > 2, seed=V + n).check()
    Drafts(3, n, V, TYPES[dtype], drawn=False, temperature=0.7, seed=V + n).check()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [3, 1000, 12345])
@pytest.mark.parametrize("n", [3, 17, 64])
@pytest.mark.parametrize("drawn", [False, True])
def test_trees(dtype, V, n, drawn):
    if V * n > 500000 and dtype == "f16":
        return
    kept = Drafts(4, n, V, TYPES[dtype], tree=True, drawn=drawn, ragged=True, temperature=1.3, seed=V + n).check()[1]
    assert max(kept) >= 1


@pytest.mark.parametrize("near", [0.0, 0.01, 3.0])
@pytest.mark.parametrize("temperature", [1e-4, 0.05, 1.0, 50.0])
def test_drafters_near_and_far(near, temperature):
    """The same distribution (nothing is turned down), nearly, and quite another one (deep in the tree of siblings)."""
    d = Drafts(16, 24, 5000, torch.float32, tree=True, temperature=temperature, near=near, seed=7)
    kept = d.check()[1]
    if near == 0.0:
        # every token of which a draft exists is followed to a leaf
        for path, b in zip(d.want()[0], range(16)):
            assert path[kept[b] - 1] not in d.parents[b]


def test_many_siblings_are_all_turned_down():
    """All drafts behind the root, none likely: as many remainders as drafts."""
    n, V = 40, 9001
    d = Drafts(6, n, V, torch.bfloat16, tree=True, seed=3, near=0.0)
    d.parents = [[-1] + [0] * (n - 1)] * 6
    d.tree = torch.tensor([_bits(p) for p in d.parents], dtype=torch.int64)
    g = torch.Generator().manual_seed(5)
    d.draft = torch.randn((6, n - 1, V), generator=g).to(torch.bfloat16)
    d.tokens = d.logits[:, 0].float().argsort(-1)[:, :n].contiguous()  # the target's least likely ones
    d.uniform = 0.9 + 0.0999 * d.uniform
    assert d.check()[1] == [1] * 6


@pytest.mark.parametrize("V", [3000, 50001])
@pytest.mark.parametrize("rest", [1, 3])
def test_a_late_sibling_is_kept_and_those_behind_it_turned_down(V, rest):
    """The root's first drafts are turned down one after another, more than the chip has
    summed remainders for, a later one is kept, and behind it drafts are turned down
    again: the remainders of both tokens pass through the same shared memory."""
    B, last = 16, 8
    n = 1 + last + 6 + rest
    d = Drafts(B, n, V, torch.float32, tree=True, seed=V + rest)
    g = torch.Generator().manual_seed(V)
    kept = [last + b % 6 for b in range(B)]  # the eighth draft of the root or a later one
    d.parents = [[-1] + [0] * (last + 6) + [k] * rest for k in kept]
    d.tree = torch.tensor([_bits(p) for p in d.parents], dtype=torch.int64)
    d.draft = torch.randn((B, n - 1, V), generator=g)
    d.logits = torch.randn((B, n, V), generator=g)
    order = d.logits.argsort(-1)
    for b, k in enumerate(kept):
        d.uniform[b, 1:] = 0.999
        d.tokens[b] = order[b, 0, :n]  # the target's least likely ones
        d.tokens[b, last + 7:] = order[b, k, :rest]
        d.tokens[b, k] = 7 + b  # likely in the target, hardly drawn: what is left of it outlasts the drafts before
        d.logits[b, 0, 7 + b], d.draft[b, 0, 7 + b], d.uniform[b, k] = 9.0, -9.0, 0.0
    for _ in range(3):
        assert d.check()[0] == [[0, k] + [-1] * (n - 2) for k in kept]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n", [1, 5, 33])
def test_the_best_token_decides(dtype, n):
    d = Drafts(6, n, 4099, TYPES[dtype], tree=n > 5, drawn=False, ragged=n > 1, temperature=0.0, seed=n)
    for b in range(6):  # paths that are the target's own, as far as a few tokens
        for i in range(1, n):
            if i % 4:
                d.tokens[b, i] = d.logits[b, d.parents[b][i]].float().argmax()
    d.check()
    d.logits[:, :, 77] = d.logits[:, :, 4000] = 99.0  # of equal ones the lowest
    assert set(d.check()[2]) <= {77, -1}
    d.logits[:] = 0.5
    assert set(d.check()[2]) <= {0, -1}


def test_logits_that_are_not_finite():
    for temperature in (1.0, 0.0):
        for drawn in (True, False):
            d = Drafts(8, 4, 3000, torch.float32, drawn=drawn, temperature=temperature, seed=1)
            d.logits[0, :, ::2] = -math.inf  # a mask
            d.logits[1, :, 1::3] = math.nan
            d.logits[2, :, 2:] = torch.finfo(torch.float32).min
            d.logits[3, 1, 5] = d.logits[3, 1, 2999] = math.inf
            d.logits[3, 0, 5] = math.inf
            d.logits[4] = -math.inf  # nothing to draw from
            d.logits[5, 1:] = math.nan
            d.logits[6, :, 1:] = -math.inf  # one token only
            if drawn:
                d.draft[0, :, 1::2] = -math.inf
                d.draft[7] = -math.inf  # as if they were drawn from nothing: kept where the target has them
                d.draft[6, 0, 9] = math.inf
            want = d.check()
            assert want[2][4] == -1 and want[2][6] in (0,)


@pytest.mark.parametrize("temperature", [0.3, 0.7, 1.1, 8.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_nan_has_no_chance(dtype, temperature):
    for drawn in (True, False):
        d = Drafts(6, 5, 3000, TYPES[dtype], drawn=drawn, temperature=temperature, seed=4)
        d.logits[0, :, ::2] = math.nan
        d.logits[1, 0, d.tokens[1, 1]] = math.nan  # of a draft
        d.logits[2, :, 100:] = math.nan
        if drawn:
            d.draft[3, 0, d.tokens[3, 1]] = math.nan
            d.draft[4, :, 1::2] = math.nan
            d.draft[5] = math.nan
        want = d.check()
        assert want[0][1][1] == -1 and 0 <= want[2][2] < 100


def test_numbers_and_tokens_at_their_ends():
    d = Drafts(6, 3, 500, torch.float16, seed=2)
    d.uniform[0] = 0.0
    d.uniform[1] = 1.0 - 2.0 ** -24
    d.tokens[2, 1] = 500  # no such token: turned down
    d.tokens[3, 1] = -1
    d.tokens[4, 1] = 2 ** 40
    d.logits[5] = d.logits[5, :1]
    d.tokens[5] = d.logits[5, 0].float().argmax()
    d.check()
    d.draft = None
    d.check()
    d.temperature = 0.0
    d.check()


def test_the_same_draft_twice():
    """Two drafts of one place that are the same token: the second is turned down where the first was."""
    d = Drafts(32, 4, 20, torch.float32, tree=True, drawn=False, seed=4)
    d.parents = [[-1, 0, 0, 0]] * 32
    d.tree = torch.tensor([_bits(p) for p in d.parents], dtype=torch.int64)
    d.tokens[:, 2] = d.tokens[:, 1]
    d.check()


def test_trees_of_any_bits():
    """A token without a bit below its own is never reached; its own bit and those above it do not count."""
    d = Drafts(4, 6, 50, torch.float32, tree=True, drawn=False, temperature=0.0, seed=4)
    d.tree = torch.tensor([[0] * 6, [2 ** 63 - 1] * 6, [-1] * 6, [1, 2, 1, 4, 5, 6]], dtype=torch.int64)
    d.check()
    d.temperature = 1.0
    d.check()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_of_any_strides(dtype):
    """Rows of a wider tensor, of odd places in memory, in another order, and the same row for all."""
    d = Drafts(3, 4, 1001, TYPES[dtype], seed=6)
    want = d.want()
    tokens, uniform = d.tokens.to(DEV), d.uniform.to(DEV)
    for shift in range(8):
        wide = torch.full((3, 5, 1001 + 24), math.nan, dtype=d.logits.dtype, device=DEV)
        wide[:, 1:, shift: shift + 1001] = d.logits.to(DEV)
        q = torch.full((3, 3, 1003 + shift), math.nan, dtype=d.logits.dtype, device=DEV).transpose(0, 1)
        q = torch.full((3, 3, 1003 + shift), math.nan, dtype=d.logits.dtype, device=DEV)
        q[..., 2: 1003] = d.draft.transpose(0, 1).to(DEV)
        got = ma.morpho_verify_drafts(wide[:, 1:, shift: shift + 1001], tokens, uniform,
                                      draft_logits=q[..., 2: 1003].transpose(0, 1))
        assert tuple(t.tolist() for t in got) == want
    d.logits[:], d.draft[:] = d.logits[:1, :1], d.draft[:1, :1]
    got = ma.morpho_verify_drafts(d.logits[:1, :1].to(DEV).expand(3, 4, 1001), tokens, uniform,
                                  draft_logits=d.draft[:1, :1].to(DEV).expand(3, 3, 1001))
    assert tuple(t.tolist() for t in got) == d.want()


def test_a_large_vocabulary():
    d = Drafts(2, 3, 1000003, torch.bfloat16, seed=8)
    d.check()
    d.temperature = 0.0
    d.check()


def test_strides_beyond_32_bits():
    d = Drafts(3, 3, 700, torch.float16, seed=9)
    want = d.check()
    far = 2 ** 30 + 3
    logits = torch.empty(2 * far + 3 * 700, dtype=torch.float16, device=DEV).as_strided((3, 3, 700), (far, 700, 1))
    draft = torch.empty(far + 3 * 700, dtype=torch.float16, device=DEV).as_strided((3, 2, 700), (700, far, 1))
    logits.copy_(d.logits)
    draft.copy_(d.draft)
    got = ma.morpho_verify_drafts(logits, d.tokens.to(DEV), d.uniform.to(DEV), draft_logits=draft)
    assert tuple(t.tolist() for t in got) == want


def test_two_graphs_in_turn():
    """Two captured calls, replayed in turn: each has its own chunks and masses."""
    ds = [Drafts(4, 6, 5000, torch.bfloat16, seed=1), Drafts(4, 20, 5000, torch.float32, tree=True, seed=2)]
    want = [d.want() for d in ds]
    inputs = [[t if t is None else t.to(DEV) for t in (d.logits, d.tokens, d.uniform, d.tree, d.draft)] for d in ds]
    call = lambda x: ma.morpho_verify_drafts(*x[:3], tree=x[3], draft_logits=x[4])  # noqa: E731
    for x in inputs:
        call(x)
    torch.cuda.synchronize()
    graphs, got = [], []
    for x in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(call(x))
        graphs.append(g)
    for _ in range(3):
        for out in got:
            for t in out:
                t.zero_()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert [tuple(t.tolist() for t in out) for out in got] == want


def test_a_captured_call_follows_its_inputs():
    for kw in ({"tree": True}, {"drawn": False}, {"temperature": 0.0}):
        ds = [Drafts(4, 6, 9000, torch.float16, ragged=True, seed=s, **kw) for s in range(3)]
        on = lambda t: None if t is None else t.to(DEV)  # noqa: E731
        names = ("logits", "tokens", "uniform", "tree", "news", "draft")
        t = {k: on(getattr(ds[0], k)) for k in names}
        call = lambda: ma.morpho_verify_drafts(t["logits"], t["tokens"], t["uniform"], tree=t["tree"],  # noqa: E731
                                               new_lens=t["news"], draft_logits=t["draft"], temperature=ds[0].temperature)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            static = call()
        for d in ds + ds[:2]:
            for k in names:
                if t[k] is not None:
                    t[k].copy_(getattr(d, k))
            graph.replay()
            torch.cuda.synchronize()
            assert tuple(x.tolist() for x in static) == d.want()
            assert tuple(x.tolist() for x in call()) == d.want()


def test_verified_tokens_have_the_targets_distribution():
    """65536 sequences of one step: the first token behind the root, within 5 sigma of the target's chances."""
    B, V, n = 65536, 6, 4
    g = torch.Generator(device=DEV).manual_seed(3)
    logits = torch.randn((1, n, V), generator=g, device=DEV)
    draft = torch.randn((1, n - 1, V), generator=g, device=DEV)
    parents = [-1, 0, 0, 1]
    tokens = torch.zeros((B, n), dtype=torch.int64, device=DEV)
    for i in range(1, n):
        q = torch.softmax(draft[0, parents[i]], -1)
        tokens[:, i] = torch.multinomial(q, B, replacement=True, generator=g)
    tree = torch.tensor(_bits(parents), dtype=torch.int64, device=DEV).expand(B, n).contiguous()
    keep, keep_lens, token = ma.morpho_verify_drafts(logits.expand(B, n, V), tokens, torch.rand((B, n), generator=g, device=DEV),
                                                     tree=tree, draft_logits=draft.expand(B, n - 1, V))
    first = torch.where(keep_lens > 1, tokens.gather(1, keep[:, 1:2].long().clamp(min=0))[:, 0], token)
    p = loop_oracle.distribution(logits[0, 0].double().cpu().numpy(), 1.0)
    seen = torch.bincount(first, minlength=V).double().cpu().numpy()
    assert (np.abs(seen - B * p) <= 5 * np.sqrt(B * p * (1 - p))).all()


def test_refused_tensors():
    d = Drafts(2, 3, 40, torch.float16, tree=True, ragged=True, seed=1)
    on = {k: getattr(d, k).to(DEV) for k in ("logits", "tokens", "uniform", "tree", "news", "draft")}

    def call(**kw):
        t = on | kw
        return ma.morpho_verify_drafts(t["logits"], t["tokens"], t["uniform"], tree=t["tree"], new_lens=t["news"],
                                       draft_logits=t["draft"], temperature=kw.get("temperature", 1.0))
    call()
    for k, bad in (("logits", on["logits"].double()), ("logits", on["logits"][0]), ("logits", on["logits"].cpu()),
                   ("logits", on["logits"].transpose(1, 2).contiguous().transpose(1, 2)), ("tokens", on["tokens"].int()),
                   ("tokens", on["tokens"][:, :2]), ("tokens", on["tokens"].cpu()), ("uniform", on["uniform"].double()),
                   ("uniform", on["uniform"].t().contiguous().t()), ("tree", on["tree"].int()), ("tree", on["tree"][:1]),
                   ("news", on["news"].long()), ("news", on["news"][:1]), ("draft", on["draft"].float()),
                   ("draft", on["draft"][:, :1]), ("draft", on["draft"].cpu()), ("draft", on["draft"][..., :39]),
                   ("temperature", -1.0), ("temperature", 1e9), ("temperature", math.nan)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call(**{k: bad})
    wide = torch.zeros((1, 65, 4), device=DEV)
    with pytest.raises(RuntimeError, match="64 drafted"):
        ma.morpho_verify_drafts(wide, torch.zeros((1, 65), dtype=torch.int64, device=DEV), torch.zeros((1, 65), device=DEV))


def test_another_stream_and_gradients():
    d = Drafts(4, 5, 3000, seed=9)
    want = d.want()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = d.run()
    side.synchronize()
    assert tuple(t.tolist() for t in got) == want
    logits = d.logits.float().to(DEV).requires_grad_(True)  # whole numbers have no gradients
    got = ma.morpho_verify_drafts(logits, d.tokens.to(DEV), d.uniform.to(DEV), draft_logits=d.draft.float().to(DEV))
    assert tuple(t.tolist() for t in got) == want and not got[2].requires_grad


@pytest.mark.parametrize("drawn", [False, True])
def test_a_large_tree_of_16_bit_logits(drawn):
    kept = Drafts(4, 64, 12345, torch.float16, tree=True, drawn=drawn, ragged=True, temperature=1.3, seed=12409).check()[1]
    assert max(kept) >= 1
