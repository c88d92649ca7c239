"""What the paged cache promises for calls that its documentation allows but that are
easy to get wrong, on the GPU."""

from __future__ import annotations

import math

import pytest
import torch

import morphottention_amd as ma
from test_gpu_cache import Problem, _check

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _ints(rows):
    return torch.tensor(rows, dtype=torch.int32, device=DEV)


# ---------------------------------------------------------------- compaction in place
@pytest.mark.parametrize("dv", [32, 64, 128])
@pytest.mark.parametrize("lead", [1, 3])
@pytest.mark.parametrize("kept", [50, 64, 65, 200, 1500])
def test_entries_below_their_place_move_nothing(dv, lead, kept):
    """Rows that open with negative entries, over several batches of either kernel: an
    entry below its place, negative or not, leaves its place as it was, and the
    others find their tokens where they were before the call."""
    g = torch.Generator().manual_seed(kept)
    H, m, P, base, span = 2, 16, 64, 13, 2 * kept
    per = -(-(base + span) // P)
    # 300 sequences in two layers, so that a workgroup of few tokens takes several heads
    B, L = (300, 2) if kept <= 64 else (2, 1)
    codes = torch.randn((L, B * per, H, P, m), generator=g).half()
    values = torch.randn((L, B * per, H, P // 8, dv, 8), generator=g).half()
    table = torch.randperm(B * per, generator=g).view(B, per)
    # some below their places all along, and rows that jump ahead halfway
    keep = torch.arange(kept).repeat(B, 1) - lead
    keep[1::2, kept // 2:] += lead + 5
    keep[:, :lead] = -1
    dc, dval = codes.to(DEV), values.to(DEV)
    ma.morpho_cache_compact(dc, dval, table.int().to(DEV), _ints([base] * B), keep.int().to(DEV))
    k = torch.arange(kept)
    for b in range(B):
        at = k[keep[b] >= k]
        to, of = base + at, base + keep[b, at]
        pt, ps = table[b, to // P], table[b, of // P]
        new = codes[:, ps, :, of % P].clone(), values[:, ps, :, of % P // 8, :, of % 8].clone()
        codes[:, pt, :, to % P] = new[0]
        values[:, pt, :, to % P // 8, :, to % 8] = new[1]
    assert torch.equal(dc.cpu(), codes) and torch.equal(dval.cpu(), values)


# ---------------------------------------------------------------- values that are not finite

def _attention_case(B, n, H, m, dv, lens, P, seed, gate=1.0):
    g = torch.Generator().manual_seed(seed)
    per = -(-(max(lens) + n) // P)
    pages = B * per + 1
    table = torch.randperm(pages, generator=g)[: B * per].view(B, per)
    codes = torch.rand((pages, H, P, m), generator=g).half()
    values = torch.randn((pages, H, P // 8, dv, 8), generator=g).half()
    phi = torch.rand((B, n, H, m), generator=g).half()
    gq, gk = (torch.full((H, m), gate).half(), torch.ones((H, m)).half())
    return codes, values, table, phi, gq, gk


def _seen(n, L, mask, mask_diag, tree):
    """[n, L + n]: which of the positions a new token sees."""
    seen = torch.ones((n, L + n), dtype=torch.bool)
    if tree is not None:
        seen[:, L:] = (tree[:, None] >> torch.arange(n)) & 1 == 1
    elif mask == "causal":
        seen = torch.tril(seen, L)
    if mask_diag:
        seen[torch.arange(n), L + torch.arange(n)] = False
    return seen


SHAPES = [(1, 2, 16, 64, 700, 64), (1, 2, 32, 128, 5000, 64), (5, 1, 64, 32, 333, 32), (20, 2, 16, 64, 500, 64),
          (50, 1, 64, 64, 3000, 128), (70, 2, 16, 64, 300, 64), (70, 1, 64, 128, 700, 256), (150, 1, 32, 32, 2500, 32),
          (130, 2, 16, 128, 40, 64)]
MASKS = [("causal", False), ("causal", True), ("full", True), ("tree", False)]


@pytest.mark.parametrize("n,H,m,dv,L,P,mask,mask_diag", [(*s, *k) for s in SHAPES for k in MASKS
                                                         if k[0] != "tree" or s[0] <= 64])
@pytest.mark.parametrize("gate", [1.0, 300.0])
def test_values_that_are_not_finite_decide_their_column(n, H, m, dv, L, P, mask, mask_diag, gate):
    """Weights are positive, so an infinite value makes its column infinite in every
    row that sees it, however small its weight is (gate 300: most vanish) and
    wherever in a tile, piece or page it lies; both infinities, or a NaN, make it
    NaN. Every other place is, bit for bit, what it is with 0 in those places."""
    lens = [L, L // 3 + 1]
    codes, values, table, phi, gq, gk = _attention_case(2, n, H, m, dv, lens, P, n + L, gate)
    g = torch.Generator().manual_seed(n)
    tree = None
    if mask == "tree":
        bits = [[1 << k | (1 << k // 2 if k else 0) for k in range(n)] for _ in range(2)]
        tree = torch.tensor([[x - 2 ** 64 if x >> 63 else x for x in row] for row in bits], dtype=torch.int64)
    # per sequence and head: (position, column, value); column 1 gets both infinities, 2 a NaN
    strange = [[[(int(torch.randint(0, lens[b] + n, (1,), generator=g)), c, v)
                 for c, v in ((0, "inf"), (1, "inf"), (1, "-inf"), (2, "nan"), (2, "inf"), (5, "-inf"), (dv - 1, "inf"),
                              (dv // 2, "-inf"), (dv // 2, "-inf"))] +
                [(0, 7, "inf"), (lens[b] + n - 1, 8, "-inf"), (31, 9, "inf"), (32, 10, "-inf"), (lens[b], 11, "inf")]
                for _ in range(H)] for b in range(2)]
    clean, sums = values.clone(), torch.zeros((2, n, H, dv))
    for b in range(2):
        seen = _seen(n, lens[b], mask, mask_diag, None if tree is None else tree[b])
        for h in range(H):
            for t, c, v in strange[b][h]:
                page, s = int(table[b, t // P]), t % P
                values[page, h, s // 8, c, s % 8] = float(v)
                clean[page, h, s // 8, c, s % 8] = 0
            # one value a place: the last that was written
            for (t, c), v in {(t, c): v for t, c, v in strange[b][h]}.items():
                sums[b, seen[:, t], h, c] += float(v)
    args = [t.to(DEV) for t in (phi, gq, gk, codes)]
    rest = dict(scale=m ** -0.5, causal=mask != "full", mask_diag=mask_diag,
                tree=None if tree is None else tree.to(DEV))
    got, want = (ma.morpho_cache_attention(*args, v.to(DEV), table.int().to(DEV), _ints(lens), **rest)
                 for v in (values, clean))
    out, ref = (t[0].cpu().view(2, n, H, dv) for t in (got, want))
    assert torch.equal(got[1], want[1])  # the sums of weights know nothing of values
    assert ref.isfinite().all()
    expect = torch.where(sums == 0, ref, sums.half())
    same = (out == expect) | (out.isnan() & expect.isnan())
    assert same.all(), (~same).nonzero()[:8].tolist()
    assert (sums == math.inf).any() and (sums == -math.inf).any() and sums.isnan().any() and (sums == 0).any()


@pytest.mark.parametrize("n", [1, 40, 70, 200])
@pytest.mark.parametrize("alike", [False, True])
def test_the_largest_value_stays_finite(n, alike):
    """The mean of values that are all the largest number is that number: weights
    rounded to 16 bits must not lift it past the range. With keys that are all
    alike but one, the weights of a row are rounded alike, up in many rows."""
    codes, values, table, phi, gq, gk = _attention_case(1, n, 2, 16, 64, [600], 64, n)
    if alike:
        codes[:] = codes[0, 0, 0]
        codes[table[0, 0], :, 0] = torch.rand(16, generator=torch.Generator().manual_seed(2)).half()
    values[..., ::2, :], values[..., 1::2, :] = 65504.0, -65504.0
    out, _ = ma.morpho_cache_attention(*(t.to(DEV) for t in (phi, gq, gk, codes, values)), table.int().to(DEV),
                                       _ints([600]), scale=0.25)
    # the output's rounding is none here; a weight's, beyond 64 tokens, at most 2^-11, and the sums' are below 2^-16
    sign = torch.ones(64, dtype=torch.float64)
    sign[1::2] = -1
    off = (out.double().cpu().view(n, 2, 64) * sign - 65504).abs().max().item()
    assert off <= 65504 * (2.0 ** -11 + 2.0 ** -16 if n > 64 else 2.0 ** -16) + 16, off


# ---------------------------------------------------------------- calls that are allowed
@pytest.mark.parametrize("n", [1, 30, 80])
@pytest.mark.parametrize("scale", [0.0, -0.5])
def test_scales_without_and_against_the_scores(n, scale):
    """At scale 0 every key that is seen weighs the same; a negative one turns the
    order of the scores round."""
    p = Problem(2, n, 2, 32, 64, [150, 33], seed=n, scale=scale)
    _check(p.attend(p.device()), p.reference())


@pytest.mark.parametrize("n", [1, 3, 100])
def test_a_sequence_without_pages_in_a_padded_batch(n):
    """What fills a batch up has no pages: nothing of it is stored, its rows see
    nothing, and the others are what they are alone."""
    g = torch.Generator().manual_seed(n)
    H, m, dv, P = 2, 16, 64, 64
    codes, values, table, _, gq, gk = (t.to(DEV) for t in _attention_case(2, n, H, m, dv, [90, 10], P, n))
    x = torch.randn((4, n, H * dv), generator=g).half().to(DEV)
    w = (torch.randn((H * m + H * dv, H * dv), generator=g) / 11).half().to(DEV)
    outs = []
    for rows in ([0, 1], [2, 0, 1, 3]):
        pool = codes.clone(), values.clone()
        full = torch.full((4, table.shape[1]), -1, dtype=torch.int32, device=DEV)
        full[:2] = table
        at = full[rows].contiguous(), _ints([[90, 10, 0, 0][r] for r in rows])
        xs = x[rows].contiguous()
        phi = ma.morpho_cache_append(xs, w, *pool, *at)
        out, lse = ma.morpho_cache_attention(phi, gq, gk, *pool, *at)
        outs.append((*pool, phi, out, lse.view(len(rows), H, n)))
    (c0, v0, phi0, out0, lse0), (c1, v1, phi1, out1, lse1) = outs
    assert torch.equal(c0, c1) and torch.equal(v0, v1)
    for one, four in ((phi0, phi1), (out0, out1), (lse0, lse1)):
        assert torch.equal(one, four[1:3])
    assert (out1[::3] == 0).all() and (lse1[::3] == -torch.finfo(torch.float32).max).all()


def test_copies_and_compactions_in_a_graph():
    """Captured once and replayed with other lists: each replay does what they say."""
    g = torch.Generator().manual_seed(4)
    H, m, dv, P, L, B, K = 2, 16, 64, 32, 2, 2, 6
    codes = torch.randn((L, 9, H, P, m), generator=g).half().to(DEV)
    values = torch.randn((L, 9, H, P // 8, dv, 8), generator=g).half().to(DEV)
    table, lens = _ints([[0, 3], [5, 1]]), _ints([0, 0])
    src, dst, keep, count = _ints([0, 1]), _ints([7, 8]), _ints([[0] * K] * B), _ints([0, 0])

    def go(c, v):
        ma.morpho_cache_copy_pages(c, v, src, dst)
        ma.morpho_cache_compact(c, v, table, lens, keep, keep_lens=count)

    go(codes.clone(), values.clone())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        go(codes, values)
    for r in range(4):
        src.copy_(_ints([r % 4, 5]))
        dst.copy_(_ints([7, 6 + 2 * (r % 2)]))
        lens.copy_(_ints([r, 20 - r]))
        keep.copy_(_ints([[1, 2, 5, 9, 30, 33], [0, 2, 4, 6, 8, 10 + r]]))
        count.copy_(_ints([r + 2, K - r]))
        want = codes.clone(), values.clone()
        go(*want)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(codes, want[0]) and torch.equal(values, want[1])
        torch.randn(1000, device=DEV).sum()  # the program's own work in between


def test_a_dropped_step_leaves_generation_as_it_was():
    """Drafts that are run and dropped, and another sequence in their pages: both
    sequences go on as if the drafts had never been."""
    H, m, dv = 2, 16, 64
    torch.manual_seed(5)
    layer = ma.MorphoAttention(H * dv, H, m, causal=True, scale=0.25, device=DEV)
    w = layer.pack_cache_weights()
    xs = torch.randn((2, 150, H * dv), device=DEV).half()
    drafts = torch.randn((1, 60, H * dv), device=DEV).half()
    outs = []
    for dropped in (False, True):
        cache = ma.MorphoCache(10, H, m, dv, page_size=32, device=DEV)
        a, b = cache.new(), cache.new()

        def run(seq, x, commit=True):
            step = cache.step([seq], x.shape[1])
            with torch.no_grad():
                y = layer.forward_cached(x.contiguous(), w, cache, step)
            cache.commit(step) if commit else cache.drop(step)
            return y
        mine = [run(a, xs[:1, :70])]
        if dropped:
            run(a, drafts, commit=False)
            assert cache.free_pages == 7
        mine += [run(b, xs[1:, :140]), run(a, xs[:1, 70:73]), run(b, xs[1:, 140:]), run(a, xs[:1, 73:150])]
        outs.append(mine)
    assert all(torch.equal(p, q) for p, q in zip(*outs))
