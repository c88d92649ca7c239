"""The paged cache's operators on the GPU against their definitions in 64 bits.

Tolerances (fp16 rounds by at most 2^-11 of a value):

* attention: the output's rounding, 2^-11 |out|, plus what the fp32 sums leave.
  A score is a sum of m products u phi with u carried to 2^-22 and at most
  2^-23 more of the running sum a step, so with S = sum |u phi| its error is at
  most (2^-22 + m 2^-23) S in base 2, taken with both signs by the weights and
  their sum; the exponential and the split of a weight add 2^-20. Summing k
  weights one after another adds k 2^-24 at most, the lanes' partial sums have
  k / 16 terms each. Beyond 64 new tokens the weights of the values are rounded
  to fp16, those of the divisor are not: sum p (1 + e) v / sum p, |e| <= 2^-11,
  is off by at most 2^-11 max |v|.
* log-sum-exp: the score's error, the row constant's of the same size, and 2^-20
  (1 + |lse|).
* append: a sum of D products in fp32, D 2^-24 sum |x w| at most, the sigmoid's
  2^-18 and the rounding to fp16.
* copies and moves: none.
"""

from __future__ import annotations

import math

import pytest
import torch

import morphottention_amd as ma

pytestmark = pytest.mark.gpu
DEV = "cuda"
FLT_MAX = torch.finfo(torch.float32).max


def _pool(pages, H, P, m, dv, layers=None, fill=float("nan")):
    lead = () if layers is None else (layers,)
    return (torch.full((*lead, pages, H, P, m), fill, dtype=torch.float16),
            torch.full((*lead, pages, H, P // 8, dv, 8), fill, dtype=torch.float16))


class Problem:
    """Random sequences in pages. What is not a token of a sequence is NaN."""

    def __init__(self, B, n, H, m, dv, lens, *, P=64, news=None, seed=0, scale=None, gate=1.0, spare=2):
        g = torch.Generator().manual_seed(seed)
        self.B, self.n, self.H, self.m, self.dv, self.P = B, n, H, m, dv, P
        self.lens, self.news = list(lens), list(news) if news is not None else [n] * B
        self.ragged = news is not None
        self.scale = m ** -0.5 if scale is None else scale
        per = max(-(-(l + n) // P) for l in lens)
        pages = B * per + spare
        self.table = torch.randperm(pages, generator=g)[: B * per].view(B, per).to(torch.int32)
        self.codes, self.values = _pool(pages, H, P, m, dv)
        self.phi = torch.rand((B, n, H, m), generator=g).half()
        self.gq = (gate * (1 + 0.3 * torch.randn((H, m), generator=g))).half()
        self.gk = (1 + 0.3 * torch.randn((H, m), generator=g)).half()
        self.k, self.v = [], []
        for b in range(B):
            total = self.lens[b] + self.news[b]
            k = torch.rand((total, H, m), generator=g).half()
            v = torch.randn((total, H, dv), generator=g).half()
            for i in range(self.news[b]):  # a new token's codes are its query's
                k[self.lens[b] + i] = self.phi[b, i]
            self.k.append(k)
            self.v.append(v)
            self.store(b)

    def store(self, b):
        for t in range(self.k[b].shape[0]):
            page, s = int(self.table[b, t // self.P]), t % self.P
            self.codes[page, :, s] = self.k[b][t]
            self.values[page, :, s // 8, :, s % 8] = self.v[b][t]

    def device(self):
        d = {k: getattr(self, k).to(DEV) for k in ("codes", "values", "table", "phi", "gq", "gk")}
        d["lens"] = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        d["new_lens"] = torch.tensor(self.news, dtype=torch.int32, device=DEV) if self.ragged else None
        return d

    def attend(self, d, **kw):
        return ma.morpho_cache_attention(d["phi"], d["gq"], d["gk"], d["codes"], d["values"], d["table"], d["lens"],
                                         new_lens=d["new_lens"], scale=self.scale, **kw)

    def reference(self, mask="causal", mask_diag=False, tree=None, drop=None):
        """out, lse and their tolerances; drop(b) -> positions that do not exist."""
        B, n, H, dv = self.B, self.n, self.H, self.dv
        out = torch.zeros((B, n, H, dv), dtype=torch.float64)
        lse = torch.full((B, H, n), -FLT_MAX, dtype=torch.float64)
        tol_out, tol_lse = torch.zeros_like(out), torch.zeros_like(lse)
        G = self.gq.double() * self.gk.double()
        for b in range(B):
            L, nb = self.lens[b], self.news[b]
            T = L + nb
            if nb == 0:
                continue
            seen = torch.ones((nb, T), dtype=torch.bool)
            if tree is not None:
                for i in range(nb):
                    for k in range(nb):
                        seen[i, L + k] = (int(tree[b, i]) >> k) & 1
            elif mask == "causal":
                seen = torch.tril(seen, L)
            if mask_diag:
                seen[torch.arange(nb), L + torch.arange(nb)] = False
            if drop is not None:
                seen[:, drop(b)] = False
            for h in range(H):
                q, k = self.phi[b, :nb, h].double(), self.k[b][:, h].double()
                v = self.v[b][:, h].double()
                u = self.scale * math.log2(math.e) * G[h] * (2 * q - 1)
                r = self.scale * math.log2(math.e) * (q @ G[h])
                for i in range(nb):
                    at = seen[i].nonzero()[:, 0]
                    if not len(at):
                        continue
                    s = k[at] @ u[i]
                    e = ((k[at].abs() @ u[i].abs()).max() * (2.0 ** -22 + self.m * 2.0 ** -23)).item()
                    top = s.max()
                    w = torch.exp2(s - top)
                    out[b, i, h] = (w / w.sum()) @ v[at]
                    lse[b, h, i] = top + torch.log2(w.sum()) - r[i]
                    rel = 2 * e * math.log(2) + 2.0 ** -20 + len(at) / 16 * 2.0 ** -24
                    if n > 64:
                        rel += 2.0 ** -11
                    tol_out[b, i, h] = out[b, i, h].abs() * 2.0 ** -11 + rel * v[at].abs().max() + 2.0 ** -25
                    tol_lse[b, h, i] = 2 * e + 2.0 ** -20 * (1 + lse[b, h, i].abs()) + len(at) / 16 * 2.0 ** -24
        return (out.reshape(B, n, H * dv), lse.reshape(B * H, n), tol_out.reshape(B, n, H * dv),
                tol_lse.reshape(B * H, n))


def _check(got, want):
    out, lse = (t.double().cpu() for t in got)
    ref_out, ref_lse, tol_out, tol_lse = want
    assert out.isfinite().all() and lse.isfinite().all()
    over = (out - ref_out).abs() - tol_out
    assert over.max() <= 0, (over.max().item(), over.argmax().item())
    over = (lse - ref_lse).abs() - tol_lse - ref_lse.abs() * (ref_lse == -FLT_MAX) * 2.0 ** -23
    assert over.max() <= 0, (over.max().item(), over.argmax().item())


# ---------------------------------------------------------------- attention
@pytest.mark.parametrize("m", [16, 32, 64])
@pytest.mark.parametrize("dv", [32, 64, 128])
@pytest.mark.parametrize("n", [1, 20, 50, 70])
def test_attention_shapes(m, dv, n):
    p = Problem(2, n, 3, m, dv, [37, 190], news=[n, max(1, n - 3)], seed=m + dv + n)
    _check(p.attend(p.device(), max_len=190 + n), p.reference())


@pytest.mark.parametrize("P", [32, 64, 128, 256])
@pytest.mark.parametrize("lens", [[0], [1], [31, 32, 33], [63, 64, 65, 0], [255, 256, 257]])
def test_single_tokens_at_page_edges(P, lens):
    p = Problem(len(lens), 1, 2, 16, 32, lens, P=P, seed=P)
    _check(p.attend(p.device()), p.reference())


@pytest.mark.parametrize("n", [2, 16, 17, 32, 33, 64, 65, 257, 300])
@pytest.mark.parametrize("mask,mask_diag", [("causal", False), ("causal", True), ("full", False), ("full", True)])
def test_masks(n, mask, mask_diag):
    p = Problem(3, n, 2, 32, 64, [0, 45, 130], P=32, news=[n, n // 2, 0], seed=n)
    _check(p.attend(p.device(), causal=mask == "causal", mask_diag=mask_diag), p.reference(mask, mask_diag))


@pytest.mark.parametrize("B,H,n,L,m,dv", [(1, 1, 1, 5000, 16, 64), (2, 2, 3, 3000, 32, 32), (1, 2, 64, 1500, 64, 128),
                                          (1, 1, 80, 2500, 16, 64), (1, 2, 300, 1200, 64, 32)])
def test_divided_keys(B, H, n, L, m, dv):
    """Lengths at which the keys are divided among workgroups; the hint of the
    longest length may be short or long without changing the result."""
    p = Problem(B, n, H, m, dv, [L - 700 * b for b in range(B)], seed=L)
    d = p.device()
    want = p.reference()
    for max_len in (None, L + n, 600, 40 * L):
        _check(p.attend(d, max_len=max_len), want)


@pytest.mark.parametrize("n", [1, 7, 16, 31, 64])
@pytest.mark.parametrize("L", [0, 50, 700])
def test_trees(n, L):
    g = torch.Generator().manual_seed(n)
    p = Problem(2, n, 2, 16, 64, [L, L + 13], news=[n, max(0, n - 2)], seed=n + L)
    tree = torch.zeros((2, n), dtype=torch.int64)
    for b in range(2):
        for k in range(n):
            parent = int(torch.randint(-1, max(k, 1), (1,), generator=g)) if k else -1
            bits = (int(tree[b, parent]) if parent >= 0 else 0) & (2 ** 64 - 1) | 1 << k
            tree[b, k] = bits - 2 ** 64 if bits >> 63 else bits
    tree[1, 0] = 0  # sees no draft: nothing at all where L is 0 ... of sequence 0 below
    tree[0, n // 2] = 0
    d = p.device()
    want = p.reference(tree=tree)
    got = p.attend(d, tree=tree.to(DEV))
    _check(got, want)
    if L == 0:
        assert (got[0][0, n // 2] == 0).all() and (got[1].view(2, 2, n)[0, :, n // 2] == -FLT_MAX).all()


def test_rows_that_see_nothing():
    p = Problem(2, 5, 2, 16, 32, [0, 0], news=[5, 3], seed=3)
    out, lse = p.attend(p.device(), mask_diag=True)
    want = p.reference(mask_diag=True)
    _check((out, lse), want)
    assert (out[:, 0] == 0).all() and (lse[:, 0] == -FLT_MAX).all()  # only its own key, which is dropped
    assert (out[1, 3:] == 0).all() and (lse.view(2, 2, 5)[1, :, 3:] == -FLT_MAX).all()  # padding


@pytest.mark.parametrize("n", [1, 5, 40, 70])
def test_what_is_not_finite_stays_with_the_rows_that_see_it(n):
    """An infinite or NaN value of a new token reaches the rows that see it, in its
    column, and no other; padding rows may hold anything."""
    p = Problem(1, n, 2, 16, 64, [40], seed=9)
    at = n // 2
    p.v[0][40 + at, 0, 3] = math.inf
    p.v[0][40 + at, 1, 7] = math.nan
    p.store(0)
    d = p.device()
    out = p.attend(d)[0].float().cpu().view(1, n, 2, 64)
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[:, at:, 0, 3] = True
    bad[:, at:, 1, 7] = True
    assert torch.equal(~out.isfinite(), bad)
    p.v[0][40 + at] = 0
    p.store(0)
    clean = p.attend(p.device())[0].float().cpu().view(1, n, 2, 64)
    assert torch.equal(clean[:, :at], out[:, :at])


@pytest.mark.parametrize("n", [1, 70])
def test_padding_codes_may_hold_anything(n):
    p = Problem(2, n, 2, 16, 32, [20, 33], news=[n, 0], seed=4)
    p.phi[1] = math.nan
    _check(p.attend(p.device()), p.reference())


@pytest.mark.parametrize("n", [3, 20, 70])
@pytest.mark.parametrize("P", [32, 64])
def test_pages_that_the_pool_does_not_have(n, P):
    """Their keys are left out, wherever they lie."""
    p = Problem(2, n, 2, 32, 64, [300, 500], P=P, seed=5)
    gone = {0: [0, 3, 300 // P], 1: [2, 5]}
    for b, rows in gone.items():
        for i, k in enumerate(rows):
            p.table[b, k] = (-1, p.codes.shape[0] + 7, 2 ** 31 - 1)[i]

    def drop(b):
        T = p.lens[b] + p.news[b]
        return [t for t in range(T) if t // P in gone[b]]
    _check(p.attend(p.device()), p.reference(drop=drop))
    _check(p.attend(p.device(), causal=False), p.reference("full", drop=drop))


def test_lengths_past_the_table_and_negative():
    p = Problem(2, 2, 2, 16, 32, [62, 100], P=64, seed=6)
    d = p.device()
    d["lens"] = torch.tensor([-5, 2 ** 31 - 1], dtype=torch.int32, device=DEV)
    d["codes"].nan_to_num_(0.5)
    d["values"].nan_to_num_(0.5)
    out, lse = p.attend(d)
    assert out.isfinite().all() and lse.isfinite().all()


@pytest.mark.parametrize("gate", [1e-3, 30.0, 200.0])
def test_score_ranges(gate):
    """Flat rows and rows with one key; the exponents' range is the row's own."""
    p = Problem(2, 4, 2, 16, 64, [400, 150], seed=7, scale=1.0, gate=gate)
    _check(p.attend(p.device()), p.reference())


@pytest.mark.parametrize("n,m,dv", [(8, 16, 64), (40, 32, 32), (70, 16, 64), (70, 32, 32), (70, 64, 64), (130, 16, 128)])
@pytest.mark.parametrize("top", [20.0, 400.0])
@pytest.mark.parametrize("order", ["rising", "falling", "peaks"])
def test_references_that_move(n, m, dv, top, order):
    """Scores up to 1.44 top: every tile passes the ones before it, none does, or a few keys do."""
    p = Problem(2, n, 2, m, dv, [450, 130], seed=m + n, scale=top / m)
    g = torch.Generator().manual_seed(n)
    p.gq, p.gk = torch.ones_like(p.gq), torch.ones_like(p.gk)
    p.phi = (1 - 0.1 * torch.rand(p.phi.shape, generator=g)).half()  # positive factors of the codes
    for b in range(2):
        T = p.k[b].shape[0]
        at = torch.linspace(0, 1, T)[:, None, None]
        if order == "falling":
            at = 1 - at
        if order == "peaks":
            at = (torch.rand((T, 1, 1), generator=g) < 0.02).float()
        p.k[b] = (at * (1 - 0.05 * torch.rand((T, 2, m), generator=g))).half()
        p.store(b)
    _check(p.attend(p.device()), p.reference())
    _check(p.attend(p.device(), causal=False), p.reference("full"))


@pytest.mark.parametrize("m,dv", [(16, 32), (16, 64), (32, 32), (32, 64)])
def test_many_sequences_of_many_rows(m, dv):
    """Three sequences 90 times over, so many row blocks that they are larger ones."""
    p = Problem(3, 130, 2, m, dv, [0, 65, 150], news=[130, 97, 128], seed=m + dv)
    d = p.device()
    for k in ("phi", "table", "lens", "new_lens"):
        d[k] = d[k].repeat(90, *[1] * (d[k].dim() - 1))
    out, lse = p.attend(d)
    want = p.reference()
    for i in (0, 1, 44, 89):
        _check((out[3 * i : 3 * i + 3], lse[6 * i : 6 * i + 6]), want)
    same = out.view(90, 3, 130, -1), lse.view(90, 6, 130)
    assert all(torch.equal(x, x[:1].expand_as(x)) for x in same)


def test_attention_repeats_bit_for_bit():
    p = Problem(2, 3, 2, 16, 64, [4000, 2500], seed=8)
    d = p.device()
    first = p.attend(d)
    for _ in range(3):
        for a, b in zip(first, p.attend(d)):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- append
def _append_reference(x, w, H, m, projection):
    z = x.double() @ w.double().t()
    e = 2.0 ** -24 * x.shape[-1] * (x.double().abs() @ w.double().abs().t())
    zc, ec = z[..., : H * m], e[..., : H * m]
    if projection == "sigmoid":
        phi, tol = torch.sigmoid(zc), ec / 4 + 2.0 ** -18 * torch.sigmoid(zc)
    elif projection == "hardtanh01":
        phi, tol = ((zc + 1) / 2).clamp(0, 1), ec / 2 + 2.0 ** -23
    else:
        phi, tol = zc, ec
    tol = tol + phi.abs() * 2.0 ** -11 + 2.0 ** -25
    v, tv = z[..., H * m:], e[..., H * m:]
    return phi, tol, v, tv + v.abs() * 2.0 ** -11 + 2.0 ** -25


def _check_append(B, n, H, m, dv, lens, news, projection, P=64):
    g = torch.Generator().manual_seed(m + dv + n)
    D = H * dv
    p = Problem(B, n, H, m, dv, lens, P=P, news=news, seed=n)
    x = torch.randn((B, n, D), generator=g).half()
    w = (torch.randn((H * m + D, D), generator=g) * D ** -0.5).half()
    d = p.device()
    codes, values = d["codes"].cpu(), d["values"].cpu()
    phi = ma.morpho_cache_append(x.to(DEV), w.to(DEV), d["codes"], d["values"], d["table"], d["lens"],
                                 new_lens=d["new_lens"], projection=projection).cpu()
    ref, tol, v, tv = _append_reference(x, w, H, m, projection)
    assert ((phi.double().reshape(B, n, H * m) - ref).abs() <= tol).all()
    dc, dval = d["codes"].cpu(), d["values"].cpu()
    for b in range(B):
        t = lens[b] + torch.arange(p.news[b])
        page, s = p.table[b].long()[t // P], t % P
        codes[page, :, s] = phi[b, : p.news[b]]
        got = dval[page, :, s // 8, :, s % 8]
        assert ((got.double().reshape(-1, D) - v[b, : p.news[b]]).abs() <= tv[b, : p.news[b]]).all()
        values[page, :, s // 8, :, s % 8] = got
    # what was not appended to is as it was, NaN included
    assert torch.equal(dc.view(torch.int16), codes.view(torch.int16))
    assert torch.equal(dval.view(torch.int16), values.view(torch.int16))


@pytest.mark.parametrize("m,dv,H", [(16, 32, 8), (16, 64, 3), (32, 64, 4), (64, 32, 5), (64, 128, 2), (32, 128, 1), (16, 32, 1)])
@pytest.mark.parametrize("B,n,lens,news", [(1, 1, [37], None), (5, 1, [0, 63, 64, 65, 128], [1, 0, 1, 1, 1]),
                                           (3, 13, [0, 60, 127], [13, 2, 0]), (2, 40, [5, 30], None),
                                           (3, 150, [0, 3, 61], [150, 149, 7])])
def test_append(m, dv, H, B, n, lens, news):
    for projection in ("sigmoid", "hardtanh01", "identity") if n == 13 else ("sigmoid",):
        _check_append(B, n, H, m, dv, lens, news, projection)


@pytest.mark.parametrize("m,dv,H", [(64, 64, 8), (16, 128, 3), (16, 64, 16)])
@pytest.mark.parametrize("T,B", [(200, 5), (500, 20), (1100, 1), (5000, 3), (5000, 100)])
def test_append_many(m, dv, H, T, B):
    """Every launch shape: the widest strips and the tiles, with sequences longer and
    shorter than 64 new tokens, starting anywhere in a group of 8."""
    n = T // B
    g = torch.Generator().manual_seed(T + B)
    lens = torch.randint(0, 70, (B,), generator=g).tolist()
    news = torch.randint(0, n + 1, (B,), generator=g).tolist()
    news[0] = n
    _check_append(B, n, H, m, dv, lens, news if B > 1 else None, "hardtanh01" if T == 500 else "sigmoid")


@pytest.mark.parametrize("n", [1, 200])
def test_append_to_places_that_are_not_there(n):
    """Positions past the table, and pages that the pool does not have, are not stored."""
    H, m, dv, P = 2, 16, 32, 32
    D = H * dv
    codes, values = (t.to(DEV) for t in _pool(4, H, P, m, dv, fill=7.0))
    table = torch.tensor([[0, -1], [9, 1]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([30, 40], dtype=torch.int32, device=DEV)
    x = torch.randn((2, n, D), device=DEV).half()
    w = torch.randn((H * m + D, D), device=DEV).half()
    ma.morpho_cache_append(x, w, codes, values, table, lens)
    assert (codes[2:] == 7).all() and (values[2:] == 7).all()
    assert (codes[0, :, :30] == 7).all() and (codes[1, :, :8] == 7).all()
    wrote = (codes[1] != 7).any(-1).any(0)
    assert wrote[8] and int(wrote.sum()) == min(n, 24)


# ---------------------------------------------------------------- copies and moves
@pytest.mark.parametrize("m,dv,P,H", [(16, 64, 64, 3), (64, 128, 256, 2), (32, 32, 32, 1), (16, 32, 128, 5)])
@pytest.mark.parametrize("layers", [None, 3])
def test_copy_pages(m, dv, P, H, layers):
    g = torch.Generator().manual_seed(P)
    codes, values = _pool(11, H, P, m, dv, layers)
    codes.normal_(generator=g)
    values.normal_(generator=g)
    src, dst = [3, 3, 0, 10, -1, 5, 11], [1, 2, 4, 9, 6, -1, 7]  # the last three are left out
    dc, dv_ = codes.to(DEV), values.to(DEV)
    ma.morpho_cache_copy_pages(dc, dv_, torch.tensor(src, dtype=torch.int32, device=DEV),
                               torch.tensor(dst, dtype=torch.int32, device=DEV))
    for a, b in zip(src[:4], dst[:4]):
        if layers is None:
            codes[b], values[b] = codes[a].clone(), values[a].clone()
        else:
            codes[:, b], values[:, b] = codes[:, a].clone(), values[:, a].clone()
    assert torch.equal(dc.cpu(), codes) and torch.equal(dv_.cpu(), values)
    none = torch.empty(0, dtype=torch.int32, device=DEV)
    ma.morpho_cache_copy_pages(dc, dv_, none, none)


@pytest.mark.parametrize("m,dv,P,H", [(16, 64, 64, 3), (64, 128, 128, 2), (32, 32, 32, 1)])
@pytest.mark.parametrize("layers", [None, 2])
@pytest.mark.parametrize("span,kept", [(1, 1), (9, 4), (60, 60), (130, 70), (200, 190), (300, 299), (400, 130), (2200, 1500)])
def test_compact(m, dv, P, H, layers, span, kept):
    g = torch.Generator().manual_seed(span + P)
    B, lens = 3, [0, 13, 70]
    per = -(-(max(lens) + span) // P)
    codes, values = _pool(B * per + 1, H, P, m, dv, layers)
    codes.normal_(generator=g)
    values.normal_(generator=g)
    table = torch.randperm(B * per + 1, generator=g)[: B * per].view(B, per).to(torch.int32)
    counts = [kept, max(0, kept - 1), 0]
    keep = torch.stack([torch.randperm(span, generator=g)[:kept].sort()[0] for _ in range(B)]).to(torch.int32)
    dc, dv_ = codes.to(DEV), values.to(DEV)
    ma.morpho_cache_compact(dc, dv_, table.to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV), keep.to(DEV),
                            keep_lens=torch.tensor(counts, dtype=torch.int32, device=DEV))
    for c, v in zip([codes] if layers is None else codes, [values] if layers is None else values):
        for b in range(B):
            for k in range(counts[b]):
                a, z = lens[b] + int(keep[b, k]), lens[b] + k
                pa, pz = int(table[b, a // P]), int(table[b, z // P])
                c[pz, :, z % P] = c[pa, :, a % P].clone()
                v[pz, :, z % P // 8, :, z % 8] = v[pa, :, a % P // 8, :, a % 8].clone()
    assert torch.equal(dc.cpu(), codes) and torch.equal(dv_.cpu(), values)


def test_compact_leaves_out_what_is_not_there():
    codes, values = (t.to(DEV) for t in _pool(3, 1, 32, 16, 32, fill=1.0))
    codes[1], values[1] = 2.0, 2.0
    table = torch.tensor([[0, 1, 5]], dtype=torch.int32, device=DEV)
    lens = torch.zeros(1, dtype=torch.int32, device=DEV)
    keep = torch.tensor([[-1, 40, 70, 90, 96, 1000]], dtype=torch.int32, device=DEV)
    ma.morpho_cache_compact(codes, values, table, lens, keep)
    assert (codes[0, 0, 1] == 2).all() and int((codes[0] == 2).all(-1).sum()) == 1
    assert (values[0, 0, 0, :, 1] == 2).all() and (values[2] == 1).all()


# ---------------------------------------------------------------- together
def _layer(dim, heads, m, seed, **kw):
    torch.manual_seed(seed)
    return ma.MorphoAttention(dim, heads, m, causal=True, scale=m ** -0.5, device=DEV, **kw)


def _close_to_forward(got, layer, x):
    """The cached path against the whole-sequence forward: codes rounded to fp16
    (2^-11 of phi <= 1) move a score by at most 2^-11 sum |u| in base 2, values
    by 2^-11, each output rounds once more on either side."""
    with torch.no_grad():
        want = layer(x).float()
    V = (x.float() @ layer.W_V.float()).abs().max().item()
    H, m = layer.num_heads, layer.cube_m
    u = layer.scale * math.log2(math.e) * (layer.gate_q.float() * layer.gate_k.float()).abs().sum(1).max().item()
    # a key's code moves by half a step of fp16 below 1, 2^-12; the query's likewise, with factor 2
    tol = 3 * u * 2.0 ** -12 * math.log(2) * 2 * V + 2.0 ** -11 * V * 2
    assert (got.float() - want).abs().max().item() <= tol


@pytest.mark.parametrize("m,dv,kw", [(16, 64, {}), (32, 32, {"projection": "hardtanh01"}), (64, 128, {"mask_diag": True})])
def test_generation_matches_the_whole_sequence(m, dv, kw):
    """A prompt in pieces, then single tokens, of two sequences of different lengths."""
    H = 4
    layer = _layer(H * dv, H, m, 1, **kw)
    w = layer.pack_cache_weights()
    cache = ma.MorphoCache(24, H, m, dv, num_layers=2, device=DEV)
    x = torch.randn((2, 200, H * dv), device=DEV).half()
    ends = [200, 171]
    seqs = [cache.new(), cache.new()]
    outs = [[], []]
    at = [0, 0]
    for n in [100, 60] + [1] * 45:
        counts = [min(n, e - a) for e, a in zip(ends, at)]
        if max(counts) == 0:
            break
        step = cache.step(seqs, counts)
        piece = torch.zeros((2, step.n, H * dv), dtype=torch.float16, device=DEV)
        for b in range(2):
            piece[b, : counts[b]] = x[b, at[b]: at[b] + counts[b]]
        with torch.no_grad():
            y = layer.forward_cached(piece, w, cache, step, layer=1)
        cache.commit(step)
        for b in range(2):
            outs[b].append(y[b, : counts[b]])
            assert (y[b, counts[b]:] == 0).all()
            at[b] += counts[b]
    assert [cache.length(s) for s in seqs] == ends
    for b in range(2):
        _close_to_forward(torch.cat(outs[b])[None], layer, x[b: b + 1, : ends[b]].contiguous())


def test_forks_drafts_and_eviction():
    """Fork, append to both, accept a path of a tree, evict: each sequence stays what
    its own tokens make it."""
    H, m, dv = 2, 16, 64
    layer = _layer(H * dv, H, m, 2)
    w = layer.pack_cache_weights()
    cache = ma.MorphoCache(40, H, m, dv, page_size=32, device=DEV)
    toks = {}

    def add(seqs, xs, kept=None, tree=None):
        step = cache.step(seqs, xs.shape[1])
        with torch.no_grad():
            y = layer.forward_cached(xs, w, cache, step, tree=tree)
        if kept is None:
            cache.commit(step)
            kept = [list(range(xs.shape[1]))] * len(seqs)
        else:
            cache.accept(step, kept)
        for i, s in enumerate(seqs):
            toks[s] = torch.cat([toks.get(s, xs[i, :0]), xs[i, kept[i]]])
        return y

    rnd = lambda b, n: torch.randn((b, n, H * dv), device=DEV).half()  # noqa: E731
    a = cache.new()
    add([a], rnd(1, 75))
    b = cache.fork(a)
    toks[b] = toks[a].clone()
    assert cache.pages(a)[:2] == cache.pages(b)[:2] and cache.pages(a)[2] != cache.pages(b)[2]
    add([a, b], rnd(2, 9))
    # a tree of 6 drafts: 0-1-2 and 0-3-4, 5 a root of its own
    parents = [-1, 0, 1, 0, 3, -1]
    bits = []
    for k, p in enumerate(parents):
        bits.append((bits[p] if p >= 0 else 0) | 1 << k)
    tree = torch.tensor([bits, bits], dtype=torch.int64, device=DEV)
    drafts = rnd(2, 6)
    old = toks[a].clone()
    y = add([a, b], drafts, kept=[[0, 3, 4], [5]], tree=tree)
    path = torch.cat([old, drafts[0, [0, 3, 4]]])[None]
    with torch.no_grad():
        want = layer(path)[0, -1].float()
    V = (path.float() @ layer.W_V.float()).abs().max().item()
    u = layer.scale * math.log2(math.e) * m
    tol = 3 * u * 2.0 ** -12 * math.log(2) * 2 * V + 2.0 ** -10 * V
    assert (y[0, 4].float() - want).abs().max().item() <= tol
    c = cache.fork(b)
    toks[c] = toks[b].clone()
    kept = [0, 1, 2, 5, 40, 41, 60, 80]
    cache.evict(c, kept)
    stored = cache.codes[0], cache.values[0]

    def codes_of(s):
        pg = torch.tensor(cache.pages(s), device=DEV)
        return stored[0][pg].transpose(1, 2).reshape(-1, H, m)[: cache.length(s)]
    assert torch.equal(codes_of(c), codes_of(b)[kept])
    for s in (a, b):
        z = add([s], rnd(1, 1))
        with torch.no_grad():
            want = layer(toks[s][None])[0, -1].float()
        assert (z[0, 0].float() - want).abs().max().item() <= tol
    for s in (a, b, c):
        cache.free(s)
    assert cache.free_pages == 40


def test_a_captured_step_follows_the_lengths():
    """Append and attention in a graph, replayed with other tokens and lengths."""
    H, m, dv, P, B = 2, 16, 64, 64, 3
    layer = _layer(H * dv, H, m, 3)
    w = layer.pack_cache_weights()
    cache = ma.MorphoCache(40, H, m, dv, page_size=P, device=DEV)
    codes, values = cache.codes[0], cache.values[0]
    codes.uniform_(0, 1)
    values.normal_()
    table = torch.randperm(40, device=DEV)[: B * 12].view(B, 12).to(torch.int32)
    lens = torch.tensor([700, 5, 63], dtype=torch.int32, device=DEV)
    x = torch.randn((B, 1, H * dv), device=DEV).half()

    def go():
        phi = ma.morpho_cache_append(x, w, codes, values, table, lens)
        return ma.morpho_cache_attention(phi, layer.gate_q, layer.gate_k, codes, values, table, lens, scale=layer.scale)

    with torch.no_grad():
        go()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out, lse = go()
        for r in range(4):
            x.copy_(torch.randn((B, 1, H * dv), device=DEV).half())
            lens.copy_(torch.tensor([100 * r, 64 + r, 766 - r], dtype=torch.int32, device=DEV))
            graph.replay()
            torch.cuda.synchronize()
            got = out.clone(), lse.clone()
            want = go()
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_a_pool_beyond_32_bits():
    """Pages more than 2^32 bytes into a pool: the same results as near its start."""
    H, m, dv, P, far = 16, 16, 64, 64, 34000  # 128 KiB of values a page
    p = Problem(2, 3, H, m, dv, [100, 190], seed=15)
    d = p.device()
    pages = p.codes.shape[0]
    big = {k: torch.empty((far + pages, *d[k].shape[1:]), dtype=torch.float16, device=DEV) for k in ("codes", "values")}
    x = torch.randn((2, 3, H * dv), device=DEV).half()
    w = (torch.randn((H * m + H * dv, H * dv), device=DEV) / 32).half()
    keep = torch.tensor([[1, 5, 60, 99], [0, 2, 3, 150]], dtype=torch.int32, device=DEV)
    zero = torch.zeros(2, dtype=torch.int32, device=DEV)
    for k in big:
        big[k][far:] = d[k]
    outs = []
    for pool, off in ((d, 0), (big, far)):
        table = d["table"] + off
        phi = ma.morpho_cache_append(x, w, pool["codes"], pool["values"], table, d["lens"])
        out, lse = ma.morpho_cache_attention(phi, d["gq"], d["gk"], pool["codes"], pool["values"], table, d["lens"],
                                             scale=p.scale)
        ma.morpho_cache_compact(pool["codes"], pool["values"], table, zero, keep)
        ma.morpho_cache_copy_pages(pool["codes"], pool["values"], table[0, :2].contiguous(), table[1, :2].contiguous())
        outs.append([phi, out, lse, pool["codes"][off:].clone(), pool["values"][off:].clone()])
    assert big["values"].numel() * 2 > 2 ** 32
    for a, b in zip(*outs):
        assert torch.equal(a.view(torch.int16) if a.dtype == torch.float16 else a,
                           b.view(torch.int16) if b.dtype == torch.float16 else b)


def test_two_graphs_in_turn():
    """Two captured calls with partial results, replayed in turn: each has its own."""
    ps = [Problem(2, n, 2, 16, 64, [3000, 2000 + n], seed=n) for n in (1, 30)]
    ds = [p.device() for p in ps]
    want = [[t.clone() for t in p.attend(d)] for p, d in zip(ps, ds)]
    torch.cuda.synchronize()
    graphs, got = [], []
    for p, d in zip(ps, ds):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(p.attend(d))
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
        ps[0].attend(ds[0])  # the program's own work in between


def test_c_abi_direct_matches_the_ops():
    """The C entry points with a workspace of the caller's, against the torch ops."""
    import ctypes

    from morphottention_amd import capi
    L = capi.lib()
    p = Problem(2, 2, 2, 16, 64, [900, 1500], seed=12)
    d = p.device()
    pool = capi.Cache(d["codes"].data_ptr(), d["values"].data_ptr(), 1, d["codes"].shape[0], 2, 16, 64, 64)
    ref = ctypes.byref(pool)
    W, stream = d["table"].shape[1], torch.cuda.current_stream().cuda_stream
    want = p.attend(d, max_len=1502)
    out, lse = torch.empty_like(want[0]), torch.empty_like(want[1])
    size = capi.cache_attention_workspace_size(pool, 2, 2, W, 1502)
    assert size > 0
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    assert L.morpho_cache_attention(d["phi"].data_ptr(), d["gq"].data_ptr(), d["gk"].data_ptr(), ref,
                                    d["table"].data_ptr(), d["lens"].data_ptr(), None, None, out.data_ptr(),
                                    lse.data_ptr(), 2, 2, W, 1502, p.scale, 1, ws.data_ptr(), size, stream) == 0
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    x, w = torch.randn((2, 2, 128), device=DEV).half(), torch.randn((160, 128), device=DEV).half() / 11
    phi = torch.empty((2, 2, 2, 16), dtype=torch.float16, device=DEV)
    mine = d["codes"].clone(), d["values"].clone()
    assert L.morpho_cache_append(x.data_ptr(), w.data_ptr(), ref, d["table"].data_ptr(), d["lens"].data_ptr(), None,
                                 phi.data_ptr(), 2, 2, W, 0, stream) == 0
    assert torch.equal(phi, ma.morpho_cache_append(x, w, mine[0], mine[1], d["table"], d["lens"]))
    assert torch.equal(mine[0].view(torch.int16), d["codes"].view(torch.int16))
    assert torch.equal(mine[1].view(torch.int16), d["values"].view(torch.int16))


def test_refused_tensors():
    """Wrong types, shapes, layouts and places raise before anything runs."""
    p = Problem(2, 2, 2, 16, 64, [9, 15], seed=13)
    d = p.device()
    call = lambda **kw: p.attend(d | kw)  # noqa: E731
    for kw, text in (({"phi": d["phi"].float()}, "float16"), ({"codes": d["codes"].cpu()}, "CUDA"),
                     ({"phi": d["phi"].transpose(0, 1)}, "contiguous"), ({"table": d["table"].long()}, "int32"),
                     ({"lens": d["lens"][:1]}, "lens must be"), ({"table": d["table"][:1]}, "table must be"),
                     ({"gq": d["gq"][:1]}, "gate_q must be"), ({"phi": d["phi"][:, :, :1].contiguous()}, "phi must be"),
                     ({"values": d["values"][:1]}, "values must be"), ({"new_lens": d["lens"].float()}, "int32"),
                     ({"codes": d["codes"][None]}, "codes must be")):
        with pytest.raises((RuntimeError, NotImplementedError), match=text if text != "CUDA" else None):
            call(**kw)
    with pytest.raises(RuntimeError, match="tree must be"):
        p.attend(d, tree=torch.zeros((2, 2), dtype=torch.int32, device=DEV))
    big = Problem(1, 65, 1, 16, 32, [3], seed=14)
    with pytest.raises(RuntimeError, match="64 drafted"):
        big.attend(big.device(), tree=torch.zeros((1, 65), dtype=torch.int64, device=DEV))
    with pytest.raises(RuntimeError, match="X must be"):
        ma.morpho_cache_append(torch.zeros((2, 2, 64), device=DEV).half(), torch.zeros((160, 128), device=DEV).half(),
                               d["codes"], d["values"], d["table"], d["lens"])
    with pytest.raises(RuntimeError, match="weights must be"):
        ma.morpho_cache_append(torch.zeros((2, 2, 128), device=DEV).half(), torch.zeros((128, 160), device=DEV).half(),
                               d["codes"], d["values"], d["table"], d["lens"])


def test_another_stream():
    p = Problem(2, 3, 2, 16, 64, [900, 1500], seed=11)
    d = p.device()
    first = p.attend(d)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        again = p.attend(d)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))
