"""The paged cache without a GPU: what its entry points refuse, its launch rules,
its fakes, and the account of pages."""

from __future__ import annotations

import ctypes
import os
import random
import shutil
import subprocess

import pytest
import torch

import morphottention_amd as ma
from morphottention_amd import cache as cache_module
from morphottention_amd import capi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000  # a pointer that no refused call follows


def _pool(**kw):
    d = dict(codes=P, values=P, layers=1, pages=4, H=2, cube_m=16, head_dim_v=64, page_size=64) | kw
    return capi.Cache(*(d[k] for k, _ in capi.Cache._fields_))


INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
BAD_POOLS = [({"layers": 0}, INVALID, b"Invalid dimensions"), ({"pages": 0}, INVALID, b"Invalid dimensions"),
             ({"H": 0}, INVALID, b"Invalid dimensions"), ({"cube_m": 24}, UNSUPPORTED, b"cube_m"),
             ({"head_dim_v": 48}, UNSUPPORTED, b"head_dim_v"), ({"page_size": 16}, UNSUPPORTED, b"page_size"),
             ({"page_size": 96}, UNSUPPORTED, b"page_size"), ({"H": 65536}, INVALID, b"too large"),
             ({"pages": 2 ** 31}, INVALID, b"too large"), ({"codes": None}, INVALID, b"Null"),
             ({"values": None}, INVALID, b"Null"), ({"codes": P + 8}, INVALID, b"16-byte"),
             ({"values": P + 2}, INVALID, b"16-byte")]


def _append(pool, X=P, W=P, table=P, lens=P, new_lens=None, phi=P, B=1, n=1, seq_pages=1, mode=0):
    return capi.lib().morpho_cache_append(X, W, pool and ctypes.byref(pool), table, lens, new_lens, phi, B, n,
                                          seq_pages, mode, None)


def _attention(pool, phi=P, gq=P, gk=P, table=P, lens=P, new_lens=None, tree=None, out=P, lse=P, B=1, n=1,
               seq_pages=1, max_len=64, scale=1.0, mode=1, ws=None, ws_bytes=0):
    return capi.lib().morpho_cache_attention(phi, gq, gk, pool and ctypes.byref(pool), table, lens, new_lens, tree,
                                             out, lse, B, n, seq_pages, max_len, scale, mode, ws, ws_bytes, None)


def _copy(pool, src=P, dst=P, count=1):
    return capi.lib().morpho_cache_copy_pages(pool and ctypes.byref(pool), src, dst, count, None)


def _compact(pool, table=P, lens=P, keep=P, keep_lens=None, B=1, cols=1, seq_pages=1):
    return capi.lib().morpho_cache_compact(pool and ctypes.byref(pool), table, lens, keep, keep_lens, B, cols,
                                           seq_pages, None)


def _message():
    return capi.lib().morpho_last_error()


@pytest.mark.parametrize("call", [_append, _attention, _copy, _compact])
def test_bad_pools_are_refused(call):
    for bad, status, text in BAD_POOLS:
        assert call(_pool(**bad)) == status, bad
        assert text in _message(), (bad, _message())
    assert call(None) == INVALID and b"Null" in _message()


@pytest.mark.parametrize("call", [_append, _attention])
def test_one_layer_at_a_time(call):
    assert call(_pool(layers=2)) == INVALID and b"one layer" in _message()


@pytest.mark.parametrize("call,kw,status,text", [
    (_append, {"X": None}, INVALID, b"Null"), (_append, {"W": None}, INVALID, b"Null"),
    (_append, {"table": None}, INVALID, b"Null"), (_append, {"lens": None}, INVALID, b"Null"),
    (_append, {"phi": None}, INVALID, b"Null"), (_append, {"X": P + 4}, INVALID, b"16-byte"),
    (_append, {"phi": P + 2}, INVALID, b"16-byte"), (_append, {"table": P + 2}, INVALID, b"4-byte"),
    (_append, {"new_lens": P + 1}, INVALID, b"4-byte"), (_append, {"mode": 1}, INVALID, b"mode"),
    (_append, {"mode": 12}, INVALID, b"mode"), (_append, {"mode": 2}, INVALID, b"mode"),
    (_append, {"B": 0}, INVALID, b"Invalid dimensions"), (_append, {"n": 0}, INVALID, b"Invalid dimensions"),
    (_append, {"n": 2 ** 22 + 1}, INVALID, b"too large"), (_append, {"B": 2 ** 40, "n": 2 ** 40}, INVALID, b"too large"),
    (_append, {"seq_pages": 2 ** 24 + 1}, INVALID, b"2^30"), (_append, {"seq_pages": 0}, INVALID, b"Invalid dimensions"),
    (_attention, {"phi": None}, INVALID, b"Null"), (_attention, {"gq": None}, INVALID, b"Null"),
    (_attention, {"gk": None}, INVALID, b"Null"), (_attention, {"out": None}, INVALID, b"Null"),
    (_attention, {"lse": None}, INVALID, b"Null"), (_attention, {"lens": None}, INVALID, b"Null"),
    (_attention, {"out": P + 8}, INVALID, b"16-byte"), (_attention, {"lens": P + 2}, INVALID, b"4-byte"),
    (_attention, {"tree": P + 4}, INVALID, b"8-byte"), (_attention, {"tree": P, "n": 65}, UNSUPPORTED, b"64 drafted"),
    (_attention, {"tree": P, "mode": 3}, INVALID, b"own bit"), (_attention, {"mode": 4}, INVALID, b"mode"),
    (_attention, {"max_len": 0}, INVALID, b"max_len"), (_attention, {"scale": float("nan")}, INVALID, b"finite"),
    (_attention, {"scale": float("inf")}, INVALID, b"finite"),
    (_attention, {"seq_pages": 100, "max_len": 6400}, WORKSPACE, b"needs"),
    (_attention, {"seq_pages": 100, "max_len": 6400, "ws": P + 16, "ws_bytes": 1 << 30}, WORKSPACE, b"256-byte"),
    (_copy, {"src": None}, INVALID, b"Null"), (_copy, {"dst": None}, INVALID, b"Null"),
    (_copy, {"src": P + 2}, INVALID, b"4-byte"), (_copy, {"count": -1}, INVALID, b"Invalid dimensions"),
    (_compact, {"keep": None}, INVALID, b"Null"), (_compact, {"table": None}, INVALID, b"Null"),
    (_compact, {"keep_lens": P + 2}, INVALID, b"4-byte"), (_compact, {"cols": -1}, INVALID, b"Invalid dimensions"),
    (_compact, {"B": 0}, INVALID, b"Invalid dimensions"),
])
def test_refusals(call, kw, status, text):
    assert call(_pool(), **kw) == status
    assert text in _message()


def test_nothing_to_do_is_no_error():
    assert _copy(_pool(), None, None, 0) == 0
    assert _compact(_pool(), cols=0) == 0


def test_workspace_sizes():
    size = capi.cache_attention_workspace_size
    assert size(_pool(), 1, 1, 1, 64) == 0                 # one piece needs none
    assert size(_pool(), 1, 1, 1000, 64000) >= 2 * 64 * 4 * 2
    assert size(_pool(), 1, 1, 1000, 1 << 40) == size(_pool(), 1, 1, 1000, 64000)  # no longer than the table
    assert size(_pool(), 1, 1, 1000, 0) == 0 and size(_pool(cube_m=8), 1, 1, 1000, 64000) == 0


def test_python_refusals():
    t = torch.zeros(1)
    with pytest.raises(ValueError, match="projection must be one of"):
        ma.morpho_cache_append(t, t, t, t, t, t, projection="relu")
    with pytest.raises(ValueError, match="max_len"):
        ma.morpho_cache_attention(t, t, t, t, t, t, t, max_len=0)
    with pytest.raises(ValueError, match="own bit"):
        ma.morpho_cache_attention(t, t, t, t, t, t, t, tree=t, mask_diag=True)
    g = torch.zeros(1, requires_grad=True)
    with pytest.raises(RuntimeError, match="no gradients"):
        ma.morpho_cache_append(g, t, t, t, t, t)
    with pytest.raises(RuntimeError, match="no gradients"):
        ma.morpho_cache_attention(t, g, t, t, t, t, t)
    layer = ma.MorphoAttention(64, 1, 16)
    with pytest.raises(ValueError, match="causal layer"):
        layer.forward_cached(t, t, None, None)
    for bad in ({"cube_m": 8}, {"head_dim": 96}, {"page_size": 48}, {"num_pages": 0}, {"num_layers": 0}):
        kw = dict(num_pages=2, num_heads=1, cube_m=16, head_dim=32) | bad
        with pytest.raises(ValueError):
            ma.MorphoCache(**kw)


def test_ops_need_gpu_tensors():
    """CPU tensors have no kernel: an error, not a fallback."""
    c = ma.MorphoCache(2, 1, 16, 32)
    ints = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        ma.morpho_cache_copy_pages(c.codes, c.values, ints, ints)


def test_fakes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        dev = "cuda"
        f = lambda *s: torch.empty(s, dtype=torch.float16, device=dev)  # noqa: E731
        i = lambda *s: torch.empty(s, dtype=torch.int32, device=dev)  # noqa: E731
        codes, values = f(9, 3, 64, 16), f(9, 3, 8, 32, 8)
        phi = ma.morpho_cache_append(f(2, 5, 96), f(144, 96), codes, values, i(2, 4), i(2))
        assert phi.shape == (2, 5, 3, 16) and phi.dtype == torch.float16
        out, lse = ma.morpho_cache_attention(phi, f(3, 16), f(3, 16), codes, values, i(2, 4), i(2))
        assert out.shape == (2, 5, 96) and lse.shape == (6, 5) and lse.dtype == torch.float32
        ma.morpho_cache_copy_pages(codes, values, i(3), i(3))
        ma.morpho_cache_compact(codes, values, i(2, 4), i(2), i(2, 7))


def test_packed_weights():
    w = ma.pack_cache_weights(torch.arange(6.).view(2, 3), torch.arange(6., 10.).view(2, 2))
    assert w.is_contiguous() and w.tolist() == [[0, 3], [1, 4], [2, 5], [6, 8], [7, 9]]
    layer = ma.MorphoAttention(64, 2, 16)
    assert layer.pack_cache_weights().shape == (96, 64) and not layer.pack_cache_weights().requires_grad


# ---------------------------------------------------------------- the account of pages
def _plain_copy(codes, values, src, dst):
    codes[:, dst.long()] = codes[:, src.long()].clone()
    values[:, dst.long()] = values[:, src.long()].clone()


def _plain_compact(codes, values, table, lens, keep, *, keep_lens=None):
    size = codes.shape[3]
    for b in range(keep.shape[0]):
        for k in range(keep.shape[1] if keep_lens is None else int(keep_lens[b])):
            a, z = int(lens[b]) + int(keep[b, k]), int(lens[b]) + k
            pa, pz = int(table[b, a // size]), int(table[b, z // size])
            codes[:, pz, :, z % size] = codes[:, pa, :, a % size].clone()


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(cache_module, "morpho_cache_copy_pages", _plain_copy)
    monkeypatch.setattr(cache_module, "morpho_cache_compact", _plain_compact)


def _check_account(c, toks):
    """Every sequence reads back its own tokens; use counts and the free list agree."""
    uses = [0] * c.num_pages
    for s, mine in toks.items():
        assert c.length(s) == len(mine)
        for p in c.pages(s):
            uses[p] += 1
        for t, value in enumerate(mine):
            assert float(c.codes[0, c.pages(s)[t // c.page_size], 0, t % c.page_size, 0]) == value, (s, t)
    assert uses == c._uses
    assert sorted(c._free) == [p for p in range(c.num_pages) if uses[p] == 0]


@pytest.mark.parametrize("seed", range(6))
def test_account(plain, seed):
    """Random steps, forks, accepted paths, truncations, evictions and frees, with
    tokens written where a step says."""
    rng = random.Random(seed)
    c = ma.MorphoCache(40, 1, 16, 32, page_size=32)
    toks: dict[int, list[float]] = {}
    stamp = 0
    for _ in range(150):
        act = rng.choice(["new", "step", "step", "step", "drop", "fork", "accept", "truncate", "evict", "free"])
        before = {s: list(t) for s, t in toks.items()}
        try:
            if act == "new" and len(toks) < 6:
                toks[c.new()] = []
            elif act in ("step", "drop", "accept") and toks:
                seqs = rng.sample(sorted(toks), rng.randint(1, len(toks)))
                counts = [rng.choice([0, 1, 1, 5, 33, 70]) for _ in seqs]
                if max(counts) == 0:
                    continue
                step = c.step(seqs, counts)
                assert step.n == max(counts) and step.max_len == max(len(toks[s]) + k for s, k in zip(seqs, counts))
                assert step.lens.tolist() == [len(toks[s]) for s in seqs]
                new = []
                for b, (s, k) in enumerate(zip(seqs, counts)):
                    mine = []
                    for i in range(k):
                        stamp = stamp % 2000 + 1
                        at = len(toks[s]) + i
                        page = int(step.table[b, at // 32])
                        assert c._uses[page] == 1  # never a page that another sequence reads
                        c.codes[0, page, 0, at % 32] = stamp
                        mine.append(float(stamp))
                    new.append(mine)
                if act == "step":
                    c.commit(step)
                    for s, mine in zip(seqs, new):
                        toks[s] += mine
                elif act == "accept":
                    kept = [sorted(rng.sample(range(k), rng.randint(0, k))) for k in counts]
                    c.accept(step, kept)
                    for s, mine, k in zip(seqs, new, kept):
                        toks[s] += [mine[i] for i in k]
            elif act == "fork" and toks and len(toks) < 8:
                s = rng.choice(sorted(toks))
                f = c.fork(s)
                toks[f] = list(toks[s])
            elif act == "truncate" and toks:
                s = rng.choice(sorted(toks))
                k = rng.randint(0, len(toks[s]))
                c.truncate(s, k)
                del toks[s][k:]
            elif act == "evict" and toks:
                s = rng.choice(sorted(toks))
                kept = sorted(rng.sample(range(len(toks[s])), rng.randint(0, len(toks[s]))))
                c.evict(s, kept)
                toks[s] = [toks[s][i] for i in kept]
            elif act == "free" and toks and rng.random() < 0.5:
                s = rng.choice(sorted(toks))
                c.free(s)
                del toks[s]
        except RuntimeError as e:
            assert "cache is full" in str(e)
            toks = before  # and nothing has changed
        _check_account(c, toks)
    for s in list(toks):
        c.free(s)
    assert c.free_pages == 40


def test_a_stale_step_is_refused(plain):
    """A step whose sequences have changed commits nothing, of any of them."""
    c = ma.MorphoCache(8, 1, 16, 32)
    a, b = c.new(), c.new()
    c.commit(c.step([a, b], 70))
    for change in (lambda: c.commit(first), lambda: c.truncate(b, 65), lambda: c.evict(b, [0, 1]), lambda: c.free(b)):
        first, step = c.step([a], 1), c.step([a, b], 3)
        change()
        before = c.length(a), c.free_pages
        for again in (lambda: c.commit(step), lambda: c.accept(step, [[0], [1]])):
            with pytest.raises((RuntimeError, KeyError)):
                again()
        assert (c.length(a), c.free_pages) == before


def test_account_refusals(plain):
    c = ma.MorphoCache(2, 1, 16, 32)
    s = c.new()
    for call in (lambda: c.step([], 1), lambda: c.step([s, s], 1), lambda: c.step([s], 0), lambda: c.step([s], [1, 2]),
                 lambda: c.step([s], [-1]), lambda: c.truncate(s, 1), lambda: c.evict(s, [0])):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: c.length(7), lambda: c.free(7), lambda: c.fork(7), lambda: c.step([7], 1), lambda: c.pages(7)):
        with pytest.raises(KeyError):
            call()
    with pytest.raises(RuntimeError, match="cache is full"):
        c.step([s], 129)
    step = c.step([s], 5)
    for kept in ([], [[5]], [[1, 1]], [[2, 1]], [[-1]]):
        with pytest.raises(ValueError):
            c.accept(step, kept)
    c.accept(step, [[0, 4]])
    assert c.length(s) == 2


# ---------------------------------------------------------------- launch rules
PROGRAM = r'''
#include <cstdio>
#include "dispatch.h"
using namespace morpho;
int main() {
  long long what, a, b, c, d, m, dv;
  while (scanf("%lld %lld %lld %lld %lld %lld %lld", &what, &a, &b, &c, &d, &m, &dv) == 7) {
    if (what == 0) {
      const CacheAttnPlan p = cache_attn_plan((int)a, (int)b, (int)c, d, (int)m, (int)dv);
      printf("%d %d %d %d\n", p.pairs ? p.qt : p.qt + 10, p.qblocks, p.nsplit, p.split_keys);
    } else if (what == 1) {
      const CacheAppendShape p = cache_append_shape((int)a, (int)b);
      printf("%d %d %d 0\n", p.tokens, p.columns, cache_append_rows((int)c, (int)d, (int)b));
    } else {
      printf("%d 0 0 0\n", cache_compact_heads(a, (int)b, (int)c, (int)d));
    }
  }
}
'''


@pytest.fixture(scope="module")
def rules(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("cache_rules")
    (d / "rules.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT}/morphottention_amd/csrc",
                    str(d / "rules.cpp"), "-o", str(d / "rules")], check=True)

    def evaluate(rows):
        text = "".join(" ".join(map(str, (*r, 16, 64)[:7])) + "\n" for r in rows)
        out = subprocess.run([str(d / "rules")], input=text, capture_output=True, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return evaluate


def test_attention_rules(rules):
    """Every row lies in a block, every position below max_len in a piece, pieces are
    whole 128 keys, and the partial results stay small."""
    rng = random.Random(1)
    cases = [(rng.choice([1, 2, 7, 64, 500]), rng.choice([1, 3, 16, 32]), rng.choice([1, 16, 17, 64, 65, 1000, 5000]),
              rng.choice([1, 127, 512, 513, 768, 769, 5000, 131072, 2 ** 30])) for _ in range(400)]
    cases = [(*c, m, dv) for c in cases for m, dv in ((16, 32), (32, 64), (64, 64), (16, 128))]
    for (B, H, n, L, m, dv), (qt, qblocks, nsplit, keys) in zip(cases, rules([(0, *c) for c in cases])):
        pairs, qt = qt < 10, qt % 10
        assert pairs == (n <= 64)
        many = m == 64 or dv == 128 or B * H * -(-n // 128) > 1024
        assert qt == (0 if n <= 16 else 2 if n > 64 and many else 1)
        assert qblocks * (64 * qt if qt else 16) >= n > (qblocks - 1) * (64 * qt if qt else 16)
        assert keys % 128 == 0 and nsplit >= 1 and nsplit * keys >= L > (nsplit - 1) * keys
        assert nsplit * keys < 2 ** 31
        assert nsplit == 1 or B * H * n * nsplit <= 2 ** 20  # partial rows
        if pairs:
            assert nsplit <= 64
        else:
            assert nsplit == 1 or nsplit * B * H * qblocks <= 1024 // qt + B * H * qblocks
    # measured points: direct at short lengths, pieces for long ones and ragged batches
    assert [r[2] for r in rules([(0, 1, 8, 1, 100), (0, 64, 16, 1, 1000), (0, 64, 16, 1, 8192), (0, 1, 16, 1, 131071),
                                 (0, 16, 32, 48, 4048), (0, 4, 16, 1000, 5096)])] == [1, 1, 8, 64, 8, 1]


def test_append_rules(rules):
    rng = random.Random(2)
    cases = []
    for _ in range(300):
        B, n = rng.choice([1, 3, 16, 64]), rng.choice([1, 12, 63, 64, 65, 256, 1000])
        cases.append((B * n, 16 * rng.randint(3, 256), B, n))
    for (T, C, B, n), (tokens, columns, rows, _) in zip(cases, rules([(1, *c) for c in cases])):
        assert (tokens, columns) in ((0, 128), (1, 1), (2, 1), (2, 2), (4, 2), (4, 4))
        assert rows == n or (n >= 64 and rows % 8 == 0 and n + 7 <= rows <= n + 14)  # room for a shift of 7
    got = rules([(1, 1, 384, 1, 1), (1, 64, 1280, 64, 1), (1, 192, 4096, 16, 12), (1, 9003, 1536, 3, 3001),
                 (1, 2048, 4096, 8, 256)])
    assert [g[:2] for g in got] == [(1, 1), (2, 2), (4, 4), (0, 128), (0, 128)]
    assert got[3][2] == 3008 and got[4][2] == 256


def test_compact_rules(rules):
    assert [r[0] for r in rules([(2, 384, 16, 64, 9), (2, 1, 16, 64, 9), (2, 24, 2, 32, 1196), (2, 512, 16, 64, 100),
                                 (2, 4, 8, 64, 100), (2, 10000, 3, 128, 64), (2, 10000, 32, 32, 5)])] \
        == [8, 1, 0, 0, 0, 4, 32]
