"""A decoding loop's operators without a GPU: their oracle, what the entry points
refuse, fakes, what sequences have in common, and a loop's account."""

from __future__ import annotations

import ctypes
import os
import random
import shutil
import subprocess

import numpy as np
import pytest
import torch

import morphottention_amd as ma
from morphottention_amd import cache as cache_module
from morphottention_amd import capi
from oracle import loop_oracle

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000  # a pointer that no refused call follows
INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3


def _message():
    return capi.lib().morpho_last_error()


# ---------------------------------------------------------------- the oracle
@pytest.mark.parametrize("tree,drawn", [(None, True), (None, False), ([1, 3, 5, 9], True), ([1, 3, 5, 9], False),
                                        ([1, 3, 7, 9], True)])
def test_verified_tokens_have_the_targets_distribution(tree, drawn):
    """The first token behind the root, over many draws of drafts and numbers, is
    distributed as the target says: each count within 5 sigma of its mean."""
    rng = np.random.default_rng(7)
    V, n, tries = 5, 4, 20000
    logits, draft = rng.normal(size=(n, V)) * 1.2, rng.normal(size=(n - 1, V)) * 1.2
    p = loop_oracle.distribution(logits[0], 1.0)
    parent = loop_oracle.parents_of(tree, n)
    # every token has the same rows of its own, so that only the root's decisions matter here
    seen = np.zeros(V)
    q = [loop_oracle.distribution(d, 1.0) for d in draft]
    for _ in range(tries):
        tokens = [0] + [int(rng.choice(V, p=q[parent[i]])) if drawn else i % V for i in range(1, n)]
        path, token = loop_oracle.verify(logits, tokens, rng.random(n).tolist(), tree=tree,
                                         draft_logits=draft if drawn else None)
        seen[tokens[path[1]] if len(path) > 1 else token] += 1
    sigma = np.sqrt(tries * p * (1 - p))
    assert (np.abs(seen - tries * p) <= 5 * sigma).all(), (seen / tries, p)


def test_oracle_edges():
    row = np.array([[0.0, np.nan, -np.inf, 1.0], [np.inf, 0.0, np.inf, 5.0]])
    assert loop_oracle.distribution(row[0], 1.0)[1:3].tolist() == [0, 0]
    assert loop_oracle.distribution(row[1], 1.0).tolist() == [0.5, 0, 0.5, 0]
    assert loop_oracle.verify(np.full((1, 3), -np.inf), [0], [0.5]) == ([0], -1)
    assert loop_oracle.verify(row, [0, 3], [0.9, 0.0], count=0) == ([], -1)
    assert loop_oracle.verify(row, [0, 3], [0.2, 0.99], temperature=0.0) == ([0, 1], 0)
    t = loop_oracle.plan(np.full((2, 2), -1), [0, 0], [0, 0], [7, 8, 9], 3, 40, [40, 33], 32)
    assert t[0].tolist() == [[9, 8], [-1, -1]] and t[3] == 1 and t[4] == [40, 0]


# ---------------------------------------------------------------- refusals
def _pool(**kw):
    d = dict(codes=P, values=P, layers=1, pages=4, H=2, cube_m=16, head_dim_v=64, page_size=64) | kw
    return capi.Cache(*(d[k] for k, _ in capi.Cache._fields_))


def _shared(pool=None, members=P, starts=P, group=P, pages=P, count=2, groups=1, max_prefix=64, max_rest=64, phi=P,
            gq=P, gk=P, table=P, lens=P, new_lens=None, tree=None, out=P, lse=P, B=2, n=1, seq_pages=4, scale=1.0,
            mode=1, ws=P, ws_bytes=1 << 30, none=False):
    s = capi.SharedPrefix(members, starts, group, pages, count, groups, max_prefix, max_rest)
    return capi.lib().morpho_cache_shared_attention(phi, gq, gk, ctypes.byref(pool or _pool()), table, lens, new_lens,
                                                    tree, None if none else ctypes.byref(s), out, lse, B, n, seq_pages,
                                                    scale, mode, ws, ws_bytes, None)


def _plan(table=P, held=P, lens=P, new_lens=None, free=P, count=P, room=8, granted=P, slots=P, B=2, n=4, seq_pages=4,
          page_size=64, ws=None, ws_bytes=0):
    return capi.lib().morpho_cache_plan(table, held, lens, new_lens, free, count, room, granted, slots, B, n, seq_pages,
                                        page_size, ws, ws_bytes, None)


def _verify(p=P, q=None, type=0, tokens=P, uniform=P, tree=None, new_lens=None, keep=P, keep_lens=P, token=P, B=2, n=4,
            vocab=100, temperature=1.0, ws=P, ws_bytes=1 << 30, none=False):
    rows = capi.Logits(p, n * vocab, vocab)
    draft = capi.Logits(q, n * vocab, vocab)
    return capi.lib().morpho_verify_drafts(None if none else ctypes.byref(rows), ctypes.byref(draft), type, tokens,
                                           uniform, tree, new_lens, keep, keep_lens, token, B, n, vocab, temperature,
                                           ws, ws_bytes, None)


LONG = {"max_prefix": 1 << 20, "seq_pages": 1 << 15}  # enough in common to be worth it


@pytest.mark.parametrize("call,kw,status,text", [
    (_shared, {"none": True}, INVALID, b"Null"), (_shared, {"pool": _pool(cube_m=24)}, UNSUPPORTED, b"cube_m"),
    (_shared, {"pool": _pool(layers=2)}, INVALID, b"one layer"), (_shared, {"pool": _pool(codes=P + 4)}, INVALID, b"16-byte"),
    (_shared, {"count": 0}, INVALID, b"members"), (_shared, {"count": 3}, INVALID, b"members"),
    (_shared, {"groups": 0}, INVALID, b"groups"), (_shared, {"groups": 3}, INVALID, b"groups"),
    (_shared, {"max_prefix": 0}, INVALID, b"max_prefix"), (_shared, {"max_rest": -1}, INVALID, b"max_rest"),
    (_shared, {"n": 65}, UNSUPPORTED, b"64 new"), (_shared, {"scale": float("inf")}, INVALID, b"finite"),
    (_shared, {"mode": 4}, INVALID, b"mode"), (_shared, {"mode": 3, "tree": P}, INVALID, b"own bit"),
    (_shared, {"members": None}, INVALID, b"Null"), (_shared, {"starts": None}, INVALID, b"Null"),
    (_shared, {"group": None}, INVALID, b"Null"), (_shared, {"pages": None}, INVALID, b"Null"),
    (_shared, {"phi": None}, INVALID, b"Null"), (_shared, {"lse": None}, INVALID, b"Null"),
    (_shared, {"group": P + 2}, INVALID, b"4-byte"), (_shared, {"starts": P + 1}, INVALID, b"4-byte"),
    (_shared, {"tree": P + 4}, INVALID, b"8-byte"), (_shared, {"out": P + 8}, INVALID, b"16-byte"),
    (_shared, LONG | {"ws": None}, WORKSPACE, b"needs"), (_shared, LONG | {"ws_bytes": 64}, WORKSPACE, b"needs"),
    (_shared, LONG | {"ws": P + 16}, WORKSPACE, b"256-byte"), (_shared, {"B": 0}, INVALID, b"Invalid dimensions"),
    (_shared, {"B": 2 ** 40, "n": 2 ** 40}, INVALID, b"too large"),
    (_plan, {"table": None}, INVALID, b"Null"), (_plan, {"held": None}, INVALID, b"Null"),
    (_plan, {"lens": None}, INVALID, b"Null"), (_plan, {"free": None}, INVALID, b"Null"),
    (_plan, {"count": None}, INVALID, b"Null"), (_plan, {"granted": None}, INVALID, b"Null"),
    (_plan, {"slots": None}, INVALID, b"Null"), (_plan, {"slots": P + 4}, INVALID, b"8-byte"),
    (_plan, {"held": P + 2}, INVALID, b"4-byte"), (_plan, {"count": P + 1}, INVALID, b"4-byte"),
    (_plan, {"page_size": 48}, UNSUPPORTED, b"page_size"), (_plan, {"B": 0}, INVALID, b"Invalid dimensions"),
    (_plan, {"n": 0}, INVALID, b"Invalid dimensions"), (_plan, {"room": -1}, INVALID, b"Invalid dimensions"),
    (_plan, {"room": 2 ** 31}, INVALID, b"Invalid dimensions"), (_plan, {"seq_pages": 2 ** 24 + 1}, INVALID, b"2^30"),
    (_plan, {"B": 2 ** 12, "n": 2 ** 11}, INVALID, b"too large"), (_plan, {"B": 2 ** 40, "n": 2 ** 40}, INVALID, b"too large"),
    (_plan, {"B": 2000}, WORKSPACE, b"needs"), (_plan, {"B": 2000, "ws": P + 16, "ws_bytes": 1 << 20}, WORKSPACE, b"256-byte"),
    (_verify, {"none": True}, INVALID, b"Null"), (_verify, {"p": None}, INVALID, b"Null"),
    (_verify, {"tokens": None}, INVALID, b"Null"), (_verify, {"uniform": None}, INVALID, b"Null"),
    (_verify, {"keep": None}, INVALID, b"Null"), (_verify, {"keep_lens": None}, INVALID, b"Null"),
    (_verify, {"token": None}, INVALID, b"Null"), (_verify, {"type": 3}, UNSUPPORTED, b"type"),
    (_verify, {"type": -1}, UNSUPPORTED, b"type"), (_verify, {"n": 65}, UNSUPPORTED, b"64 drafted"),
    (_verify, {"n": 0}, INVALID, b"Invalid dimensions"), (_verify, {"B": 0}, INVALID, b"Invalid dimensions"),
    (_verify, {"vocab": 0}, INVALID, b"Invalid dimensions"), (_verify, {"vocab": 4000001}, INVALID, b"vocab"),
    (_verify, {"B": 2 ** 40}, INVALID, b"too large"), (_verify, {"B": 2 ** 22, "vocab": 100000}, INVALID, b"too large"),
    (_verify, {"temperature": -1.0}, INVALID, b"temperature"), (_verify, {"temperature": 1e-5}, INVALID, b"temperature"),
    (_verify, {"temperature": float("nan")}, INVALID, b"temperature"), (_verify, {"temperature": float("inf")}, INVALID, b"temperature"),
    (_verify, {"p": P + 1}, INVALID, b"aligned"), (_verify, {"p": P + 2, "type": 2}, INVALID, b"aligned"),
    (_verify, {"q": P + 1}, INVALID, b"aligned"), (_verify, {"tokens": P + 4}, INVALID, b"8-byte"),
    (_verify, {"uniform": P + 2}, INVALID, b"4-byte"), (_verify, {"tree": P + 4}, INVALID, b"8-byte"),
    (_verify, {"ws": None}, WORKSPACE, b"needs"), (_verify, {"ws_bytes": 32}, WORKSPACE, b"needs"),
    (_verify, {"ws": P + 32}, WORKSPACE, b"256-byte"),
])
def test_refusals(call, kw, status, text):
    assert call(**kw) == status
    assert text in _message()


def test_workspace_sizes():
    lib = capi.lib()
    assert lib.morpho_cache_plan_workspace_size(64, 12) == 0 and lib.morpho_cache_plan_workspace_size(0, 1) == 0
    assert lib.morpho_cache_plan_workspace_size(2000, 1) >= 16 + 2000 * 16
    assert lib.morpho_cache_plan_workspace_size(1, 100000) > 0
    size = lib.morpho_verify_workspace_size
    assert size(2, 4, 100, 0, 1, 0, 1.0) > 0 and size(2, 65, 100, 0, 1, 0, 1.0) == 0
    assert size(2, 4, 100, 0, 1, 0, -1.0) == 0 and size(2, 4, 100, 5, 1, 0, 1.0) == 0
    size = lib.morpho_cache_shared_attention_workspace_size
    pool = _pool()
    assert size(ctypes.byref(pool), 2, 1, 4, 2, 1, 64, 64) == 0  # not worth it: one kernel without pieces
    assert size(ctypes.byref(pool), 2, 1, 1 << 15, 2, 1, 1 << 20, 64) >= 2 * 2 * 2 * (64 * 4 + 16)
    assert size(ctypes.byref(pool), 2, 65, 1 << 15, 2, 1, 1 << 20, 64) == 0
    # no longer than the table
    assert size(ctypes.byref(pool), 2, 1, 1 << 15, 2, 1, 1 << 40, 1 << 40) == \
        size(ctypes.byref(pool), 2, 1, 1 << 15, 2, 1, 1 << 21, 1 << 21)


def test_python_refusals():
    t = torch.zeros(1)
    with pytest.raises(ValueError, match="max_prefix"):
        ma.morpho_cache_attention(t, t, t, t, t, t, t, shared=ma.SharedPrefix(t, t, t, t, max_prefix=-1))
    for groups, pages in (([], []), ([[0]], [1, 2]), ([[0], []], [1, 1]), ([[0, 0]], [1]), ([[0, 2]], [1]), ([[-1]], [1]),
                          ([[0], [0]], [1, 1]), ([[0]], [-1])):
        with pytest.raises(ValueError):
            ma.SharedPrefix.of(groups, pages, 2)
    c = ma.MorphoCache(8, 1, 16, 32, page_size=32)
    a = c.new()
    for bad in (dict(seqs=[], n=1, room=9), dict(seqs=[a, a], n=1, room=9), dict(seqs=[a], n=0, room=9),
                dict(seqs=[a], n=10, room=9), dict(seqs=[a], n=1, room=9, pages=-1)):
        with pytest.raises(ValueError):
            c.loop(**bad)
    with pytest.raises(RuntimeError, match="full"):
        c.loop([a], 1, 9, pages=9)
    assert c.free_pages == 8 and c.length(a) == 0


def test_ops_need_gpu_tensors():
    """CPU tensors have no kernel: an error, not a fallback."""
    ints = torch.zeros((1, 1), dtype=torch.int32)
    with pytest.raises(NotImplementedError):
        ma.morpho_cache_plan(ints, ints[0], ints[0], ints[0], ints[0], 1)
    with pytest.raises(NotImplementedError):
        ma.morpho_verify_drafts(torch.zeros(1, 1, 5), torch.zeros((1, 1), dtype=torch.int64), torch.zeros(1, 1))


def test_fakes():
    from torch._subclasses.fake_tensor import FakeTensorMode
    with FakeTensorMode():
        f = lambda *s, t=torch.float16: torch.empty(s, dtype=t, device="cuda")  # noqa: E731
        i = lambda *s: f(*s, t=torch.int32)  # noqa: E731
        shared = ma.SharedPrefix(i(2), i(2), i(2), i(1))
        out, lse = ma.morpho_cache_attention(f(2, 5, 3, 16), f(3, 16), f(3, 16), f(9, 3, 64, 16), f(9, 3, 8, 32, 8), i(2, 4),
                                             i(2), shared=shared)
        assert out.shape == (2, 5, 96) and out.dtype == torch.float16 and lse.shape == (6, 5) and lse.dtype == torch.float32
        granted, slots = ma.morpho_cache_plan(i(2, 4), i(2), i(2), i(9), i(1), 7, page_size=32)
        assert granted.shape == (2,) and granted.dtype == torch.int32
        assert slots.shape == (2, 7) and slots.dtype == torch.int64
        keep, keep_lens, token = ma.morpho_verify_drafts(f(2, 5, 99, t=torch.bfloat16), f(2, 5, t=torch.int64),
                                                         f(2, 5, t=torch.float32))
        assert keep.shape == (2, 5) and keep_lens.shape == (2,) and token.shape == (2,)
        assert keep.dtype == keep_lens.dtype == torch.int32 and token.dtype == torch.int64


# ---------------------------------------------------------------- launch rules
RULES = r'''
#include <cstdio>
#include "dispatch.h"
using namespace morpho;
int main() {
  for (long long B : {1, 4, 64, 300, 65536})
    for (long long H : {1, 16, 128})
      for (long long n : {1, 7, 16, 17, 64})
        for (long long G : {1LL, B})
          for (long long len : {32LL, 512LL, 8192LL, 65536LL, 1LL << 30})
            for (int dv : {32, 64, 128}) {
              if (B * n > (1 << 22) || B * n * H > (1 << 23)) continue;
              const CacheSharedPlan p = cache_shared_plan(B, H, n, B, G, len, len, 16, dv);
              const long long rows = B * H * n, parts = p.np + p.rest.nsplit;
              if (p.apart && p.rest.split_keys < 1) printf("apart");
              if (p.np < 1 || p.split_keys % 128 || (long long)p.np * p.split_keys < len ||
                  (long long)p.rblocks * (p.qt ? 16 * p.qt : 64) < B * n + ((p.qt ? 16 * p.qt : 64) - 1) * (G > 1 ? 1 : 0) ||
                  (p.np > 1 && rows * p.np > (1 << 20) + rows) || (!p.apart && rows > (1 << 20) && parts > 4))
                printf("B%lld H%lld n%lld G%lld len%lld: np %d of %d, rblocks %d of 16 x %d\n", B, H, n, G, len, p.np,
                       p.split_keys, p.rblocks, p.qt);
            }
  for (long long rows : {1LL, 9LL, 700LL, 100000LL})
    for (int vocab : {1, 7, 255, 2048, 32000, 50001, 128000, 1000003, kVerifyMaxVocab})
      for (int size : {2, 4})
        for (int kind = 0; kind < 8; ++kind) {
          const VerifyPlan p = verify_plan(rows, 7, vocab, size, kind & 1, kind & 2, kind & 4);
          // a row that starts at the last element of 16 bytes has all its elements in the chunks
          if ((p.pieces != 1 && p.pieces != 4) || p.chunk != 64 * 16 / size * p.pieces ||
              (long long)p.chunks * p.chunk < vocab + 16 / size - 1 || p.chunks > kVerifyMaxChunks || p.rounds < 0 ||
              ((kind & 4) && p.rounds))
            printf("rows %lld vocab %d size %d: %d chunks of %d\n", rows, vocab, size, p.chunks, p.chunk);
        }
}
'''


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_launch_rules(tmp_path):
    (tmp_path / "rules.cpp").write_text(RULES)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", f"-I{ROOT}/morphottention_amd/csrc",
                    str(tmp_path / "rules.cpp"), "-o", str(tmp_path / "rules")], check=True)
    assert subprocess.run([str(tmp_path / "rules")], capture_output=True, text=True, check=True).stdout == ""


# ---------------------------------------------------------------- what is in common
def test_groups_spare_the_most_pages():
    rows = [[1, 2, 3, 10], [1, 2, 3, 11], [1, 2, 20], [7, 8], [7, 8], [9]]
    full = [4, 4, 3, 2, 2, 1]
    # 1, 2 in three rows spare 4 pages, 1, 2, 3 in two of them 3
    assert sorted(cache_module._groups(rows, full)) == [([0, 1, 2], 2), ([3, 4], 2)]
    rows[0:2] = [[1, 2, 3, 4, 5, 10], [1, 2, 3, 4, 5, 11]]
    full[0:2] = [6, 6]
    assert sorted(cache_module._groups(rows, full)) == [([0, 1], 5), ([3, 4], 2)]
    assert cache_module._groups(rows, [0] * 6) == [] and cache_module._groups([[1], [2]], [1, 1]) == []
    assert cache_module._groups([[1, 2], [1, 2]], [2, 1]) == [([0, 1], 1)]  # the other's second page is not full


def test_groups_of_forks_of_forks():
    """Each row a fork of the one before, a page longer: as deep as there are rows."""
    rows = [list(range(min(i + 1, 1499))) + [10000 + 2000 * i + j for j in range(3)] for i in range(1500)]
    groups = cache_module._groups(rows, [len(r) for r in rows])
    members = [b for k, _ in groups for b in k]
    assert groups and len(set(members)) == len(members)
    for k, common in groups:
        assert len(k) > 1 and common > 0 and all(rows[b][:common] == rows[k[0]][:common] for b in k)


def test_shared_prefix_of():
    s = ma.SharedPrefix.of([[3, 0], [2]], [5, 1], 4)
    assert s.members.tolist() == [3, 0, 2] and s.starts.tolist() == [0, 2, 3] and s.group.tolist() == [0, -1, 1, 0]
    assert s.pages.tolist() == [5, 1] and all(t.dtype == torch.int32 for t in (s.members, s.starts, s.group, s.pages))


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


def _plain_plan(table, held, lens, free_pages, free_count, n, *, new_lens=None, page_size=64):
    got = loop_oracle.plan(table.numpy(), held.tolist(), lens.tolist(), free_pages.tolist(), int(free_count), n,
                           None if new_lens is None else new_lens.tolist(), page_size)
    table.copy_(torch.from_numpy(got[0]))
    held.copy_(torch.tensor(got[1]))
    free_pages.copy_(torch.tensor(got[2]))
    free_count.fill_(got[3])
    return torch.tensor(got[4], dtype=torch.int32), torch.from_numpy(got[5])


@pytest.fixture
def plain(monkeypatch):
    monkeypatch.setattr(cache_module, "morpho_cache_copy_pages", _plain_copy)
    monkeypatch.setattr(cache_module, "morpho_cache_compact", _plain_compact)
    monkeypatch.setattr(cache_module, "morpho_cache_plan", _plain_plan)


def test_steps_know_what_forks_share(plain):
    c = ma.MorphoCache(60, 1, 16, 32, page_size=32)
    a = c.new()
    c.commit(c.step([a], 100))
    b, d, e = c.fork(a), c.fork(a), c.new()
    assert c.step([a, e], 1, shared=True).shared is None and c.step([a, b], 1).shared is None
    step = c.step([e, d, a, b], [5, 1, 2, 40], shared=True)
    s = step.shared
    assert s.members.tolist() == [1, 2, 3] and s.starts.tolist() == [0, 3] and s.group.tolist() == [-1, 0, 0, 0]
    assert s.pages.tolist() == [3] and s.max_prefix == 96 and s.max_rest == 44
    rows = step.table[1:, :3]
    assert (rows == rows[0]).all()


@pytest.mark.parametrize("seed", range(6))
def test_loop_account(plain, seed):
    """Loops among the cache's other calls: every sequence reads back its own tokens,
    use counts and the free list agree."""
    rng = random.Random(seed)
    c = ma.MorphoCache(60, 1, 16, 32, page_size=32)
    toks: dict[int, list[float]] = {}
    stamp = 0

    def write(page, at):
        nonlocal stamp
        stamp = stamp % 2000 + 1
        c.codes[0, page, 0, at % 32] = stamp
        return float(stamp)

    for _ in range(25):
        if len(toks) < 6:
            toks[c.new()] = []
        s = rng.choice(sorted(toks))
        k = rng.choice([1, 31, 33, 64])
        if c.free_pages > 4:
            step = c.step([s], k)
            toks[s] += [write(int(step.table[0, (len(toks[s]) + i) // 32]), len(toks[s]) + i) for i in range(k)]
            c.commit(step)
        if rng.random() < 0.5 and len(toks) < 8 and c.free_pages > 2:
            f = c.fork(s)
            toks[f] = list(toks[s])
        seqs = rng.sample(sorted(toks), rng.randint(1, len(toks)))
        n = rng.choice([1, 5, 40])
        stale = c.step([seqs[0]], 1) if c.free_pages else None
        room = max(len(toks[q]) for q in seqs) + n + rng.choice([0, 50, 100])
        if c.free_pages < len(seqs):
            c.free(s)
            del toks[s]
            continue
        with c.loop(seqs, n, room, pages=rng.choice([None, None, 2]) if c.free_pages > 2 + len(seqs) else 0,
                    shared=rng.random() < 0.5) as loop:
            refused = [lambda: c.length(seqs[0]), lambda: c.fork(seqs[0]), lambda: c.step(seqs, 1),
                       lambda: c.truncate(seqs[0], 0), lambda: c.free(seqs[0]), lambda: c.evict(seqs[0], []),
                       lambda: c.loop(seqs, 1, 500)] + ([lambda: c.commit(stale)] if stale is not None else [])
            for call in refused:
                with pytest.raises(RuntimeError, match="in a loop"):
                    call()
            for _ in range(rng.randint(0, 4)):
                news = torch.tensor([rng.randint(0, n) for _ in seqs], dtype=torch.int32) if rng.random() < 0.4 else None
                step = loop.step(news)
                old = loop.lens.tolist()
                mine = []
                for b in range(len(seqs)):
                    new = []
                    for i in range(int(step.new_lens[b])):
                        page = int(loop.table[b, (old[b] + i) // 32])
                        assert c._uses[page] == 1 and int(loop.slots[b, i]) == page * 32 + (old[b] + i) % 32
                        new.append(write(page, old[b] + i))
                    mine.append(new)
                act = rng.choice(["all", "some", "none"])
                if act == "all":
                    loop.accept(step)
                    for q, new in zip(seqs, mine):
                        toks[q] += new
                elif act == "some":
                    kept = [sorted(rng.sample(range(len(new)), rng.randint(0, len(new)))) for new in mine]
                    loop.accept(step, torch.tensor([k + [-1] * (n - len(k)) for k in kept], dtype=torch.int32),
                                torch.tensor([len(k) for k in kept], dtype=torch.int32))
                    for q, new, k in zip(seqs, mine, kept):
                        toks[q] += [new[i] for i in k]
        uses = [0] * c.num_pages
        for q, mine in toks.items():
            assert c.length(q) == len(mine)
            for p in c.pages(q):
                uses[p] += 1
            for t, value in enumerate(mine):
                assert float(c.codes[0, c.pages(q)[t // 32], 0, t % 32, 0]) == value, (q, t)
        assert uses == c._uses
        assert sorted(c._free) == [p for p in range(c.num_pages) if uses[p] == 0]


def test_loop_refusals(plain):
    c = ma.MorphoCache(20, 1, 16, 32, page_size=32)
    other = ma.MorphoCache(20, 1, 16, 32, page_size=32)
    a = c.new()
    loop = c.loop([a], 2, 64)
    first = loop.step()
    x = torch.zeros(1, 2, 32)
    c._check(first, x)
    second = loop.step()
    c._check(second, x)
    with pytest.raises(RuntimeError, match="another step"):
        c._check(first, x)
    with pytest.raises(RuntimeError, match="another step"):
        loop.accept(first)
    with pytest.raises(RuntimeError, match="another cache"):
        other._check(second, x)
    with pytest.raises(ValueError, match="rows of"):
        c._check(second, x[:, :1])
    with pytest.raises(ValueError, match="go together"):
        loop.accept(second, torch.zeros((1, 2), dtype=torch.int32))
    for call in (c.commit, c.drop, lambda s: c.accept(s, [[0]])):
        with pytest.raises(RuntimeError, match="loop"):
            call(second)
    # counts that cannot be: no sequence becomes shorter, none gets more than it was granted
    for k in (-7, 0):
        loop.accept(loop.step(), torch.zeros((1, 2), dtype=torch.int32), torch.tensor([k], dtype=torch.int32))
        assert loop.lens.tolist() == [0]
    second = loop.step()
    loop.accept(second, torch.tensor([[0, 1]], dtype=torch.int32), torch.tensor([9], dtype=torch.int32))
    for call in (lambda: loop.accept(second), lambda: c._check(second, x)):
        with pytest.raises(RuntimeError, match="taken the step's tokens"):
            call()
    assert loop.lens.tolist() == [2]
    loop.close()
    loop.close()
    assert c.length(a) == 2 and c.free_pages == 19
    for call in (loop.step, lambda: loop.accept(second), lambda: c._check(second, x)):
        with pytest.raises(RuntimeError, match="closed"):
            call()
    # verified tensors, read from the device
    step = c.step([a], 5)
    c.accept(step, (torch.tensor([[0, 3, -1, -1, -1]], dtype=torch.int32), torch.tensor([2], dtype=torch.int32)))
    assert c.length(a) == 4


def test_loops_leave_the_cache_as_it_was_when_they_cannot_start(plain):
    c = ma.MorphoCache(4, 1, 16, 32, page_size=32)
    a = c.new()
    c.commit(c.step([a], 40))
    b = c.fork(a)  # a's second page is not full: b has a copy
    with pytest.raises(RuntimeError, match="full"):
        c.loop([a, b], 1, 41, pages=2)
    assert c.free_pages == 1 and c.length(a) == c.length(b) == 40
    with c.loop([a, b], 1, 41) as loop:
        assert loop.free_count.tolist() == [0]
    assert c.free_pages == 1 and len(c.pages(a)) == 2


def test_a_loop_that_cannot_start_leaves_no_step_with_pages_of_others(plain, monkeypatch):
    """A step that was made before still owns its pages after the failure, or is refused."""
    c = ma.MorphoCache(6, 1, 16, 32, page_size=32)
    a, b = c.new(), c.new()
    step = c.step([a], 64)
    for pages in (7, 100):
        with pytest.raises(RuntimeError, match=f"{pages} pages needed, 6 of 6 free"):
            c.loop([a], 1, 200, pages=pages)
    other = c.step([b], 64)
    assert not set(step.table[0].tolist()) & set(other.table[0].tolist())
    c.commit(step)
    assert c.length(a) == 64 and len(c.pages(a)) == 2

    late = c.step([a], 64)
    ints = c._ints

    def fails(rows):
        if rows == [64]:  # the lengths, after tables are built
            raise RuntimeError("out of memory")
        return ints(rows)
    with monkeypatch.context() as m, pytest.raises(RuntimeError, match="out of memory"):
        m.setattr(c, "_ints", fails)
        c.loop([a], 1, 128)
    assert c.free_pages == 2 and c.length(a) == 64
    again = c.step([b], 128)  # takes what the failed loop and the step had
    assert len(set(again.table[0].tolist())) == 4
    with pytest.raises(RuntimeError, match="changed"):
        c.commit(late)
    with pytest.raises(RuntimeError, match="changed"):
        c._check(late, torch.zeros(1, 64, 32))
    assert c.length(a) == 64 and len(c.pages(a)) == 2


def test_a_loop_takes_what_its_sequences_had_claimed(plain):
    c = ma.MorphoCache(6, 1, 16, 32, page_size=32)
    a = c.new()
    step = c.step([a], 160)
    with c.loop([a], 1, 200, pages=6) as loop:
        assert loop.free_count.tolist() == [6]
    with pytest.raises(RuntimeError, match="changed"):
        c.commit(step)
    assert c.free_pages == 6


@pytest.mark.parametrize("room", [32, 40, 41, 44, 63, 64])
def test_no_sequence_of_a_loop_gets_more_tokens_than_its_room(plain, room):
    """Also where its last page has places behind it: all of a step's new tokens, or none."""
    c = ma.MorphoCache(12, 1, 16, 32, page_size=32)
    a, b = c.new(), c.new()
    c.commit(c.step([b], 3))
    n, want = 5, [0, 3]
    with c.loop([a, b], n, room) as loop:
        for news in [None] * 14 + [[9, -3], [2, 1], [1, 1], [1, 2], [1, 1], [1, 1], [1, 1]]:
            step = loop.step(None if news is None else torch.tensor(news, dtype=torch.int32))
            asked = [n, n] if news is None else [min(max(k, 0), n) for k in news]
            got = [k if have + k <= room else 0 for k, have in zip(asked, want)]
            assert step.new_lens.tolist() == got
            for b_, k in enumerate(got):
                assert (loop.slots[b_, :k] >= 0).all() and (loop.slots[b_, k:] == -1).all()
            loop.accept(step)
            want = [have + k for have, k in zip(want, got)]
            assert loop.lens.tolist() == want
        assert want[0] <= room and want[1] <= room and max(want) > room - 5
    assert c.length(a) == want[0] and c.length(b) == want[1]


@pytest.mark.parametrize("room", [40, 64])
def test_a_loops_counts_are_one_for_each_sequence(plain, room):
    c = ma.MorphoCache(6, 1, 16, 32, page_size=32)
    with c.loop([c.new(), c.new()], 5, room) as loop:
        for bad in (torch.ones(1, dtype=torch.int32), torch.ones((1, 2), dtype=torch.int32), torch.ones(2, dtype=torch.int64)):
            with pytest.raises(ValueError, match="new_lens"):
                loop.step(bad)
        assert loop.step(torch.tensor([1, 5], dtype=torch.int32)).new_lens.tolist() == [1, 5]


@pytest.mark.parametrize("hints", [{"max_prefix": 0}, {"max_rest": 0}, {"max_rest": -5}, {"max_prefix": 64, "max_rest": 0}])
def test_hints_that_are_not_positive(hints):
    t = torch.zeros(1)
    with pytest.raises(ValueError, match="positive"):
        ma.morpho_cache_attention(t, t, t, t, t, t, t, shared=ma.SharedPrefix(t, t, t, t, **hints))


def test_powers_of_the_verification():
    """Its table holds the doubles next to 2^(i / 256), less i 2^44, and its cubic is 2^(r / 256)
    to 2^-45 for |r| <= 1/2."""
    import math
    import re
    import struct
    from decimal import Decimal, localcontext
    with open(f"{ROOT}/morphottention_amd/csrc/kernels_verify.hip") as f:
        src = f.read()
    table = [int(x, 16) for x in re.findall(r"0x[0-9a-f]{16}", src[src.index("kExp2Table[kTable] = {"):src.index("};")])]
    cubic = [float.fromhex(x) for x in re.findall(r"0x1\.[0-9a-f]{13}p-\d+", src[src.index("double exp2_256("):])[:4]]
    assert len(table) == 256
    with localcontext() as c:
        c.prec = 60
        ln2 = Decimal(2).ln()
        for i, entry in enumerate(table):
            bits = struct.unpack("<Q", struct.pack("<d", float((ln2 * i / 256).exp())))[0]
            assert bits - (i << 44) == entry, i
        for k in range(-200, 201):
            r, y = Decimal(k) / 400, Decimal(0)
            for a in cubic:
                y = y * r + Decimal(a)
            assert abs(y / (ln2 * r / 256).exp() - 1) <= Decimal(math.ldexp(1, -45)), k
