"""Sharing as the cache finds it: forks of prompts large enough that what they have
in common is read once (64 MB of reading spared), stepped by the host's account and by
a loop, against the same sequences each reading its own.

Tolerance: both results are a rounding to fp16 (2^-11 of the value) and at most D away
from the exact one, so 2^-10 of the value and 2 D apart. D = (2 e ln 2 + 2^-20 + k 2^-28)
max |v| for k keys, as in test_gpu_cache, with a score's error e = S (2^-22 + m 2^-23) and
S = scale log2(e) sum_c |G_c (2 phi_c - 1) phi_c| <= scale log2(e) m for gates of 1."""

from __future__ import annotations

import math
import random

import pytest
import torch

import morphottention_amd as ma
from morphottention_amd import capi

pytestmark = pytest.mark.gpu
DEV = "cuda"
H, M, DV, P = 16, 16, 64, 64
D = H * DV


def _layer():
    torch.manual_seed(3)
    layer = ma.MorphoAttention(D, H, M, causal=True, dtype=torch.float16, device=DEV)
    return layer, layer.pack_cache_weights()


def _near(got, want, layer, cache, keys):
    S = layer.scale * math.log2(math.e) * M
    e = S * (2.0 ** -22 + M * 2.0 ** -23)
    far = (2 * e * math.log(2) + 2.0 ** -20 + keys * 2.0 ** -28) * cache.values.abs().max().float()
    got, want = got.float(), want.float()
    assert got.isfinite().all()
    over = (got - want).abs() - 2.0 ** -10 * torch.maximum(got.abs(), want.abs()) - 2 * far
    assert over.max() <= 0, over.max().item()


def _launched(call):
    """The call's result, and whether its attention read common keys once."""
    capi.timing_enable(True)
    try:
        capi.timing_read()
        out = call()
        torch.cuda.synchronize()
        return out, "cache_shared" in {name for name, _ in capi.timing_read()}
    finally:
        capi.timing_enable(False)


def _take(layer, w, cache, seqs, n, seed):
    """n new tokens of each, by the host's account."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    step = cache.step(seqs, n)
    out = layer.forward_cached(torch.randn(len(seqs), n, D, generator=g, device=DEV).half(), w, cache, step)
    cache.commit(step)
    return out


def _forest(layer, w, cache, seed):
    """Forks of two prompts, forks of a fork that has grown, and sequences of nobody, in any order."""
    a, b, alone = cache.new(), cache.new(), [cache.new() for _ in range(3)]
    _take(layer, w, cache, [a], 586, 1)
    _take(layer, w, cache, [b], 768, 2)
    _take(layer, w, cache, alone, 90, 3)
    first = [a] + [cache.fork(a) for _ in range(40)]
    second = [b] + [cache.fork(b) for _ in range(30)]
    _take(layer, w, cache, first[:1], 130, 4)
    deep = [cache.fork(a) for _ in range(8)]
    seqs = first + second + alone + deep
    random.Random(seed).shuffle(seqs)
    return seqs


@pytest.mark.parametrize("n", [1, 2, 5, 20, 64])
def test_steps_of_forks(n):
    """Single tokens, chains and pieces: each step's output with and without sharing, and
    the groups that the cache finds are groups of the same pages."""
    layer, w = _layer()
    cache = ma.MorphoCache(500, H, M, DV, page_size=P, device=DEV)
    with torch.no_grad():
        seqs = _forest(layer, w, cache, n)
        g = torch.Generator(device=DEV).manual_seed(n)
        for turn in range(3):
            x = torch.randn(len(seqs), n, D, generator=g, device=DEV).half()
            counts = n if turn else [1 + (7 * i) % n for i in range(len(seqs))]
            step = cache.step(seqs, counts, shared=True)
            s = step.shared
            starts, members, group = s.starts.tolist(), s.members.tolist(), s.group.tolist()
            assert len(members) >= 71 and max(s.pages.tolist()) >= 12
            for k, pages in enumerate(s.pages.tolist()):
                mine = members[starts[k]: starts[k + 1]]
                rows = step.table[mine, :pages]
                assert (rows == rows[0]).all() and all(group[m] == k for m in mine)
                assert all(cache.length(seqs[m]) >= pages * P for m in mine)
            y, shared = _launched(lambda: layer.forward_cached(x, w, cache, step))
            assert shared
            step.shared = None
            z, shared = _launched(lambda: layer.forward_cached(x, w, cache, step))  # stores the same again
            assert not shared
            _near(y, z, layer, cache, 1100)
            cache.commit(step)


@pytest.mark.parametrize("n", [1, 3, 20])
def test_a_loop_of_forks(n):
    """A loop's steps, eager and replayed, against the host's account without sharing: the
    same tokens are kept, so that every step's outputs can be compared."""
    layer, w = _layer()
    turns = 5
    rng = random.Random(n)
    g = torch.Generator(device=DEV).manual_seed(n)
    got, lengths = {}, {}
    with torch.no_grad():
        for how in ("host", "eager", "captured"):
            cache = ma.MorphoCache(500, H, M, DV, page_size=P, device=DEV)
            seqs = _forest(layer, w, cache, n)
            B = len(seqs)
            if how == "host":
                xs = torch.randn(turns, B, n, D, generator=g, device=DEV).half()
                kept = [[sorted(rng.sample(range(n), rng.randint(0, n))) for _ in range(B)] for _ in range(turns)]
                got[how] = []
                for x, keep in zip(xs, kept):
                    step = cache.step(seqs, n)
                    got[how].append(layer.forward_cached(x, w, cache, step))
                    cache.accept(step, keep)
                lengths[how] = [cache.length(s) for s in seqs]
                continue
            longest = max(cache.length(s) for s in seqs)
            with cache.loop(seqs, n, longest + turns * n, shared=True) as loop:
                x = torch.empty(B, n, D, dtype=torch.float16, device=DEV)
                keep = torch.empty(B, n, dtype=torch.int32, device=DEV)
                keep_lens = torch.empty(B, dtype=torch.int32, device=DEV)

                def load(turn):
                    x.copy_(xs[turn])
                    keep.copy_(torch.tensor([k + [-1] * (n - len(k)) for k in kept[turn]], dtype=torch.int32))
                    keep_lens.copy_(torch.tensor([len(k) for k in kept[turn]], dtype=torch.int32))

                def one():
                    step = loop.step()
                    y = layer.forward_cached(x, w, cache, step)
                    loop.accept(step, keep, keep_lens)
                    return y, step.new_lens
                run = one
                if how == "captured":
                    account = (loop.table, loop.held, loop.lens, loop.free_pages, loop.free_count)
                    state = [t.clone() for t in account]
                    load(0)
                    side = torch.cuda.Stream()
                    side.wait_stream(torch.cuda.current_stream())
                    with torch.cuda.stream(side):
                        one()
                    torch.cuda.current_stream().wait_stream(side)
                    graph = torch.cuda.CUDAGraph()
                    with torch.cuda.graph(graph):
                        static = one()
                    for t, v in zip(account, state):
                        t.copy_(v)

                    def run():
                        graph.replay()
                        return static
                got[how] = []
                for turn in range(turns):
                    load(turn)
                    if how == "eager":
                        (y, granted), shared = _launched(run)
                        assert shared
                    else:
                        y, granted = run()
                        torch.cuda.synchronize()
                    assert granted.tolist() == [n] * B
                    got[how].append(y.clone())
            lengths[how] = [cache.length(s) for s in seqs]
            for y, z in zip(got[how], got["host"]):
                _near(y, z, layer, cache, 1100)
        for y, z in zip(got["captured"], got["eager"]):
            assert torch.equal(y, z)
    assert lengths["host"] == lengths["eager"] == lengths["captured"]
