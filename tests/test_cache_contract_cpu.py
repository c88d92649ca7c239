"""What the paged cache promises for calls that its documentation allows but that are
easy to get wrong, without a GPU."""

from __future__ import annotations

import copy
import dataclasses
import os
import random
import shutil
import subprocess

import pytest
import torch

import morphottention_amd as ma
from morphottention_amd import autograd
from morphottention_amd import cache as cache_module

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


# ---------------------------------------------------------------- compaction in place
COMPACT = r'''
#include <cstdio>
#include <vector>
#include "dispatch.h"
// A row's tokens 0 .. n - 1 moved as a workgroup moves them: batches in order,
// each read whole before it is written.
int main() {
  int n, batch, count;
  while (scanf("%d %d %d", &n, &batch, &count) == 3) {
    std::vector<int> keep(count), token(n), got(count);
    for (int& k : keep) scanf("%d", &k);
    for (int i = 0; i < n; ++i) token[i] = i;
    for (int k0 = 0; k0 < count; k0 += batch) {
      const int k1 = k0 + batch < count ? k0 + batch : count;
      for (int k = k0; k < k1; ++k) {
        const int from = morpho::cache_compact_source(keep[k], k);
        got[k] = from >= 0 && from < n ? token[from] : -1;
      }
      for (int k = k0; k < k1; ++k)
        if (got[k] >= 0 && k < n) token[k] = got[k];
    }
    for (int i = 0; i < n; ++i) printf("%d ", token[i]);
    printf("\n");
  }
}
'''


@pytest.fixture(scope="module")
def compact(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    d = tmp_path_factory.mktemp("cache_compact")
    (d / "compact.cpp").write_text(COMPACT)
    subprocess.run(["g++", "-std=c++17", "-O1", f"-I{ROOT}/morphottention_amd/csrc", str(d / "compact.cpp"), "-o",
                    str(d / "compact")], check=True)

    def move(rows):
        text = "".join(f"{n} {batch} {len(keep)} {' '.join(map(str, keep))}\n" for n, batch, keep in rows)
        out = subprocess.run([str(d / "compact")], input=text, capture_output=True, text=True, check=True).stdout
        return [list(map(int, line.split())) for line in out.splitlines()]

    return move


def test_compaction_in_batches_is_the_move_at_once(compact):
    """Every entry takes its token from where it was before the call, in batches of
    any length and whatever the row holds; one below its place moves nothing."""
    rng = random.Random(3)
    rows = [(60, 16, [-1, *range(40)]), (60, 16, [-2, -1, *range(3, 40)]), (20, 4, [5, 5, 4, 1, 19, 20, 7])]
    for _ in range(300):
        n = rng.randint(1, 60)
        keep = [rng.randint(-3, n + 3) for _ in range(rng.randint(1, n))]
        rows += [(n, batch, k) for batch in (1, 4, 16) for k in (keep, sorted(keep))]
    for (n, batch, keep), got in zip(rows, compact(rows)):
        want = list(range(n))
        for k, entry in enumerate(keep):
            if k <= entry < n:
                want[k] = entry
        assert got == want, (n, batch, keep)


# ---------------------------------------------------------------- steps
@pytest.fixture
def recorded(monkeypatch):
    """The kernels' calls, recorded instead of made."""
    calls = []
    for module, name in ((autograd, "morpho_cache_append"), (autograd, "morpho_cache_attention"),
                         (cache_module, "morpho_cache_copy_pages"), (cache_module, "morpho_cache_compact")):
        def record(*args, _name=name, **kw):
            calls.append(_name)
            return torch.zeros(1), torch.zeros(1)
        monkeypatch.setattr(module, name, record)
    return calls


def _layer(**kw):
    return ma.MorphoAttention(64, 2, 16, causal=True, **kw)


def test_forward_cached_refuses_a_step_that_is_not_good_any_more(recorded):
    """After the step's sequence was freed, shortened or committed its pages may be
    another sequence's: nothing is stored."""
    layer = _layer()
    weights = layer.pack_cache_weights()
    x = torch.zeros((1, 3, 64), dtype=torch.float16)
    for change in ("free", "truncate", "evict", "commit", "accept"):
        c = ma.MorphoCache(8, 2, 16, 32, page_size=32)
        a = c.new()
        c.commit(c.step([a], 40))
        step = c.step([a], 3)
        with torch.no_grad():
            layer.forward_cached(x, weights, c, step)
        assert recorded == ["morpho_cache_append", "morpho_cache_attention"]
        {"free": lambda: c.free(a), "truncate": lambda: c.truncate(a, 40), "evict": lambda: c.evict(a, [0, 1]),
         "commit": lambda: c.commit(step), "accept": lambda: c.accept(step, [[0, 1]])}[change]()
        recorded.clear()
        with torch.no_grad(), pytest.raises(KeyError if change == "free" else RuntimeError):
            layer.forward_cached(x, weights, c, step)
        assert not recorded, change


@pytest.mark.parametrize("shape", [(2, 7, 64), (1, 8, 64), (3, 8, 64), (3, 9, 64), (2, 0, 64), (16, 64), (128,)])
@pytest.mark.parametrize("counts", [8, [8, 3]])
def test_forward_cached_refuses_tokens_that_are_not_the_steps(recorded, shape, counts):
    """Fewer tokens would leave committed places unwritten, more would be stored
    without being the step's."""
    layer = _layer()
    c = ma.MorphoCache(8, 2, 16, 32, page_size=32)
    step = c.step([c.new(), c.new()], counts)
    with torch.no_grad(), pytest.raises(ValueError, match="2 rows of 8 tokens"):
        layer.forward_cached(torch.zeros(shape, dtype=torch.float16), layer.pack_cache_weights(), c, step)
    assert not recorded


def test_forward_cached_takes_wider_padding_only_where_counts_tell(recorded):
    """A step of equal counts has no list of them on the device: a ninth token would
    be stored. Where the counts differ it is padding."""
    layer = _layer()
    weights, x = layer.pack_cache_weights(), torch.zeros((2, 9, 64), dtype=torch.float16)
    c = ma.MorphoCache(8, 2, 16, 32, page_size=32)
    with torch.no_grad():
        with pytest.raises(ValueError, match="2 rows of 8 tokens"):
            layer.forward_cached(x, weights, c, c.step([c.new(), c.new()], 8))
        assert not recorded
        layer.forward_cached(x, weights, c, c.step([c.new(), c.new()], [8, 3]))
        assert recorded


def test_forward_cached_raises_where_a_gradient_would_be_needed(recorded):
    """Of the input, the packed weights or any parameter: none is dropped silently."""
    layer = _layer()
    weights, x = layer.pack_cache_weights(), torch.zeros((1, 3, 64), dtype=torch.float16)
    c = ma.MorphoCache(8, 2, 16, 32, page_size=32)
    step = c.step([c.new()], 3)
    for p in layer.parameters():
        p.requires_grad_(False)
    for t in (x, weights, *layer.parameters()):
        t.requires_grad_(True)
        with pytest.raises(RuntimeError, match="no gradients"):
            layer.forward_cached(x, weights, c, step)
        assert not recorded
        with torch.no_grad():
            layer.forward_cached(x, weights, c, step)
        t.requires_grad_(False)
        recorded.clear()
    layer.forward_cached(x, weights, c, step)  # a frozen layer needs none
    assert recorded


def test_a_step_of_another_cache_is_refused(recorded):
    """Caches number their sequences alike (a draft model's and its target's): a step
    of one names pages that mean nothing in the other."""
    layer = _layer()
    weights, x = layer.pack_cache_weights(), torch.zeros((1, 3, 64), dtype=torch.float16)
    one, two = (ma.MorphoCache(8, 2, 16, 32, page_size=32) for _ in range(2))
    a, b = one.new(), two.new()
    assert a == b
    step = one.step([a], 3)
    with torch.no_grad():
        for call in (lambda: layer.forward_cached(x, weights, two, step), lambda: two.commit(step),
                     lambda: two.accept(step, [[1]])):
            with pytest.raises(RuntimeError, match="another cache"):
                call()
    assert not recorded and two.length(b) == 0 and two.pages(b) == ()
    one.commit(step)
    assert one.length(a) == 3


def test_a_sequence_without_new_tokens_keeps_its_pages(recorded):
    """A count of 0 writes nothing, so a shared page that is not full is not copied,
    and a full pool is no obstacle."""
    c = ma.MorphoCache(3, 2, 16, 32, page_size=32)
    a = c.new()
    c.commit(c.step([a], 64))
    b = c.fork(a)
    c.truncate(b, 40)
    before = c.pages(b)
    assert before == c.pages(a)
    c.commit(c.step([a, b], [3, 0]))  # the last page is a's third
    assert c.pages(b) == before and c.free_pages == 0 and not recorded
    c.free(a)
    c.commit(c.step([b], 1))
    assert c.pages(b) == before and not recorded  # nobody else has it any more


def test_a_dropped_step_gives_its_pages_back(recorded):
    """By drop(), or when nobody has it any more: the pool is as it was, and another
    sequence can have the pages."""
    c = ma.MorphoCache(8, 2, 16, 32, page_size=32)
    a, b = c.new(), c.new()
    c.commit(c.step([a], 40))
    assert c.free_pages == 6
    c.step([a], 7 * 32 - 40)
    assert c.free_pages == 6 and c.length(a) == 40
    step = c.step([a], 7 * 32 - 40)
    assert c.free_pages == 1
    c.drop(step)
    assert c.free_pages == 6
    with torch.no_grad():
        for call in (lambda: c.commit(step), lambda: c.accept(step, [[0]]),
                     lambda: _layer().forward_cached(torch.zeros((1, step.n, 64)), None, c, step)):
            with pytest.raises(RuntimeError):
                call()
    c.drop(step)  # again: nothing left to do
    try:
        step = c.step([a], 100)
        raise KeyError("between step and commit")
    except KeyError:
        del step
    c.commit(c.step([b], 6 * 32))  # all that a's tokens leave
    assert c.free_pages == 0 and c.length(a) == 40 and not recorded


def test_a_step_that_is_there_keeps_its_pages(recorded):
    """A full pool takes nothing from a step that can still be committed, from its
    copies, or from another step of the same sequence."""
    c = ma.MorphoCache(8, 2, 16, 32, page_size=32)
    a, b = c.new(), c.new()
    step = c.step([a], 5 * 32)
    with pytest.raises(RuntimeError, match="cache is full"):
        c.step([b], 4 * 32)
    step = dataclasses.replace(step, table=step.table.clone())
    with pytest.raises(RuntimeError, match="cache is full"):
        c.step([b], 4 * 32)
    step = copy.copy(step)
    shorter, longer = c.step([a], 70), c.step([a], 7 * 32)
    assert c.free_pages == 1
    c.drop(longer)
    assert c.free_pages == 3
    c.drop(shorter)
    assert c.free_pages == 3
    c.commit(step)
    assert c.length(a) == 5 * 32 and len(c.pages(a)) == 5
    with pytest.raises(RuntimeError, match="another cache"):
        ma.MorphoCache(8, 2, 16, 32).drop(step)
    c.drop(step)  # it is committed: no harm
    assert c.length(a) == 5 * 32 and c.free_pages == 3
    other = c.step([a], 1)
    long = c.step([a], 64)
    c.commit(other)  # the long one is not good any more, and claims nothing
    assert c.free_pages == 2 and long is not None


@pytest.mark.parametrize("seed", range(8))
def test_account_with_steps_in_flight(recorded, seed):
    """Several steps at once, committed, accepted or dropped in any order: no page has
    two owners or is lost, a step's pages are its own until it ends, and those
    that nobody claims can be had."""
    rng = random.Random(seed)
    c = ma.MorphoCache(24, 2, 16, 32, page_size=32)
    steps, seqs = [], [c.new() for _ in range(4)]
    for _ in range(300):
        act = rng.choice(["step", "step", "step", "commit", "accept", "drop", "lose", "truncate", "fork", "free", "evict"])
        s = rng.choice(seqs)
        try:
            if act == "step":
                mine = rng.sample(seqs, rng.randint(1, 3))
                counts = [rng.choice([0, 1, 33, 100]) for _ in mine]
                if max(counts):
                    steps.append(c.step(mine, counts))
            elif act in ("commit", "accept") and steps:
                step = steps.pop(rng.randrange(len(steps)))
                c.commit(step) if act == "commit" else c.accept(step, [list(range(0, k, 2)) for k in step.counts])
            elif act == "drop" and steps:
                c.drop(steps.pop(rng.randrange(len(steps))))
            elif act == "lose" and steps:
                del steps[rng.randrange(len(steps))]
            elif act == "truncate":
                c.truncate(s, rng.randint(0, c.length(s)))
            elif act == "evict":
                c.evict(s, list(range(0, c.length(s), 2)))
            elif act == "fork" and len(seqs) < 7:
                seqs.append(c.fork(s))
            elif act == "free" and len(seqs) > 3:
                c.free(s)
                seqs.remove(s)
        except (RuntimeError, KeyError) as e:
            assert any(t in str(e) for t in ("cache is full", "have changed", "no sequence"))
        uses = [0] * c.num_pages
        for s in seqs:
            for p in c.pages(s):
                uses[p] += 1
            assert len(c.pages(s)) * 32 >= c.length(s)
        assert uses == c._uses and sorted(c._free) == [p for p in range(c.num_pages) if not uses[p]]
        good = []
        for step in steps:
            try:
                c._still(step)
            except (RuntimeError, KeyError):
                continue
            good.append(step)
            for b, (s, k) in enumerate(zip(step.seqs, step.counts)):
                for t in range(c.length(s), c.length(s) + k):
                    page = int(step.table[b, t // 32])
                    assert c.pages(s)[t // 32] == page and uses[page] == 1
    steps.clear()
    good.clear()
    del step
    assert c.free_pages == 24 - len({p for s in seqs for p in c.pages(s)[: -(-c.length(s) // 32)]})
    for s in seqs:
        c.free(s)
    assert c.free_pages == 24 and not c._claims and not c._grown


def test_a_copy_that_fails_changes_no_account(monkeypatch):
    """Where the pages cannot be copied (the copy raises, as host tensors in a graph
    capture do), no sequence gets a page without its tokens, and none is lost."""
    c = ma.MorphoCache(8, 2, 16, 32, page_size=32)
    a = c.new()
    c.commit(c.step([a], 64))
    b = c.fork(a)
    c.truncate(b, 40)
    before = c.pages(a), c.pages(b), c.free_pages, list(c._uses)

    def fail(*args):
        raise RuntimeError("no copy")
    monkeypatch.setattr(cache_module, "morpho_cache_copy_pages", fail)
    for call in (lambda: c.fork(b), lambda: c.step([b], 1), lambda: c.step([a, b], [64, 3]), lambda: c.evict(a, [1, 2])):
        with pytest.raises(RuntimeError, match="no copy"):
            call()
        assert (c.pages(a), c.pages(b), c.free_pages, c._uses) == before
        assert sorted(c._free) == [p for p in range(8) if not c._uses[p]]
