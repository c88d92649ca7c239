"""Serving a causal morpho-attention layer from a paged cache.

No reference counterpart: the reference computes whole sequences only. The
score of a query and a key is

    s_ij = scale sum_c G_c (2 phi_ic phi_jc - phi_ic - phi_jc),  G = gate_q * gate_k,

so what later tokens need of an earlier one is its codes ``phi`` and its values
``x W_V``. Both are kept in float16 pages:

* ``codes``  ``[layers, pages, H, page_size, cube_m]``;
* ``values`` ``[layers, pages, H, page_size // 8, head_dim, 8]``: column ``c`` of
  token ``t`` of a page at ``[t // 8, c, t % 8]``, the order in which the value
  product reads them.

The functions work on such tensors directly, with a ``table`` ``[B, seq_pages]``
(int32, each sequence's pages in order) and ``lens`` ``[B]`` (int32, its tokens
before the new ones) in device memory, and may be captured in a graph:

* :func:`morpho_cache_append` projects new tokens and stores them;
* :func:`morpho_cache_attention` lets them attend: one token a sequence, pieces
  of a prompt, or a tree of drafted tokens;
* :func:`morpho_cache_copy_pages` and :func:`morpho_cache_compact` copy pages and
  move kept tokens together, in all layers at once.

:class:`MorphoCache` owns the tensors and keeps account of the pages (sharing
between forks, copies on write, rollback). ``MorphoAttention.forward_cached``
runs a layer on it.

The cache serves inference: none of this is differentiable, and a call that
would need a gradient raises.
"""

from __future__ import annotations

import itertools
from dataclasses import dataclass, field

import torch

from ._ops import add_op_namespace_prefix, ops


@torch.library.register_fake(add_op_namespace_prefix("cache_append"))
def _cache_append_fake(X, weights, codes, values, table, lens, new_lens=None, variant=0):
    return X.new_empty((X.shape[0], X.shape[1], codes.shape[1], codes.shape[3]))


@torch.library.register_fake(add_op_namespace_prefix("cache_attention"))
def _cache_attention_fake(phi, gate_q, gate_k, codes, values, table, lens, new_lens, tree, scale, causal, variant=0,
                          max_len=0):
    B, n, H, _m = phi.shape
    return [phi.new_empty((B, n, H * values.shape[3])), phi.new_empty((B * H, n), dtype=torch.float32)]


@torch.library.register_fake(add_op_namespace_prefix("cache_copy_pages"))
def _cache_copy_pages_fake(codes, values, src, dst):
    return None


@torch.library.register_fake(add_op_namespace_prefix("cache_compact"))
def _cache_compact_fake(codes, values, table, lens, keep, keep_lens=None):
    return None


_PROJECTION_BITS = {"sigmoid": 0, "hardtanh01": 4, "identity": 8}
_MASK_DIAG = 2


def refuse_grad(*tensors) -> None:
    """Raise if a gradient of one of the tensors would be needed."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("the cache serves inference and has no gradients: call it under torch.no_grad()")


def pack_cache_weights(W_phi: torch.Tensor, W_V: torch.Tensor) -> torch.Tensor:
    """``[W_phi | W_V]`` transposed, ``[H * cube_m + D, D]``: the weights as
    :func:`morpho_cache_append` reads them. Done once, and again after the
    weights have changed."""
    return torch.cat((W_phi.detach(), W_V.detach()), 1).t().contiguous()


def morpho_cache_append(x: torch.Tensor, weights: torch.Tensor, codes: torch.Tensor, values: torch.Tensor,
                        table: torch.Tensor, lens: torch.Tensor, *, new_lens: torch.Tensor | None = None,
                        projection: str = "sigmoid") -> torch.Tensor:
    """Project new tokens and store their codes and values in one layer's pages.

    :param x: the new tokens ``[B, n, D]``, float16.
    :param weights: :func:`pack_cache_weights` of the layer.
    :param codes: ``[pages, H, page_size, cube_m]``, written.
    :param values: ``[pages, H, page_size // 8, head_dim, 8]``, written.
    :param table: int32 ``[B, seq_pages]``, the pages of each sequence. Two
        sequences must not share a page that is appended to.
    :param lens: int32 ``[B]``, tokens of each sequence before the new ones; new
        token ``i`` goes to position ``lens[b] + i``. A position past the table
        or on a page that the pool does not have is not stored.
    :param new_lens: int32 ``[B]``, new tokens of each sequence where not all
        have ``n``; the rows behind them are padding and not stored.
    :param projection: the layer's cube projection.
    :returns: the codes ``[B, n, H, cube_m]`` of every row, as they are stored.
    """
    if projection not in _PROJECTION_BITS:
        raise ValueError(f"projection must be one of {sorted(_PROJECTION_BITS)} (got {projection!r})")
    refuse_grad(x, weights)
    return ops.cache_append(x, weights, codes, values, table, lens, new_lens, _PROJECTION_BITS[projection])


def morpho_cache_attention(phi: torch.Tensor, gate_q: torch.Tensor, gate_k: torch.Tensor, codes: torch.Tensor,
                           values: torch.Tensor, table: torch.Tensor, lens: torch.Tensor, *,
                           new_lens: torch.Tensor | None = None, tree: torch.Tensor | None = None, scale: float = 1.0,
                           causal: bool = True, mask_diag: bool = False,
                           max_len: int | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Attention of new tokens, appended before, over their sequences.

    :param phi: their codes ``[B, n, H, cube_m]``, from :func:`morpho_cache_append`.
    :param codes, values, table, lens, new_lens: as there (``lens`` still counts
        the tokens before the new ones). Keys on a page that the pool does not
        have are left out.
    :param tree: int64 ``[B, n]``, ``n <= 64``: the new tokens are drafts. Token
        ``i`` sees the ``lens[b]`` tokens before them and draft ``k`` where bit
        ``k`` of ``tree[b, i]`` is set (its own bit among them). Replaces
        ``causal`` and ``mask_diag``.
    :param causal: new token ``i`` sees positions up to ``lens[b] + i``; else all.
    :param mask_diag: drop each token's own key.
    :param max_len: at least the longest ``lens[b] + new_lens[b]``. Sets how the
        work is split, not what is computed; the table's whole length if not given.
    :returns: ``out`` ``[B, n, D]`` and the base-2 log-sum-exp of the row scores
        ``[B * H, n]`` (float32). A row that sees nothing, and a padding row,
        has 0 and ``-FLT_MAX``. ``scale * gate_q * gate_k`` has to stay below
        22,700 (codes within [0, 1]), as in the whole-sequence forward. Up to 64
        new tokens the result is exact to fp32 rounding; beyond, where the weights
        are the bound, each is rounded to float16 once (2^-11 of its value), as in
        the whole-sequence forward: ``n`` of at most 64 a call avoids that.
    """
    if max_len is not None and max_len <= 0:
        raise ValueError(f"max_len must be positive (got {max_len})")
    if tree is not None and mask_diag:
        raise ValueError("mask_diag with a tree: leave a draft's own bit out instead")
    refuse_grad(phi, gate_q, gate_k)
    out, lse = ops.cache_attention(phi, gate_q, gate_k, codes, values, table, lens, new_lens, tree, scale, causal,
                                   _MASK_DIAG if mask_diag else 0, max_len or 0)
    return out, lse


def morpho_cache_copy_pages(codes: torch.Tensor, values: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy page ``src[k]`` to page ``dst[k]`` (int32 ``[pairs]``), in every layer
    when ``codes`` and ``values`` have a leading layer dimension. No page may be
    written twice, or written and read. Pairs with a page that the pool does
    not have are left out."""
    ops.cache_copy_pages(codes, values, src, dst)


def morpho_cache_compact(codes: torch.Tensor, values: torch.Tensor, table: torch.Tensor, lens: torch.Tensor,
                         keep: torch.Tensor, *, keep_lens: torch.Tensor | None = None) -> None:
    """Move token ``lens[b] + keep[b, k]`` to position ``lens[b] + k``, in place and
    in every layer: the accepted path of a tree to the front of its drafts
    (``lens``: the tokens before them), or what is left after tokens were
    evicted (``lens``: 0). No other sequence of the call may have a page that
    tokens move to.

    :param keep: int32 ``[B, kept]``; has to ascend along each row, none twice. An
        entry below its own place (``keep[b, k] < k``, negative ones among them)
        moves nothing.
    :param keep_lens: int32 ``[B]``, how many of them count.
    """
    ops.cache_compact(codes, values, table, lens, keep, keep_lens)


# What changes the tokens of a sequence gives it a new stamp. They rise and are
# never given twice, by one cache or several: a step is good only for the
# sequences that it was made for.
_stamps = itertools.count()


class _Claim:
    """A step's claim on the pages of its new tokens. It ends with the step (and its
    copies): when the cache takes the step back, or when nobody has it any more."""

    def __init__(self, claims: dict[int, dict[int, int]], mine: dict[int, int]) -> None:
        self.claims, self.key, self.dropped = claims, next(_stamps), False
        claims[self.key] = mine

    def end(self) -> None:
        self.claims.pop(self.key, None)

    __del__ = end


@dataclass
class CacheStep:
    """New tokens of some sequences: what one forward pass of all layers needs."""

    seqs: list[int]
    counts: list[int]
    n: int
    table: torch.Tensor
    lens: torch.Tensor
    new_lens: torch.Tensor | None
    max_len: int
    stamps: list[int]
    claim: _Claim | None = field(default=None, repr=False, compare=False)


class MorphoCache:
    """Pages of key codes and values, and which sequence has which of them.

    :param num_pages: pages of each layer.
    :param num_heads, cube_m, head_dim: of the layers' ``MorphoAttention``.
    :param num_layers: layers that share the account of pages.
    :param page_size: tokens a page: 32, 64, 128 or 256.
    :param device: where the pages are; the kernels need a ROCm device.

    A step appends tokens to some sequences and is then committed::

        seq = cache.new()
        step = cache.step([seq], x.shape[1])          # pages for the new tokens
        for i, layer in enumerate(layers):
            x = layer.forward_cached(x, weights[i], cache, step, layer=i)
        cache.commit(step)

    Until then the sequences keep their old lengths, so a step that is dropped
    leaves their tokens as they were. Its pages are free again after :meth:`drop`,
    or once nobody has the step any more (an exception, say). After a tree of
    drafts :meth:`accept` takes the accepted tokens instead. A step is good for
    one commit, and only as long as its sequences have not changed otherwise.
    Steps of one sequence that are made before either is committed write to the
    same places.
    """

    def __init__(self, num_pages: int, num_heads: int, cube_m: int, head_dim: int, *, num_layers: int = 1,
                 page_size: int = 64, device: torch.device | str | None = None) -> None:
        if cube_m not in (16, 32, 64):
            raise ValueError(f"cube_m must be 16, 32 or 64 (got {cube_m})")
        if head_dim not in (32, 64, 128):
            raise ValueError(f"head_dim must be 32, 64 or 128 (got {head_dim})")
        if page_size not in (32, 64, 128, 256):
            raise ValueError(f"page_size must be 32, 64, 128 or 256 (got {page_size})")
        if min(num_pages, num_heads, num_layers) <= 0:
            raise ValueError("num_pages, num_heads and num_layers must be positive")
        self.page_size = page_size
        self.num_pages = num_pages
        self.codes = torch.zeros((num_layers, num_pages, num_heads, page_size, cube_m), dtype=torch.float16,
                                 device=device)
        self.values = torch.zeros((num_layers, num_pages, num_heads, page_size // 8, head_dim, 8), dtype=torch.float16,
                                  device=device)
        self._free = list(range(num_pages - 1, -1, -1))
        self._uses = [0] * num_pages
        self._pages: dict[int, list[int]] = {}
        self._lens: dict[int, int] = {}
        self._stamp: dict[int, int] = {}
        # of each step that is neither committed nor dropped: its stamp, and {seq: end of the new tokens}
        self._claims: dict[int, dict[int, int]] = {}
        self._grown: set[int] = set()  # sequences that may have pages past their tokens
        self._next = 0

    # ---- account
    @property
    def free_pages(self) -> int:
        """Pages that no sequence has, and no step claims for one."""
        self._shrink()
        return len(self._free)

    def length(self, seq: int) -> int:
        """Committed tokens of a sequence."""
        return self._lens[self._known(seq)]

    def pages(self, seq: int) -> tuple[int, ...]:
        """The pages of a sequence, in order (with those of a step that is not committed yet)."""
        return tuple(self._pages[self._known(seq)])

    def _known(self, seq: int) -> int:
        if seq not in self._pages:
            raise KeyError(f"no sequence {seq}")
        return seq

    def _take(self, count: int) -> list[int]:
        if count > len(self._free):
            raise RuntimeError(f"the cache is full: {count} pages needed, {len(self._free)} of {self.num_pages} free")
        got = [self._free.pop() for _ in range(count)]
        for p in got:
            self._uses[p] = 1
        return got

    def _drop(self, pages) -> None:
        for p in pages:
            self._uses[p] -= 1
            if self._uses[p] == 0:
                self._free.append(p)

    def _cut(self, seq: int, length: int) -> bool:
        """Give up the pages of a sequence past ``length`` tokens."""
        keep = -(-length // self.page_size)
        gone = self._pages[seq][keep:]
        self._drop(gone)
        del self._pages[seq][keep:]
        return bool(gone)

    def _shrink(self) -> None:
        """Give up the pages past the tokens of sequences that no step claims any more."""
        claims = self._claims.copy().items()  # of which any may end while this runs
        for seq in list(self._grown):
            ends = [claim[seq] for stamp, claim in claims if seq in claim and stamp > self._stamp[seq]]
            if not ends:
                self._grown.discard(seq)
            if self._cut(seq, max([self._lens[seq], *ends])) and not ends:
                self._stamp[seq] = next(_stamps)  # nor is a step good that was taken apart

    def new(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._pages[seq], self._lens[seq], self._stamp[seq] = [], 0, next(_stamps)
        return seq

    def free(self, seq: int) -> None:
        """Give a sequence up; its pages that no fork shares are free again."""
        self._drop(self._pages.pop(self._known(seq)))
        del self._lens[seq], self._stamp[seq]
        self._grown.discard(seq)

    def _ints(self, rows) -> torch.Tensor:
        return torch.tensor(rows, dtype=torch.int32, device=self.codes.device)

    def _copies(self, pages: list[int], fresh: list[int]) -> None:
        """Copy pages to taken ones, before the account says so: where that raises
        (while a graph is captured, say), all of ``fresh`` are free again."""
        try:
            if pages:
                morpho_cache_copy_pages(self.codes, self.values, self._ints(pages), self._ints(fresh[: len(pages)]))
        except BaseException:
            self._drop(fresh)
            raise

    def fork(self, seq: int) -> int:
        """A new sequence with the same tokens. Full pages are shared; a page
        that is not full is copied, since both will append to theirs."""
        length = self._lens[self._known(seq)]
        full, rest = divmod(length, self.page_size)
        if rest and not self._free:
            self._shrink()
        own = self._take(1) if rest else []
        self._copies(self._pages[seq][full : full + len(own)], own)
        shared = self._pages[seq][:full]
        for p in shared:
            self._uses[p] += 1
        new = self.new()
        self._pages[new], self._lens[new] = shared + own, length
        return new

    def truncate(self, seq: int, length: int) -> None:
        """Forget the tokens of a sequence from position ``length`` on."""
        if not 0 <= length <= self._lens[self._known(seq)]:
            raise ValueError(f"length must be 0 .. {self._lens[seq]} (got {length})")
        self._cut(seq, length)
        self._grown.discard(seq)
        self._lens[seq] = length
        self._stamp[seq] = next(_stamps)

    def _missing(self, wanted: list[tuple[int, int, int]]) -> tuple[list[tuple[int, int]], list[int]]:
        """For each (seq, first, end): which of the pages that hold positions first ..
        end - 1 are shared (seq, index), and how many there are none of."""
        P = self.page_size
        shared, grow = [], []
        spare: dict[int, int] = {}
        for seq, first, end in wanted:
            have = self._pages[seq]
            # a shared page is copied for all its users but the last: count down
            for k in range(first // P, min(len(have), -(-end // P))):
                p = have[k]
                left = spare.get(p, self._uses[p])
                if left > 1:
                    shared.append((seq, k))
                    spare[p] = left - 1
            grow.append(max(0, -(-end // P) - len(have)))
        return shared, grow

    def _own(self, wanted: list[tuple[int, int, int]]) -> None:
        """For each (seq, first, end): the pages that hold positions first .. end - 1
        exist and belong to the sequence alone. No sequence's tokens or pages for
        them change when the pool has too few pages left."""
        shared, grow = self._missing(wanted)
        need = len(shared) + sum(grow)
        if need > len(self._free):
            self._shrink()
            shared, grow = self._missing(wanted)  # it may have taken pages of these sequences
            need = len(shared) + sum(grow)
        if not need:
            return
        fresh = self._take(need)
        self._copies([self._pages[seq][k] for seq, k in shared], fresh)
        pages = iter(fresh)
        for seq, k in shared:
            self._uses[self._pages[seq][k]] -= 1
            self._pages[seq][k] = next(pages)
        for (seq, _, _), count in zip(wanted, grow):
            self._pages[seq] += itertools.islice(pages, count)

    # ---- steps
    def step(self, seqs: list[int], counts: int | list[int]) -> CacheStep:
        """Pages for new tokens of some sequences: ``counts`` tokens of each, or a
        list with as many for each."""
        seqs = list(seqs)
        if not seqs or len(set(seqs)) != len(seqs):
            raise ValueError("a step takes one or more different sequences")
        counts = [counts] * len(seqs) if isinstance(counts, int) else list(counts)
        if len(counts) != len(seqs) or min(counts) < 0 or max(counts) == 0:
            raise ValueError("counts must be one number, or one for each sequence, not negative and not all 0")
        ends = [self._lens[self._known(s)] + c for s, c in zip(seqs, counts)]
        self._own([(s, self._lens[s], e) for s, c, e in zip(seqs, counts, ends) if c])
        self._grown.update(seqs)
        claim = _Claim(self._claims, dict(zip(seqs, ends)))
        width = max(-(-e // self.page_size) for e in ends)
        rows = [(self._pages[s] + [-1] * width)[:width] for s in seqs]
        n = max(counts)
        return CacheStep(seqs, counts, n, self._ints(rows), self._ints([self._lens[s] for s in seqs]),
                         self._ints(counts) if min(counts) < n else None, max(ends), [self._stamp[s] for s in seqs], claim)

    def drop(self, step: CacheStep) -> None:
        """Give a step up that is not committed: its pages past the tokens of its
        sequences are free again. (A page that it copied on write stays the
        sequence's own.)"""
        if step.claim is None or step.claim.claims is not self._claims:
            raise RuntimeError("the step is another cache's")
        step.claim.dropped = True
        step.claim.end()
        self._shrink()

    def _still(self, step: CacheStep) -> None:
        if step.claim is not None and step.claim.dropped:
            raise RuntimeError("the step was dropped")
        if any(self._stamp[self._known(s)] != stamp for s, stamp in zip(step.seqs, step.stamps)):
            raise RuntimeError("the step's sequences have changed since it was made, or are another cache's")

    def _check(self, step: CacheStep, x: torch.Tensor) -> None:
        """Raise if ``x`` are not the step's new tokens, ``[sequences, step.n, ...]``, or
        if the step is not good any more: its pages may be another sequence's. Where
        the counts differ the kernels know them, and ``x`` may be padded further."""
        self._still(step)
        B, n = len(step.seqs), step.n
        if x.dim() < 2 or x.shape[0] != B or x.shape[1] < n or (x.shape[1] > n and step.new_lens is None):
            raise ValueError(f"x must have {B} rows of {n} tokens, as the step has (got {tuple(x.shape)})")

    def commit(self, step: CacheStep) -> None:
        """The step's tokens belong to their sequences."""
        self._still(step)
        stamp = next(_stamps)
        for s, c in zip(step.seqs, step.counts):
            self._lens[s] = length = self._lens[s] + c
            self._stamp[s] = stamp
            if (len(self._pages[s]) - 1) * self.page_size >= length:
                self._cut(s, length)  # what other steps claimed: none is good any more
        self._grown.difference_update(step.seqs)
        if step.claim is not None:
            step.claim.end()

    def accept(self, step: CacheStep, kept: list[list[int]]) -> None:
        """After a step of drafts: of each sequence the drafts ``kept[b]`` (ascending
        places among its drafts, e.g. the accepted path) are its next tokens,
        the others are dropped."""
        self._still(step)
        if len(kept) != len(step.seqs):
            raise ValueError("kept must have a list for each sequence of the step")
        for k, c in zip(kept, step.counts):
            if any(a >= b for a, b in zip(k, k[1:])) or (k and not 0 <= k[0] <= k[-1] < c):
                raise ValueError(f"kept places must ascend within 0 .. {c - 1} (got {k})")
        if any(k != list(range(len(k))) for k in kept):
            most = max(len(k) for k in kept)
            morpho_cache_compact(self.codes, self.values, step.table, step.lens,
                                 self._ints([list(k) + [0] * (most - len(k)) for k in kept]),
                                 keep_lens=self._ints([len(k) for k in kept]))
        for s, k in zip(step.seqs, kept):
            self._lens[s] += len(k)
            self.truncate(s, self._lens[s])
        if step.claim is not None:
            step.claim.end()

    def evict(self, seq: int, kept: list[int]) -> None:
        """Keep only the tokens at positions ``kept`` (ascending) of a sequence; they
        move together. Pages that forks share are copied first."""
        length = self._lens[self._known(seq)]
        if any(a >= b for a, b in zip(kept, kept[1:])) or (kept and not 0 <= kept[0] <= kept[-1] < length):
            raise ValueError(f"kept positions must ascend within 0 .. {length - 1}")
        still = next((i for i, k in enumerate(kept) if i != k), len(kept))  # these stay where they are
        if still < len(kept):
            self._own([(seq, still, len(kept))])
            morpho_cache_compact(self.codes, self.values, self._ints([self._pages[seq]]), self._ints([still]),
                                 self._ints([[k - still for k in kept[still:]]]))
        self.truncate(seq, len(kept))
