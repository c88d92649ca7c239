"""What the paged cache promises for calls that its documentation allows but that are
easy to get wrong, on the GPU."""

from __future__ import annotations

import pytest
import torch

import morphottention_amd as ma

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
