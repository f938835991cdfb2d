"""Host side of the paged-cache calls: the rotary axis map's counts."""
from __future__ import annotations

import pytest
import torch


@pytest.mark.parametrize("sections", [[24, 20, 20], [16, 24, 24], [8, 12, 12], [9, 23], [6, 3, 3], [0, 5], [5, 0, 0], [1, 30, 2, 7],
                                      [64]])
def test_interleaved_axes_have_the_documented_counts(fqkv, sections):
    """Axis a > 0: its section, capped at the pairs of its residue class; axis 0: the rest."""
    n, A = sum(sections), len(sections)
    ids = fqkv.rope_axes(sections, interleaved=True, device="cpu")
    want = [min(s, len(range(a, n, A))) for a, s in enumerate(sections)]
    want[0] = n - sum(want[1:])
    assert torch.bincount(ids, minlength=A).tolist() == want
    assert all(a in (0, i % A) for i, a in enumerate(ids.tolist()))


def test_interleaved_axes_documented_examples(fqkv):
    counts = lambda s: torch.bincount(fqkv.rope_axes(s, interleaved=True, device="cpu")).tolist()  # noqa: E731
    assert counts([16, 24, 24]) == [22, 21, 21] and counts([24, 20, 20]) == [24, 20, 20]
    assert "[16, 24, 24] gives 22, 21 and 21" in fqkv.rope_axes.__doc__
