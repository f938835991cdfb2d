"""GPU tests of evictions whose selection one CTA makes of 4097 to 16384 old tokens (16 per thread, held in registers) and
a little more, and of appends of which no token is good."""
from __future__ import annotations

import pytest
import torch

from test_paged_gpu import Cache, _clean, _evict_check, _tables

pytestmark = pytest.mark.gpu

RECENT = 7
LENS = [4097 + RECENT, 5001, 8193, 9000, 16384 + RECENT, 16385 + RECENT, 20000, 300]


def _weights(kind, shape, seed):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(shape, generator=g).exp()
    if kind == "ties":             # few values: the last bin holds thousands of equal keys
        return (w * 4).floor()
    if kind == "equal":
        return torch.ones(shape)
    if kind == "one binade":       # all keys of one first digit, more than the shared memory holds at 4097 and above
        return 1 + torch.rand(shape, generator=g) * 0.2
    return w                       # distinct; few keys in the last bin where the budget cuts a tail


@pytest.mark.parametrize("kind", ["distinct", "ties", "equal", "one binade"])
@pytest.mark.parametrize("budget", [40, 1501, 4090, 6000, 15000])  # from 4097 on a step lists more than it can stage
def test_one_block_selects_thousands(fqkv, kind, budget):
    c = Cache(fqkv, LENS, 1, 64, 256, False, seed=budget)
    assert c.cap <= 24576  # one CTA per selection
    w = _weights(kind, (c.B, 1, c.cap), budget).cuda()
    _evict_check(fqkv, c, w, budget, RECENT, in_place=budget == 1501)
    _clean(fqkv)


def test_one_block_selects_with_heads_of_their_own(fqkv):
    """int8, three KV heads with other weights each, odd pages."""
    c = Cache(fqkv, [5001, 4668, 16300], 3, 128, 48, True, seed=5)
    assert c.cap <= 24576
    w = torch.cat([_weights(k, (c.B, 1, c.cap), 9) for k in ("distinct", "ties", "one binade")], 1).contiguous().cuda()
    w[0, 0, ::5] = float("nan")
    w[2, 1, ::3] = float("inf")
    _evict_check(fqkv, c, w, 1501, 333)
    _clean(fqkv)


@pytest.mark.parametrize("T", [3, 1500])
@pytest.mark.parametrize("int8", [False, True])
def test_append_with_a_bad_axis_writes_nothing(fqkv, int8, T):
    """A pair whose axis names no position row spoils every token, in the few-token and the prompt kernel."""
    D, Hq, Hkv = 64, 4, 2
    c = Cache(fqkv, [0], Hkv, D, 16, int8, room=T)
    pools = [c.K, c.V] + ([c.Ks, c.Vs] if int8 else [])
    for p in pools:
        p.zero_()
    cos, sin = _tables(64, D)
    i = torch.arange(T, dtype=torch.int32).cuda()
    axes = fqkv.rope_axes([20, 12])
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1)).half().cuda()
    q_out = torch.full((T, Hq, D), 5.0, dtype=torch.float16, device="cuda")
    for bad in (2, -1):
        axes[7] = bad
        fqkv.rope_qkv_append_paged(qkv, cos, sin, torch.stack([i % 64, i % 63]), i, c.table, q_out, c.K, c.V, c.Ks, c.Vs, axes=axes,
                                   seq_ids=torch.zeros_like(i))
        with pytest.raises(RuntimeError, match="out of range"):
            fqkv.ops.check_device_status(torch.device("cuda", 0), "append")
        assert bool((q_out == 5).all()) and not any(bool(p.any()) for p in pools)
    _clean(fqkv)
