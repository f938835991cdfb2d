"""Failure paths of the paged kernels without a GPU fault: waits that run out and are recorded."""
from __future__ import annotations

import pytest
import torch

from test_paged_gpu import PLANS, Cache, _clean, _q, _tables

pytestmark = pytest.mark.gpu


def _announced_only(fqkv, call):
    """Status of a call whose copies are announced, but never issued, to consumers that give up at once."""
    lib = fqkv.native.lib()
    torch.cuda.synchronize()
    lib.fqkv_set_wait_timeout_ms(50)
    lib.fqkv_debug_skip_loads(2)
    try:
        call()
        torch.cuda.synchronize()
    finally:
        lib.fqkv_debug_skip_loads(0)
        lib.fqkv_set_wait_timeout_ms(2000)
    return fqkv.ops.device_status(torch.device("cuda", 0))


@pytest.mark.parametrize("int8", [False, True])
@PLANS
def test_attention_waits_for_copies_in_flight(fqkv, int8, line):
    """A CTA of one to three tiles never asks for a free stage, so nothing tells its producer that the consumers gave up; it
    waits for its copies all the same: here they never land, and that wait runs out (63)."""
    c = Cache(fqkv, [300, 70], 2, 128, 16, int8)
    if line:
        c.widen()
    q = _q(2, 8, 128)
    assert _announced_only(fqkv, lambda: c.attend(fqkv, q)) == 63
    c.check(fqkv, q, c.attend(fqkv, q))
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
def test_append_waits_for_copies_in_flight(fqkv, int8):
    """As above: 1200 tokens, one or two for a block."""
    D, Hq, Hkv, T = 64, 4, 2, 1200
    c = Cache(fqkv, [0, 0], Hkv, D, 16, int8, room=600)
    cos, sin = _tables(600, D)
    i = torch.arange(T, dtype=torch.int32).cuda()
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1)).half().cuda()
    q_out = torch.zeros(T, Hq, D, dtype=torch.float16, device="cuda")
    call = lambda: fqkv.rope_qkv_append_paged(qkv, cos, sin, i % 600, i % 600, c.table, q_out, c.K, c.V, c.Ks, c.Vs,  # noqa: E731
                                              seq_ids=i // 600)
    assert _announced_only(fqkv, call) == 63
    assert not bool(q_out.any())
    call()
    torch.cuda.synchronize()
    assert bool((q_out != 0).flatten(1).any(1).all())
    _clean(fqkv)
