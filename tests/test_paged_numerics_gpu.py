"""GPU tests of the paged attention where small terms decide the result, against float64.

Bounds as in ``test_paged_gpu.py``, with the term for probabilities below the fp16 range made as small as the kernels'
scaling of them makes it: an fp16 cache's are scaled by 2^15 (half a subnormal step is 2^-25 2^-15 of the row's largest), an
int8 cache's by what puts the largest V scale in [2^13, 2^14).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import paged as op
from test_paged_gpu import PLANS, U16, Cache, _clean, _q

pytestmark = pytest.mark.gpu


def _one_dominant_key(fqkv, n, D, heads, int8, seed):
    """One sequence: token 0 takes nearly all of every head's weight and its value is 0, all others score 0; so the output
    is what the small weights add up to.  Head h's small weights are 2^-x of the largest, x from 15 to 36."""
    c = Cache(fqkv, [n], 1, D, 64, int8, seed=seed, extra_pages=0)
    g = torch.Generator().manual_seed(seed)
    P, page = c.P, c.page
    K = torch.randn(P, 1, page, D, generator=g)
    K[..., 0] = 0
    V = torch.rand(P, 1, page, D, generator=g) * 8 + 56
    first = int(c.table[0, 0])
    K[first, 0, 0] = 0
    K[first, 0, 0, 0] = 16
    V[first, 0, 0] = 0
    if int8:
        (c.K, c.Ks), (c.V, c.Vs) = fqkv.qpt(K.half().cuda()), fqkv.qpt(V.half().cuda())
    else:
        c.K, c.V = K.half().cuda(), V.half().cuda()
    x = torch.linspace(15.0, 36.0, heads, dtype=torch.float64)
    q = torch.zeros(1, heads, D)
    q[0, :, 0] = (x * np.log(2.0) * np.sqrt(D) / 16).float()
    return c, q.half().cuda()


def _bound(r, n, D, int8):
    # the longest chain of fp32 additions: of O an MMA per 16 keys and warp, of L one per key of a lane (2 half steps each)
    steps = n / 64 + n / 32 + 64
    ds = (D + 8) * 2.0 ** -23 * r["smax"][..., None]
    small = n * (2.0 ** -37 if int8 else 2.0 ** -40) * r["vmax"]
    return U16 * np.abs(r["out"]) + 2.0 ** -25 + (U16 + 2 * ds + steps * 2.0 ** -23) * r["absum"] + small


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("heads", [1, 8, 16])
@PLANS
def test_many_small_weights_beside_a_dominant_one(fqkv, int8, D, heads, line):
    n = 8000
    c, q = _one_dominant_key(fqkv, n, D, heads, int8, seed=D + heads)
    if line:
        c.widen()
    out = c.attend(fqkv, q).double().cpu().numpy()
    K, V = c.values()
    r = op.paged_attention(q.cpu().double().numpy(), K, V, c.table.cpu().numpy(), [n])
    assert (np.abs(out - r["out"]) <= _bound(r, n, D, int8)).all(), np.abs(out / r["out"] - 1).max(-1)
    w = torch.zeros(1, 1, c.cap, device="cuda")
    out = c.attend(fqkv, q, weights=w).double().cpu().numpy()
    assert (np.abs(out - r["out"]) <= _bound(r, n, D, int8)).all()
    ds = (D + 8) * 2.0 ** -23 * r["smax"][0][:, None]
    p = r["p"][0]
    assert (np.abs(w[0, 0, :n].double().cpu().numpy() - p.sum(0)) <= ((2 * ds + n * 2.0 ** -23) * p).sum(0) + 1e-37).all()
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
def test_long_sequences_with_a_dominant_key(fqkv, int8):
    """600 sequences of 128K tokens on the same pages: every CTA goes through about a whole one, the dominant key first."""
    n, D, B = 131072, 64, 600
    c, q = _one_dominant_key(fqkv, n, D, 8, int8, seed=1)
    K, V = c.values()
    r = op.paged_attention(q.cpu().double().numpy(), K, V, c.table.cpu().numpy(), [n])
    c.table, c.lens = c.table.expand(B, -1).contiguous(), c.lens.expand(B).contiguous()
    out = c.attend(fqkv, q.expand(B, -1, -1).contiguous()).double().cpu().numpy()
    assert (np.abs(out - r["out"]) <= _bound(r, n, D, int8)).all(), np.abs(out / r["out"] - 1).max((0, 2))
    _clean(fqkv)


@pytest.mark.parametrize("D,Hq", [(64, 4), (128, 8), (128, 24)])
@PLANS
def test_int8_scales_of_either_sign(fqkv, D, Hq, line):
    """V scales all negative, of both signs, and negative first; K scales of both signs."""
    c = Cache(fqkv, [300, 300, 300], 2, D, 16, True, seed=D)
    g = torch.Generator().manual_seed(4)
    sign = (torch.randint(2, c.Ks.shape, generator=g) * 2 - 1).half().cuda()
    c.Ks = c.Ks * sign
    c.Vs[c.table[0, :19].long()] *= -1
    c.Vs = c.Vs.contiguous()
    for i in range(19):
        c.Vs[int(c.table[1, i])] *= sign[int(c.table[1, i])]
        if i < 9:  # small negative ones, then larger positive ones
            c.Vs[int(c.table[2, i])] *= -2.0 ** -6
    if line:
        c.widen()
    q = _q(3, Hq, D)
    c.check(fqkv, q, c.attend(fqkv, q))
    w = torch.zeros(3, 2, c.cap, device="cuda")
    out = c.attend(fqkv, q, weights=w)
    c.check(fqkv, q, out, torch.zeros_like(w), w)
    _clean(fqkv)
