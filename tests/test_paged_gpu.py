"""GPU tests of the paged-cache operators against their float64 definitions (``oracle/paged.py``).

Bounds, derived from the arithmetic (u16 = 2^-11, u8 = 2^-8: half a step of fp16 and bf16, relative):

* a score: D exact products and their sum in fp32, a few more fp32 roundings; taking a whole step (2^-23) for each,
  since tensor cores may truncate: ds = (D + 8) 2^-23 max_j sum_i |q_i k_ji| / sqrt(D) (absolute, natural units).
* a softmax weight: its own and its sum's score errors, exp2 and fp32 sums: relative 2 ds + 2^-18.
* the output: weights rounded to fp16 (u16 relative; below 2^-14 of the row's largest, 2^-25 absolute and N of them), times
  V exactly, summed in fp32 (N 2^-23 is taken up by 2^-18 for N <= 2^13 ... 2^5 blocks), then rounded once:
  |o - ref| <= u |ref| + (u16 + 2 ds + 2^-17) sum p |v| + N 2^-25 max |v|.
* accumulated weights: the relative error of each term on what is added, and one fp32 step on the sum.
"""
from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import paged as op
from oracle import quant as oq

pytestmark = pytest.mark.gpu

U16, U8 = 2.0 ** -11, 2.0 ** -8


class Cache:
    """A paged cache on the GPU whose unused slots, scales and table entries hold what must not matter."""

    def __init__(self, fqkv, lens, Hkv, D, page, int8, nhd=False, seed=0, extra_pages=2, room=0, sigma=1.0):
        g = torch.Generator().manual_seed(seed)
        B = len(lens)
        held = [-(-(n + room) // page) for n in lens]
        self.P = max(1, sum(held) + extra_pages)
        order = torch.randperm(self.P, generator=g).tolist()
        self.table = torch.randint(-2 ** 31, 2 ** 31 - 1, (B, max(held + [0]) + 1), generator=g, dtype=torch.int64)
        at = 0
        for b, m in enumerate(held):
            self.table[b, :m] = torch.tensor(order[at:at + m], dtype=torch.int64)
            at += m
        self.table = self.table.to(torch.int32).cuda()
        self.lens = torch.tensor(lens, dtype=torch.int32).cuda()
        self.B, self.Hkv, self.D, self.page, self.int8 = B, Hkv, D, page, int8
        self.cap = self.table.shape[1] * page
        used = torch.zeros(self.P, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for j in range(n):
                used[int(self.table[b, j // page]), j % page] = True
        pools, scales = [], []
        for _ in range(2):
            x = (torch.randn(self.P, Hkv, page, D, generator=g) * sigma).half()
            if int8:
                codes, sc = fqkv.qpt(x.cuda())
                codes = torch.where(used.cuda()[:, None, :, None], codes, torch.full_like(codes, -128))
                sc = torch.where(used.cuda()[:, None], sc, torch.full_like(sc, float("nan")))
                scales.append(sc.contiguous())
                x = codes
            else:
                bad = torch.tensor([float("nan"), float("inf"), -float("inf"), 65504.0])[
                    torch.randint(4, x.shape, generator=g)].half()
                x = torch.where(used[:, None, :, None], x, bad).cuda()
            pools.append(x.transpose(1, 2).contiguous().transpose(1, 2) if nhd else x.contiguous())
        self.K, self.V = pools
        self.Ks, self.Vs = scales if int8 else (None, None)

    def widen(self):
        """More columns in the table than clusters take: the plan that puts all tiles in one line."""
        more = 8192 // self.page + 1
        junk = torch.randint(-2 ** 31, 2 ** 31 - 1, (self.B, more), generator=torch.Generator().manual_seed(more),
                             dtype=torch.int64).to(torch.int32).cuda()
        self.table = torch.cat([self.table, junk], 1).contiguous()
        self.cap = self.table.shape[1] * self.page
        return self

    def values(self):
        out = []
        for x, s in ((self.K, self.Ks), (self.V, self.Vs)):
            v = x.cpu().double()
            out.append((v * s.cpu().double()[..., None] if self.int8 else v).numpy())
        return out

    def attend(self, fqkv, q, **kw):
        if self.int8:
            return fqkv.decode_attn_gqa_int8_paged(q, self.K, self.V, self.Ks, self.Vs, self.table, self.lens, **kw)
        return fqkv.decode_attn_gqa_paged(q, self.K, self.V, self.table, self.lens, **kw)

    def check(self, fqkv, q, out, w_old=None, w_new=None):
        K, V = self.values()
        lens = self.lens.clamp(0, self.cap).tolist()
        r = op.paged_attention(q.cpu().double().numpy(), K, V, self.table.cpu().numpy(), lens)
        got = out.double().cpu().numpy()
        u = U8 if out.dtype == torch.bfloat16 else U16
        ds = (self.D + 8) * 2.0 ** -23 * r["smax"]
        tol = u * np.abs(r["out"]) + (U16 + 2 * ds[..., None] + 2.0 ** -17) * r["absum"] \
            + max(lens + [1]) * 2.0 ** -25 * r["vmax"] * (np.array(lens)[:, None, None] > 0)
        assert np.isfinite(got).all()
        assert (np.abs(got - r["out"]) <= tol).all(), float((np.abs(got - r["out"]) - tol).max())
        if w_new is not None:
            w_old, w_new = w_old.double().cpu().numpy(), w_new.double().cpu().numpy()
            G = q.shape[1] // self.Hkv
            for b, n in enumerate(lens):
                assert (w_new[b, :, n:] == w_old[b, :, n:]).all()  # slots past the length: untouched
                rel = (2 * ds[b] + 2.0 ** -18).reshape(self.Hkv, G, 1)
                p = r["p"][b].reshape(self.Hkv, G, n)
                want = w_old[b, :, :n] + p.sum(1)
                wtol = 2 * (rel * p).sum(1) + 2.0 ** -23 * np.abs(want) + 1e-37
                assert (np.abs(w_new[b, :, :n] - want) <= wtol).all()


def _q(B, Hq, D, seed=1, sigma=1.0):
    return (torch.randn(B, Hq, D, generator=torch.Generator().manual_seed(seed)) * sigma).half().cuda()


def _clean(fqkv):
    assert fqkv.ops.device_status(torch.device("cuda", 0)) == 0


# The two ways the work is split: a thread-block cluster per (sequence, KV head) for small capacities, all tiles in one
# line otherwise (and always when weights are accumulated).
PLANS = pytest.mark.parametrize("line", [False, True])

EDGE = [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200]


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 208])
@PLANS
def test_attention_edge_lengths(fqkv, int8, D, page, line):
    c = Cache(fqkv, EDGE, 2, D, page, int8, seed=page)
    if line:
        c.widen()
    q = _q(c.B, 8, D)
    c.check(fqkv, q, c.attend(fqkv, q))
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (5, 5), (6, 3), (7, 1), (8, 1), (9, 1), (16, 1), (17, 1), (40, 2), (32, 8)])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_head_layouts(fqkv, int8, Hq, Hkv, D):
    c = Cache(fqkv, [0, 301, 64, 90], Hkv, D, 16, int8, nhd=True, seed=Hq)
    q = _q(c.B, Hq, D, sigma=2.0)
    w = torch.rand(c.B, Hkv, c.cap, generator=torch.Generator().manual_seed(3)).cuda()
    w0 = w.clone()
    out = torch.full((c.B, Hq, D), 7.0, dtype=torch.bfloat16, device="cuda")
    assert c.attend(fqkv, q, out=out, weights=w) is out
    c.check(fqkv, q, out, w0, w)
    c.check(fqkv, q, c.attend(fqkv, q))
    c.check(fqkv, q, c.widen().attend(fqkv, q))
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens", [[5000], [4097, 1], [1, 0, 0, 2500], [0, 0, 0], [3] * 70 + [0] * 40 + [700] + [64] * 200,
                                  [0] * 300 + [130] + [1] * 555 + [0, 65]])
def test_attention_splits_and_batches(fqkv, int8, lens):
    """Units that cross many CTAs, and batches past one warp's scan, with and without the weights."""
    c = Cache(fqkv, lens, 1 if len(lens) > 9 else 2, 64, 32, int8, seed=len(lens))
    q = _q(c.B, 4, 64, sigma=3.0)
    out = c.attend(fqkv, q)
    c.check(fqkv, q, out)
    w = torch.zeros(c.B, c.Hkv, c.cap, device="cuda")
    w0 = w.clone()
    out2 = c.attend(fqkv, q, weights=w)
    c.check(fqkv, q, out2, w0, w)
    # nothing depends on timing (with weights the work may be split in another way: other last bits)
    assert torch.equal(out, c.attend(fqkv, q)) and torch.equal(out2, c.attend(fqkv, q, weights=w))
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
def test_attention_ignores_lengths_past_the_table(fqkv, int8):
    """Lengths are clamped to the table: negative ones are empty, larger ones end with the last page."""
    c = Cache(fqkv, [16, 48], 2, 64, 16, int8)
    c.table = c.table[:, :3].contiguous()
    c.cap = 48
    c.lens = torch.tensor([-5, 1000], dtype=torch.int32).cuda()
    q = _q(2, 4, 64)
    c.check(fqkv, q, c.attend(fqkv, q))
    _clean(fqkv)


@PLANS
def test_attention_int8_scales_of_every_size(fqkv, line):
    """Scales from subnormal to the largest, and zero, in one sequence: small ones keep their precision where
    they are alone, and a later large one rescales what came before."""
    c = Cache(fqkv, [400, 400, 400], 2, 128, 16, True)
    g = torch.Generator().manual_seed(5)
    e = torch.randint(-20, 4, (c.P, c.Hkv, c.page), generator=g).float()
    used = torch.isfinite(c.Vs)
    c.Vs = torch.where(used, torch.exp2(e).half().cuda(), c.Vs)
    for i in range(25):  # sequence 1: ascending over its pages; sequence 2: only subnormal and zero scales
        c.Vs[int(c.table[1, i])] = 2.0 ** (i - 20)
        c.Vs[int(c.table[2, i])] = 0.0 if i % 2 else 2.0 ** -23
    if line:
        c.widen()
    q = _q(3, 8, 128)
    out = c.attend(fqkv, q)
    K, V = c.values()
    r = op.paged_attention(q.cpu().double().numpy(), K, V, c.table.cpu().numpy(), [400] * 3)
    got, ds = out.double().cpu().numpy(), (128 + 8) * 2.0 ** -23 * r["smax"]
    # as the file's bound, but a term below the fp16 range is 2^-25 of a frame whose largest scale is at 2^13 or above
    tol = U16 * np.abs(r["out"]) + (U16 + 2 * ds[..., None] + 2.0 ** -17) * r["absum"] + 2.0 ** -25
    for b in range(3):
        vb = op.gather(V, c.table[b].cpu().numpy(), 400)
        tol[b] += 400 * 2.0 ** -38 * 2 * np.abs(vb).max()
    assert (np.abs(got - r["out"]) <= tol).all()
    _clean(fqkv)


@PLANS
def test_attention_masked_lowest_and_infinite_values(fqkv, line):
    """Rows whose scores reach the fp16 range's ends; an infinite key in an attended slot makes that row NaN only."""
    c = Cache(fqkv, [130, 130], 1, 64, 16, False)
    c.K[int(c.table[0, 2]), 0, 3] = 0
    c.K[int(c.table[0, 2]), 0, 3, 0] = -65504.0
    if line:
        c.widen()
    q = _q(2, 4, 64)
    c.check(fqkv, q, c.attend(fqkv, q))
    c.K[int(c.table[0, 2]), 0, 3, 0] = float("nan")
    out = c.attend(fqkv, q)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1]).all()
    _clean(fqkv)


def test_attention_pool_strides_halves_and_offsets(fqkv):
    """K and V as halves of one tensor, layers stacked, a table that is a slice, an odd start in the pool."""
    B, Hq, Hkv, D, page, P = 3, 8, 2, 64, 16, 40
    g = torch.Generator().manual_seed(9)
    kv = torch.randn(2, P, 2, Hkv, page, D, generator=g).half().cuda()  # [layer, page, K/V, ...]
    c = Cache(fqkv, [30, 77, 100], Hkv, D, page, False)
    c.K, c.V = kv[1, 3:, 0], kv[1, 3:, 1]
    wide = torch.full((B, 20), -1, dtype=torch.int32, device="cuda")
    wide[:, 5:5 + c.table.shape[1]] = c.table
    c.table = wide[:, 5:5 + c.table.shape[1]]
    q = _q(B, Hq, D)
    c.check(fqkv, q, c.attend(fqkv, q))
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
def test_one_page_per_sequence_is_the_dense_cache(fqkv, int8):
    B, Hq, Hkv, N, D = 3, 8, 2, 160, 128
    g = torch.Generator().manual_seed(2)
    K, V = (torch.randn(B, Hkv, N, D, generator=g).half().cuda() for _ in range(2))
    q = _q(B, Hq, D)
    table = torch.arange(B, dtype=torch.int32, device="cuda")[:, None]
    lens = torch.full((B,), N, dtype=torch.int32, device="cuda")
    if int8:
        (K, Ks), (V, Vs) = fqkv.qpt(K), fqkv.qpt(V)
        a, b = fqkv.decode_attn_gqa_int8_paged(q, K, V, Ks, Vs, table, lens), fqkv.decode_attn_gqa_int8(q, K, V, Ks, Vs)
    else:
        a, b = fqkv.decode_attn_gqa_paged(q, K, V, table, lens), fqkv.decode_attn_gqa(q, K, V, 8)
    # both sides within the file's bound of the same value, |v| <= 6 and |o| <= 1 for these draws
    assert float((a.float() - b.float()).abs().max()) <= 2 * (U16 + (U16 + 2.0 ** -12) * 6 + N * 2.0 ** -25 * 6)


@pytest.mark.parametrize("int8", [False, True])
def test_pool_past_32_bit_offsets(fqkv, int8):
    """Pages whose element offsets pass 2^32: attention, append and eviction reach the same far rows."""
    Hkv, D, page = 8, 128, 64
    P = (2 ** 32 + 2 ** 24) // (Hkv * D * page)
    dt = torch.int8 if int8 else torch.float16
    K, V = (torch.empty(P, Hkv, page, D, dtype=dt, device="cuda") for _ in range(2))
    Ks = Vs = None
    if int8:
        Ks, Vs = (torch.empty(P, Hkv, page, dtype=torch.float16, device="cuda") for _ in range(2))
    n, Hq = 100, 8
    table = torch.tensor([[P - 1, P - 3, 0]], dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(4)
    qkv = torch.randn(n, (Hq + 2 * Hkv) * D, generator=g).half().cuda()
    cos, sin = torch.ones(1, D // 2, device="cuda"), torch.zeros(1, D // 2, device="cuda")
    zero = torch.zeros(n, dtype=torch.int32, device="cuda")
    q_out = torch.empty(n, Hq, D, dtype=torch.float16, device="cuda")
    fqkv.rope_qkv_append_paged(qkv, cos, sin, zero, torch.arange(n, dtype=torch.int32, device="cuda"), table, q_out, K, V,
                               Ks, Vs, seq_ids=zero)
    c = Cache.__new__(Cache)
    c.B, c.Hkv, c.D, c.page, c.int8, c.cap = 1, Hkv, D, page, int8, 192
    c.lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = q_out[-1:].contiguous()
    c.K, c.V, c.Ks, c.Vs, c.table = K, V, Ks, Vs, table
    w = torch.zeros(1, Hkv, 192, device="cuda")
    out = c.attend(fqkv, q, weights=w)
    near = Cache.__new__(Cache)  # the same two pages in a small pool, for the oracle
    near.__dict__.update(c.__dict__)
    ids = [P - 1, P - 3]
    near.K, near.V = K[ids], V[ids]
    if int8:
        near.Ks, near.Vs = Ks[ids], Vs[ids]
    near.table = torch.tensor([[0, 1, 7]], dtype=torch.int32, device="cuda")
    near.check(fqkv, q, out, torch.zeros_like(w), w)
    k = near.K.double() if not int8 else near.K.double() * near.Ks.double()[..., None]
    src = qkv.view(n, -1, D)[:, Hq:Hq + Hkv].double()
    for j in (0, 63, 64, 99):
        d = (k[j // 64, :, j % 64] - src[j]).abs().max()
        assert float(d) <= (float(src[j].abs().max()) / 127 if int8 else 0.0)
    before = [x[ids].clone() for x in (K, V)]
    new = fqkv.evict_kvcache_paged(K, V, table, c.lens, w.clone(), 70, 20, Ks, Vs)
    assert new.tolist() == [70]
    wn = w.cpu().numpy()
    for h in range(Hkv):
        keep = op.kept_tokens(wn[0, h, :n], 70, 20)
        for x, old in zip((K, V), before):
            now = torch.cat([x[P - 1, h], x[P - 3, h]])[:70]
            assert torch.equal(now, torch.cat([old[0, h], old[1, h]])[torch.from_numpy(keep).cuda()])
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
@PLANS
def test_bad_page_is_reported_and_stays_inside_its_sequence(fqkv, int8, line):
    c = Cache(fqkv, [40, 100, 33], 2, 64, 16, int8)
    if line:
        c.widen()
    q = _q(3, 8, 64)
    good = c.attend(fqkv, q).clone()
    for bad in (c.P, -1, 2 ** 31 - 1, -2 ** 31):
        t = c.table.clone()
        t[1, 2] = bad
        c2 = Cache.__new__(Cache)
        c2.__dict__.update(c.__dict__)
        c2.table = t
        out = c2.attend(fqkv, q)
        with pytest.raises(RuntimeError, match="page outside the pool"):
            fqkv.ops.check_device_status(torch.device("cuda", 0), "paged decode")
        assert torch.equal(out[0], good[0]) and torch.equal(out[2], good[2])
    _clean(fqkv)


@PLANS
def test_attention_stalled_pipeline_gives_up(fqkv, line):
    """The failure path of the other decode kernels: tiles that never arrive end the launch with status 61."""
    lib = fqkv.native.lib()
    for int8 in (False, True):
        c = Cache(fqkv, [300, 70], 2, 128, 16, int8)
        if line:
            c.widen()
        q = _q(2, 8, 128)
        lib.fqkv_set_wait_timeout_ms(50)
        lib.fqkv_debug_skip_loads(1)
        try:
            c.attend(fqkv, q)
            torch.cuda.synchronize()
        finally:
            lib.fqkv_debug_skip_loads(0)
            lib.fqkv_set_wait_timeout_ms(2000)
        st = ctypes.c_int(-1)
        fqkv.native.check(lib.fqkv_device_status(ctypes.byref(st), 1), "status")
        assert st.value == 61
        c.check(fqkv, q, c.attend(fqkv, q))
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
def test_attention_graph_follows_lengths_and_shares_a_workspace(fqkv, int8):
    """Two captured calls on one workspace, replayed in turn as lengths and tables change; then another stream."""
    c = Cache(fqkv, [400, 260, 5], 2, 64, 16, int8)
    d = Cache(fqkv, [64, 1, 500], 2, 64, 16, int8, seed=8)
    q = _q(3, 8, 64)
    nb = max(fqkv.paged_workspace_bytes("int8" if int8 else "fp16", 3, 8, 2, x.cap, 64, weights=True) for x in (c, d))
    ws = torch.empty(nb, dtype=torch.uint8, device="cuda")
    outs = [torch.empty(3, 8, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    ws_w = [torch.zeros(3, 2, x.cap, device="cuda") for x in (c, d)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x, o, w in zip((c, d), outs, ws_w):
            x.attend(fqkv, q, out=o, workspace=ws, weights=w)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for x, o, w in zip((c, d), outs, ws_w):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.attend(fqkv, q, out=o, workspace=ws, weights=w)
        graphs.append(g)
    for lens in ([400, 260, 5], [1, 0, 3], [399, 17, 0]):
        c.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        for w in ws_w:
            w.zero_()
        for g in graphs * 2:
            g.replay()
        torch.cuda.synchronize()
        for x, o, w in zip((c, d), outs, ws_w):
            x.check(fqkv, q, o, torch.zeros_like(w), w / 2)
    with torch.cuda.stream(side):
        d.attend(fqkv, q, out=outs[0], weights=ws_w[0].new_zeros(ws_w[1].shape))
    side.synchronize()
    assert torch.equal(outs[0], outs[1])
    # without weights: the cluster plan, captured, and eager on the other stream
    with torch.cuda.stream(side):
        d.attend(fqkv, q, out=outs[1])
    side.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        d.attend(fqkv, q, out=outs[0])
    for lens in ([64, 1, 500], [0, 1, 480], [3, 0, 0]):
        d.lens.copy_(torch.tensor(lens, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        d.check(fqkv, q, outs[0])
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("lens,Hkv", [([8000], 1), ([3900, 10], 8), ([2000, 1, 0, 700, 2040, 5, 64, 1999], 8), ([120] * 9, 3),
                                      ([6000], 1), ([3900, 10, 2500, 64], 8), ([1000] * 9, 8), ([1000] * 14 + [0, 1, 513, 512], 8)])
def test_attention_clusters_of_every_size(fqkv, int8, lens, Hkv):
    """Sixteen, eight, four and two CTAs per unit, with CTAs that get no tile."""
    c = Cache(fqkv, lens, Hkv, 128, 64, int8, seed=len(lens), extra_pages=0)
    q = _q(c.B, Hkv * 3, 128, sigma=2.0)
    out = c.attend(fqkv, q)
    c.check(fqkv, q, out)
    assert torch.equal(out, c.attend(fqkv, q))
    _clean(fqkv)


# ------------------------------------------------------------------ append
def _tables(rows, D, base=10000.0):
    inv = base ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    a = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return a.cos().float().cuda(), a.sin().float().cuda()


def _check_append(fqkv, c, before, qkv, cos, sin, pos, axes, slots, seqs, q_out, q_before):
    """What an append into the fp16 cache c left, against float64; returns nothing."""
    T, Hq, D = q_out.shape
    Hkv = c.Hkv
    x = qkv[:, :(Hq + 2 * Hkv) * D].cpu().double().numpy().reshape(T, -1, D)
    y, a = op.rope(x[:, :Hq + Hkv], cos.cpu().numpy(), sin.cpu().numpy(), pos.cpu().numpy(), axes)
    # three fp32 roundings of terms up to a, then fp16 (2^-25: half its smallest step)
    tol = U16 * np.abs(y) + 2.0 ** -22 * a + 2.0 ** -25
    got_q = q_out.cpu().double().numpy()
    wantK, wantV = (p.cpu().double().numpy().copy() for p in before)
    K, V = c.K.cpu().double().numpy(), c.V.cpu().double().numpy()
    touched = np.zeros(K.shape[:3], bool)
    for t in range(T):
        s = int(slots[t])
        if s < 0:
            assert torch.equal(q_out[t], q_before[t])
            continue
        assert (np.abs(got_q[t] - y[t, :Hq]) <= tol[t, :Hq]).all()
        pg, off = int(c.table[int(seqs[t]), s // c.page]), s % c.page
        assert (np.abs(K[pg, :, off] - y[t, Hq:]) <= tol[t, Hq:]).all()
        wantV[pg, :, off] = torch.from_numpy(x[t, Hq + Hkv:]).half().double().numpy()
        touched[pg, :, off] = True
    np.testing.assert_array_equal(V, wantV)
    np.testing.assert_array_equal(K[~touched], wantK[~touched])


@pytest.mark.parametrize("model", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,Hq,Hkv,axes,interleaved", [(64, 8, 2, 1, False), (128, 7, 7, 3, False), (64, 3, 1, 3, True),
                                                        (128, 33, 11, 2, True), (128, 1, 1, 1, False)])
@pytest.mark.parametrize("tokens", ["decode", "packed", "many", "prefill"])
def test_append(fqkv, model, D, Hq, Hkv, axes, interleaved, tokens):
    g = torch.Generator().manual_seed(D + Hq)
    lens = [5, 0, 31, 16] if tokens in ("decode", "packed") else [0, 0]
    room = {"decode": 1, "packed": 17, "many": 300, "prefill": 900}[tokens]  # prefill: more than 1000 tokens, the other kernel
    cos, sin = _tables(500, D)
    sec = {1: [D // 2], 2: [D // 2 - 9, 9], 3: [D // 2 - 2 * (D // 8), D // 8, D // 8]}[axes]
    amap = fqkv.rope_axes(sec, interleaved)
    for int8 in (False, True):
        c = Cache(fqkv, lens, Hkv, D, 16, int8, nhd=Hq == 3, room=room)
        c.K = torch.nan_to_num(c.K.float(), 1.0, 2.0, 3.0).to(c.K.dtype) if not int8 else c.K
        c.V = torch.nan_to_num(c.V.float(), 1.0, 2.0, 3.0).to(c.V.dtype) if not int8 else c.V
        if tokens == "decode":
            T, slots, seqs = c.B, c.lens.clone(), None
            slots[2] = -1
            seq_list = torch.arange(c.B)
        else:
            pairs = [(b, lens[b] + i) for b in range(c.B) for i in range(room)]
            order = torch.randperm(len(pairs), generator=torch.Generator().manual_seed(1)).tolist()
            pairs = [pairs[i] for i in order] + [(0, -1), (10 ** 9, -7)]  # padding tokens may name any sequence
            T = len(pairs)
            slots = torch.tensor([s for _, s in pairs], dtype=torch.int32).cuda()
            seq_list = torch.tensor([b for b, _ in pairs])
            seqs = seq_list.to(torch.int32).cuda()
        wide = torch.randn(T, (Hq + 2 * Hkv) * D + 24, generator=torch.Generator().manual_seed(6)).to(model).cuda()
        qkv = wide[:, 8:8 + (Hq + 2 * Hkv) * D]  # rows 16 bytes into a wider tensor
        if not int8:  # both caches take the same tokens
            pos = torch.randint(500, (axes, T), generator=g, dtype=torch.int32).cuda()
        q_out = torch.full((T, Hq, D), 3.0, dtype=torch.float16, device="cuda")
        q0, kv0 = q_out.clone(), (c.K.clone(), c.V.clone())
        args = (qkv, cos, sin, pos if axes > 1 else pos[0], slots, c.table, q_out, c.K, c.V)
        kw = dict(axes=amap if axes > 1 else None, seq_ids=seqs)
        fqkv.rope_qkv_append_paged(*args, c.Ks, c.Vs, **kw)
        if not int8:
            _check_append(fqkv, c, kv0, qkv, cos, sin, pos, amap.cpu().numpy(), slots.cpu(), seq_list, q_out, q0)
            first = c, q_out, slots.cpu(), seq_list
            continue
        # int8: the quantizer's codes and scale of the very rows that the fp16 cache got
        f, fq, sl, sq = first
        assert torch.equal(fq, q_out)
        for t in range(T):
            s = int(sl[t])
            if s < 0:
                continue
            at = lambda x: (int(x.table[int(sq[t]), s // 16]), slice(None), s % 16)  # noqa: E731
            for half, codes, sc in ((f.K, c.K, c.Ks), (f.V, c.V, c.Vs)):
                want, ws = oq.quantize_int8_per_token(half[at(f)].cpu().numpy())
                np.testing.assert_array_equal(codes[at(c)].cpu().numpy(), want)
                np.testing.assert_array_equal(sc[at(c)].cpu().numpy(), ws)
    _clean(fqkv)


def test_append_int8_zero_tiny_and_nonfinite_rows(fqkv):
    """Rows of zeros, subnormals, inf and NaN take the quantizer's own rules."""
    D, T = 64, 6
    c = Cache(fqkv, [0], 1, D, 16, True, room=T)
    qkv = torch.randn(T, 3 * D, generator=torch.Generator().manual_seed(1)).half().cuda()
    qkv[0] = 0
    qkv[1] = 2.0 ** -24
    qkv[2, 2 * D + 5] = float("inf")
    qkv[3, 2 * D + 7] = float("nan")
    qkv[4, 2 * D:] = 65504.0
    cos, sin = torch.ones(1, D // 2, device="cuda"), torch.zeros(1, D // 2, device="cuda")
    i = torch.arange(T, dtype=torch.int32, device="cuda")
    fqkv.rope_qkv_append_paged(qkv, cos, sin, torch.zeros_like(i), i, c.table, torch.empty(T, 1, D, dtype=torch.float16,
                               device="cuda"), c.K, c.V, c.Ks, c.Vs, seq_ids=torch.zeros_like(i))
    pg = int(c.table[0, 0])
    for off, codes, sc in ((D, c.K, c.Ks), (2 * D, c.V, c.Vs)):
        want, ws = oq.quantize_int8_per_token(qkv[:, off:off + D].cpu().numpy())
        np.testing.assert_array_equal(codes[pg, 0, :T].cpu().numpy(), want)
        np.testing.assert_array_equal(sc[pg, 0, :T].cpu().numpy(), ws)
    _clean(fqkv)


@pytest.mark.parametrize("what", ["slot", "sequence", "position", "axis", "page"])
def test_append_out_of_range_token_is_reported_and_not_written(fqkv, what):
    D, Hkv, T = 64, 2, 3
    c = Cache(fqkv, [4, 4, 4], Hkv, D, 16, False, room=1)
    c.K, c.V = torch.zeros_like(c.K), torch.zeros_like(c.V)
    cos, sin = _tables(32, D)
    pos = torch.tensor([[1, 2, 3], [4, 5, 6]], dtype=torch.int32).cuda()
    slots, seqs = c.lens.clone(), torch.arange(3, dtype=torch.int32, device="cuda")
    axes = fqkv.rope_axes([20, 12])
    if what == "slot":
        slots[1] = c.cap
    elif what == "sequence":
        seqs[1] = 3
    elif what == "position":
        pos[1, 1] = 32
    elif what == "page":
        c.table[1, 0] = c.P
    else:
        axes[7] = 2
    q_out = torch.full((T, 4, D), 5.0, dtype=torch.float16, device="cuda")
    qkv = torch.randn(T, 8 * D, generator=torch.Generator().manual_seed(1)).half().cuda()
    fqkv.rope_qkv_append_paged(qkv, cos, sin, pos, slots, c.table, q_out, c.K, c.V, axes=axes, seq_ids=seqs)
    with pytest.raises(RuntimeError, match="page outside" if what == "page" else "out of range"):
        fqkv.ops.check_device_status(torch.device("cuda", 0), "append")
    if what != "axis":
        assert (q_out[1] == 5).all() and not (q_out[0] == 5).all() and not (q_out[2] == 5).all()
        rows = c.V.abs().sum((1, 3)) > 0
        assert int(rows.sum()) == 2
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
def test_append_prefill_with_bad_tokens_and_padding(fqkv, int8):
    """Among 1500 tokens some are padding and one of each kind is out of range: only those are left out."""
    D, Hq, Hkv, T = 128, 4, 2, 1500
    c = Cache(fqkv, [0, 0], Hkv, D, 32, int8, room=800)
    c.K, c.V = torch.zeros_like(c.K), torch.zeros_like(c.V)
    cos, sin = _tables(64, D)
    i = torch.arange(T, dtype=torch.int32)
    slots, seqs, pos = i % 750, i // 750, torch.stack([i % 64, i % 63, i % 62])
    c.table[1, 9] = c.P + 5                        # slots 288 .. 319 of sequence 1: tokens 1038 .. 1069
    slots[7], seqs[8], pos[1, 9], slots[10] = c.cap, 2, 64, -1
    bad = [7, 8, 9, 10] + list(range(1038, 1070))
    qkv = (torch.rand(T, (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1)) + 0.5).bfloat16().cuda()
    q_out = torch.full((T, Hq, D), 5.0, dtype=torch.float16, device="cuda")
    fqkv.rope_qkv_append_paged(qkv, cos, sin, pos.contiguous().cuda(), slots.cuda(), c.table, q_out, c.K, c.V, c.Ks, c.Vs,
                               axes=fqkv.rope_axes([16, 24, 24]), seq_ids=seqs.cuda())
    with pytest.raises(RuntimeError, match="page outside|out of range"):
        fqkv.ops.check_device_status(torch.device("cuda", 0), "append")
    left = (q_out == 5).flatten(1).all(1).cpu()
    assert left.nonzero().flatten().tolist() == bad
    written = (c.V != 0).flatten(3).any(3).any(1)   # v is never 0 here
    want = torch.zeros_like(written)
    for t in range(T):
        if t not in bad:
            want[int(c.table[int(seqs[t]), int(slots[t]) // 32]), int(slots[t]) % 32] = True
    assert torch.equal(written, want)
    _clean(fqkv)


def test_append_stalled_pipeline_gives_up(fqkv):
    """Rows that never arrive: the prefill kernel's waits end with status 61 and the context stays usable."""
    lib = fqkv.native.lib()
    D, Hq, Hkv, T = 64, 4, 2, 1200
    c = Cache(fqkv, [0, 0], Hkv, D, 16, False, room=600)
    cos, sin = _tables(600, D)
    i = torch.arange(T, dtype=torch.int32).cuda()
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=torch.Generator().manual_seed(1)).half().cuda()
    q_out = torch.zeros(T, Hq, D, dtype=torch.float16, device="cuda")
    call = lambda: fqkv.rope_qkv_append_paged(qkv, cos, sin, i % 600, i % 600, c.table, q_out, c.K, c.V,  # noqa: E731
                                              seq_ids=i // 600)
    lib.fqkv_set_wait_timeout_ms(50)
    lib.fqkv_debug_skip_loads(1)
    try:
        call()
        torch.cuda.synchronize()
    finally:
        lib.fqkv_debug_skip_loads(0)
        lib.fqkv_set_wait_timeout_ms(2000)
    assert fqkv.ops.device_status(torch.device("cuda", 0)) == 61
    call()
    torch.cuda.synchronize()
    assert bool((q_out != 0).flatten(1).any(1).all())
    _clean(fqkv)


# ------------------------------------------------------------------ eviction
def _evict_check(fqkv, c, w, budget, recent, in_place=False):
    lens = c.lens.tolist()
    table = c.table.cpu().numpy()
    pools = [c.K, c.V] + ([c.Ks, c.Vs] if c.int8 else [])
    want = [p.cpu().clone() for p in pools]
    w0 = w.cpu().numpy().copy()
    wout = w if in_place else torch.full_like(w, -3.0)
    want_w = w0.copy() if in_place else np.full_like(w0, -3.0)
    for b, n in enumerate(lens):
        for h in range(c.Hkv):
            if n <= budget:
                want_w[b, h, :n] = w0[b, h, :n]
                continue
            keep = op.kept_tokens(w0[b, h, :n], budget, recent)
            src = [(int(table[b, j // c.page]), int(j % c.page)) for j in keep]
            rows = [[p[pg, h, s].clone() for pg, s in src] for p in want]
            for i in range(budget):
                for p, r in zip(want, rows):
                    p[int(table[b, i // c.page]), h, i % c.page] = r[i]
            want_w[b, h, :n] = 0
            want_w[b, h, :budget] = w0[b, h, keep]
    lens_out = c.lens if in_place else None
    new = fqkv.evict_kvcache_paged(c.K, c.V, c.table, c.lens, w, budget, recent, c.Ks, c.Vs,
                                   weights_out=None if in_place else wout, lens_out=lens_out)
    assert new.tolist() == [min(n, budget) for n in lens]
    for p, x in zip(pools, want):
        a, b = p.cpu(), x
        view = torch.int8 if p.dtype == torch.int8 else torch.int16
        assert torch.equal(a.contiguous().view(view), b.contiguous().view(view))
    np.testing.assert_array_equal(wout.cpu().numpy(), want_w)


@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("page", [16, 48, 64])
@pytest.mark.parametrize("budget,recent", [(1, 0), (1, 1), (40, 7), (64, 64), (64, 0), (65, 1), (300, 100), (5000, 3)])
def test_evict(fqkv, int8, D, page, budget, recent):
    c = Cache(fqkv, [0, 1, 64, 65, 66, 301, 500], 2, D, page, int8, nhd=page == 48, seed=budget)
    g = torch.Generator().manual_seed(budget + recent)
    w = torch.rand(c.B, 2, c.cap, generator=g).mul(16).floor().cuda()  # 16 values: ties everywhere
    _evict_check(fqkv, c, w, budget, recent, in_place=recent % 2 == 1)
    _clean(fqkv)


@pytest.mark.parametrize("n,budget,recent", [(40000, 9000, 100), (40000, 39999, 0), (70001, 257, 256), (20000, 1, 0)])
def test_evict_long(fqkv, n, budget, recent):
    c = Cache(fqkv, [n], 1, 64, 256, False, seed=n)
    g = torch.Generator().manual_seed(n)
    w = torch.randn(1, 1, c.cap, generator=g).exp().cuda()
    _evict_check(fqkv, c, w, budget, recent)
    c2 = Cache(fqkv, [n], 1, 64, 256, True, seed=n)
    w2 = (w * 4).floor()
    _evict_check(fqkv, c2, w2, budget, recent, in_place=True)
    _clean(fqkv)


@pytest.mark.parametrize("lens,Hkv,budget,recent", [([100001, 77], 1, 700, 30), ([26001, 40, 31000, 0] + [301] * 20, 4, 300, 11),
                                                    ([26001] + [9] * 8, 4, 6000, 0)])
def test_evict_long_by_clusters_and_by_one_block(fqkv, lens, Hkv, budget, recent):
    """Eight blocks per selection; one block in several steps, where there are many (sequence, head) pairs."""
    c = Cache(fqkv, lens, Hkv, 64, 64, False, seed=budget)
    w = torch.randn(c.B, Hkv, c.cap, generator=torch.Generator().manual_seed(budget)).exp().mul(8).floor().cuda()
    _evict_check(fqkv, c, w, budget, recent)
    _clean(fqkv)


def test_evict_odd_weights(fqkv):
    """NaN above +inf above numbers, both zeros alike, negative weights, all equal."""
    c = Cache(fqkv, [200, 200, 200, 200], 1, 64, 16, False)
    w = torch.randn(4, 1, c.cap, generator=torch.Generator().manual_seed(3))
    w[0, 0, ::7] = float("nan")
    w[0, 0, 1::7] = float("inf")
    w[0, 0, 2::7] = -float("inf")
    w[1] = 0.0
    w[1, 0, ::2] = -0.0
    w[2] = float("nan")
    w[3] = -w[3].abs()
    for budget, recent in ((20, 3), (60, 10), (199, 0)):
        c = Cache(fqkv, [200, 200, 200, 200], 1, 64, 16, False)
        _evict_check(fqkv, c, w.cuda(), budget, recent)
    _clean(fqkv)


def test_evict_already_in_place_and_single_gap(fqkv):
    """Nothing but the last tokens to drop; and one gap in the middle of many chunks."""
    for gap in (None, 0, 777, 1999):
        c = Cache(fqkv, [2000], 2, 128, 16, False, seed=1)
        w = torch.ones(1, 2, c.cap, device="cuda")
        if gap is not None:
            w[:, :, gap] = 0
        _evict_check(fqkv, c, w, 1999, 0)
    _clean(fqkv)


def test_evict_bad_page_is_reported(fqkv):
    c = Cache(fqkv, [100, 100], 1, 64, 16, False)
    w = torch.rand(2, 1, c.cap, generator=torch.Generator().manual_seed(1)).cuda()
    good = Cache(fqkv, [100, 100], 1, 64, 16, False)
    fqkv.evict_kvcache_paged(good.K, good.V, good.table, good.lens, w.clone(), 50, 10)
    c.table[0, 3] = -1
    fqkv.evict_kvcache_paged(c.K, c.V, c.table, c.lens, w.clone(), 50, 10)
    with pytest.raises(RuntimeError, match="page outside the pool"):
        fqkv.ops.check_device_status(torch.device("cuda", 0), "eviction")
    for i in range(4):  # the other sequence is whole
        pg = int(c.table[1, i])
        assert torch.equal(c.K[pg].view(torch.int16), good.K[pg].view(torch.int16))
    _clean(fqkv)


# ------------------------------------------------------------------ calls at the edges of what is documented
@pytest.mark.parametrize("int8", [False, True])
def test_zero_queries_and_tiny_capacities(fqkv, int8):
    """q = 0 is the mean over the tokens; a capacity of one tile needs no parts, with weights and without."""
    c = Cache(fqkv, [16, 3, 0, 1], 2, 64, 16, int8)
    assert c.cap == 32
    q = _q(4, 6, 64)
    q[0] = 0
    q[1, 2] = 0
    c.check(fqkv, q, c.attend(fqkv, q))
    w = torch.rand(4, 2, c.cap, generator=torch.Generator().manual_seed(2)).cuda()
    w0 = w.clone()
    c.check(fqkv, q, c.attend(fqkv, q, weights=w), w0, w)
    c.check(fqkv, q, c.widen().attend(fqkv, q))
    _clean(fqkv)


def test_empty_batches_and_no_tokens(fqkv):
    K = torch.zeros(2, 1, 16, 64, dtype=torch.float16, device="cuda")
    none, table = torch.zeros(0, dtype=torch.int32, device="cuda"), torch.zeros(0, 3, dtype=torch.int32, device="cuda")
    out = fqkv.decode_attn_gqa_paged(K.new_zeros(0, 2, 64), K, K, table, none)
    assert out.shape == (0, 2, 64)
    assert fqkv.evict_kvcache_paged(K, K, table, none, torch.zeros(0, 1, 48, device="cuda"), 4, 1).shape == (0,)
    cos = torch.ones(4, 32, device="cuda")
    one = torch.zeros(1, 3, dtype=torch.int32, device="cuda")
    fqkv.rope_qkv_append_paged(K.new_zeros(0, 4 * 64), cos, cos, none, none, one, K.new_zeros(0, 2, 64), K, K)
    _clean(fqkv)


@pytest.mark.parametrize("int8", [False, True])
def test_two_streams_at_once(fqkv, int8):
    """Eight calls on two streams, nothing waiting between them, each with its own scratch: the results of calls
    made alone."""
    caches = [Cache(fqkv, lens, 2, 64, 16, int8, seed=i) for i, lens in enumerate(([700, 90, 3], [33, 1200, 64]))]
    caches[1].widen()
    q = _q(3, 8, 64)
    alone = [c.attend(fqkv, q).clone() for c in caches]
    w = [torch.rand(3, 2, c.cap, generator=torch.Generator().manual_seed(4)).cuda() for c in caches]
    kept = []
    for c, x in zip(caches, w):  # an eviction made alone, on copies
        k, v = c.K.clone(), c.V.clone()
        extra = (None, None) if not int8 else (c.Ks.clone(), c.Vs.clone())
        fqkv.evict_kvcache_paged(k, v, c.table, c.lens, x.clone(), 50, 9, *extra)
        kept.append((k, v))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(4):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                outs[i].append(caches[i].attend(fqkv, q))
    for i, st in enumerate(streams):
        with torch.cuda.stream(st):
            fqkv.evict_kvcache_paged(caches[i].K, caches[i].V, caches[i].table, caches[i].lens, w[i], 50, 9, caches[i].Ks,
                                     caches[i].Vs)
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])
        for a, b in zip((caches[i].K, caches[i].V), kept[i]):
            dt = torch.int8 if int8 else torch.int16
            assert torch.equal(a.contiguous().view(dt), b.contiguous().view(dt))
    _clean(fqkv)


def test_sliced_positions_and_tables(fqkv):
    """Rows of wider tensors for positions, the table and the pools, in the append and the eviction."""
    D, Hq, Hkv, page, B = 64, 4, 2, 16, 3
    g = torch.Generator().manual_seed(3)
    big = torch.zeros(2, 12, Hkv, page, D, dtype=torch.float16, device="cuda")
    K, V = big[0, 1:], big[1, 1:]
    wide = torch.full((B, 9), -5, dtype=torch.int32, device="cuda")
    wide[:, 4:6] = torch.tensor([[3, 7], [0, 5], [9, 2]], dtype=torch.int32)
    table = wide[:, 4:7]
    cos, sin = _tables(64, D)
    T = 3 * 20
    pos_wide = torch.randint(64, (5, T + 13), generator=g, dtype=torch.int32).cuda()
    pos = pos_wide[1:3, 6:6 + T]
    seqs = (torch.arange(T, dtype=torch.int32) // 20).cuda()
    slots = (torch.arange(T, dtype=torch.int32) % 20).cuda()
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).half().cuda()
    axes = fqkv.rope_axes([20, 12])
    q1, q2 = (torch.empty(T, Hq, D, dtype=torch.float16, device="cuda") for _ in range(2))
    fqkv.rope_qkv_append_paged(qkv, cos, sin, pos, slots, table, q1, K, V, axes=axes, seq_ids=seqs)
    K2, V2 = torch.zeros_like(K).contiguous(), torch.zeros_like(V).contiguous()
    fqkv.rope_qkv_append_paged(qkv, cos, sin, pos.contiguous(), slots, table.contiguous(), q2, K2, V2, axes=axes, seq_ids=seqs)
    assert torch.equal(q1, q2) and torch.equal(K, K2) and torch.equal(V, V2) and float(K2.abs().sum()) > 0
    assert float(big[:, 0].abs().sum()) == 0
    lens = torch.full((B,), 20, dtype=torch.int32, device="cuda")
    w = torch.rand(B, Hkv, 3 * page, generator=g).cuda()
    a = fqkv.evict_kvcache_paged(K, V, table, lens, w.clone(), 9, 4)
    b = fqkv.evict_kvcache_paged(K2, V2, table.contiguous(), lens, w.clone(), 9, 4)
    assert torch.equal(a, b) and torch.equal(K, K2) and torch.equal(V, V2)
    _clean(fqkv)


def test_refusals_of_the_python_layer(fqkv):
    c = Cache(fqkv, [20, 5], 2, 64, 16, False)
    i8 = Cache(fqkv, [20, 5], 2, 64, 16, True)
    q = _q(2, 4, 64)
    w = torch.zeros(2, 2, c.cap, device="cuda")

    def attn(match, **kw):
        a = dict(q=q, K=c.K, V=c.V, block_table=c.table, seq_lens=c.lens)
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            fqkv.decode_attn_gqa_paged(**a)

    attn("^fp16", q=q.float())
    attn("^fp16", q=q.transpose(1, 2).contiguous().transpose(1, 2))
    attn("^shape", q=q[:1])
    attn("^shape", V=c.V[:1])
    attn("^fp16", K=i8.K, V=i8.V)
    attn("^stride", K=c.K.transpose(2, 3).contiguous().transpose(2, 3))
    attn("^D", K=c.K[..., :32], V=c.V[..., :32], q=q[..., :32].contiguous())
    attn("^block_table", block_table=c.table.long())
    attn("^seq_lens", seq_lens=c.lens.long())
    attn("^seq_lens", seq_lens=c.lens[:1])
    attn("^cuda", seq_lens=c.lens.cpu())
    attn("^weights", weights=w[:, :1])
    attn("^weights", weights=w.half())
    attn("^dtype", out=torch.empty(2, 4, 64, device="cuda"))
    attn("^shape", out=torch.empty(2, 4, 32, dtype=torch.float16, device="cuda"))
    attn("^workspace", workspace=torch.empty(1000, dtype=torch.uint8))
    attn("needed", workspace=torch.empty(16, dtype=torch.uint8, device="cuda"), weights=w)
    attn("multiple of 16", K=c.K[:, :, :8], V=c.V[:, :, :8])
    attn("multiple of Hkv", q=_q(2, 3, 64))
    with pytest.raises(RuntimeError, match="^fp16"):
        fqkv.decode_attn_gqa_int8_paged(q, i8.K, i8.V, i8.Ks, None, i8.table, i8.lens)
    with pytest.raises(RuntimeError, match="^shape"):
        fqkv.decode_attn_gqa_int8_paged(q, i8.K, i8.V, i8.Ks[:1], i8.Vs, i8.table, i8.lens)

    def evict(match, **kw):
        a = dict(K=c.K, V=c.V, block_table=c.table, seq_lens=c.lens, weights=w, budget=4, recent=1)
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            fqkv.evict_kvcache_paged(**a)

    evict("budget", budget=0, recent=0)
    evict("budget", budget=-3, recent=-3)
    evict("recent", budget=0)
    evict("recent", recent=5)
    evict("^weights", weights=w[:, :, :-1])
    evict("^weights_out", weights_out=w.double())
    evict("^lens_out", lens_out=c.lens[:1])
    evict("^fp16", Ks=i8.Ks)
    evict("needed", workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))
    both = torch.zeros(w.numel() + 16, device="cuda")
    evict("overlap", weights=both[:w.numel()].view(w.shape), weights_out=both[16:].view(w.shape))

    cos = torch.ones(8, 32, device="cuda")
    qkv = torch.zeros(2, 8 * 64, dtype=torch.float16, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")

    def append(match, **kw):
        a = dict(qkv=qkv, cos_table=cos, sin_table=cos, positions=i, slots=i, block_table=c.table, q_out=q.clone(), K=c.K, V=c.V)
        a.update(kw)
        with pytest.raises(RuntimeError, match=match):
            fqkv.rope_qkv_append_paged(**a)

    append("^dtype", qkv=qkv.float())
    append("^shape", qkv=qkv[:, :-64])
    append("^shape", qkv=qkv[:1])
    append("^tables", cos_table=cos.half())
    append("^tables", sin_table=cos[:, :16])
    append("^positions", positions=i[:1])
    append("^axes", positions=torch.stack([i, i]))
    append("^axes", positions=torch.stack([i, i]), axes=i)
    append("^slots", slots=i.long())
    append("^seq_ids", seq_ids=i[:1])
    append("aligned", qkv=torch.zeros(2, 8 * 64 + 4, dtype=torch.float16, device="cuda")[:, 4:])
    _clean(fqkv)


def test_one_position_row_for_all_axes(fqkv):
    """Text tokens: the same position on every axis, as an expanded view; as one axis."""
    D, Hq, Hkv, T = 128, 4, 1, 5
    g = torch.Generator().manual_seed(8)
    cos, sin = _tables(64, D)
    K, V, K2, V2 = (torch.zeros(T, Hkv, 16, D, dtype=torch.float16, device="cuda") for _ in range(4))
    table = torch.arange(T, dtype=torch.int32, device="cuda")[:, None]
    pos = torch.randint(64, (T,), generator=g, dtype=torch.int32).cuda()
    slots = torch.arange(T, dtype=torch.int32, device="cuda")
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).to(torch.bfloat16).cuda()
    q1, q2 = (torch.empty(T, Hq, D, dtype=torch.float16, device="cuda") for _ in range(2))
    fqkv.rope_qkv_append_paged(qkv, cos, sin, pos.expand(3, T), slots, table, q1, K, V, axes=fqkv.rope_axes([20, 22, 22]))
    fqkv.rope_qkv_append_paged(qkv, cos, sin, pos, slots, table, q2, K2, V2)
    assert torch.equal(q1, q2) and torch.equal(K, K2) and torch.equal(V, V2) and float(K.abs().sum()) > 0
    _clean(fqkv)


def test_a_budget_past_every_integer_evicts_nothing(fqkv):
    c = Cache(fqkv, [20, 5], 2, 64, 16, False)
    w = torch.rand(2, 2, c.cap, device="cuda")
    k, w0 = c.K.clone(), w.clone()
    assert fqkv.evict_kvcache_paged(c.K, c.V, c.table, c.lens, w, 2 ** 64 + 1, 2 ** 64).tolist() == [20, 5]
    assert torch.equal(c.K.view(torch.int16), k.view(torch.int16)) and torch.equal(w, w0)
    _clean(fqkv)


@pytest.mark.parametrize("wide", [False, True])
def test_a_zero_probability_times_an_infinite_value(fqkv, wide):
    """A key of score -inf in one tile whose value is inf: 0 * inf is NaN in both plans, as in the definition."""
    B, D, page = 1, 64, 16
    K = torch.zeros(40, 1, page, D, dtype=torch.float16, device="cuda")
    V = torch.ones(40, 1, page, D, dtype=torch.float16, device="cuda")
    q = torch.zeros(B, 2, D, dtype=torch.float16, device="cuda")
    q[:, :, 0] = 1
    K[:4, :, :, 0] = float("-inf")  # the whole first tile of 64 keys
    V[1, 0, 3, 7] = float("inf")
    table = torch.arange(40, dtype=torch.int32, device="cuda")[None]
    if wide:
        table = torch.cat([table, table.new_zeros(1, 1000)], 1).contiguous()
    out = fqkv.decode_attn_gqa_paged(q, K, V, table, torch.tensor([640], dtype=torch.int32, device="cuda"))
    assert bool(out[:, :, 7].isnan().all())
    rest = torch.ones(D, dtype=torch.bool, device="cuda")
    rest[7] = False
    assert torch.equal(out[:, :, rest], torch.ones_like(out[:, :, rest]))
    _clean(fqkv)


# ------------------------------------------------------------------ together
@pytest.mark.parametrize("int8", [False, True])
def test_decode_loop_with_eviction(fqkv, int8):
    """Packed prompts, then steps of append, attention with weights and eviction, everything in place, captured
    once; each step is checked against float64 on the state before it."""
    B, Hq, Hkv, D, page, budget, recent, steps = 3, 8, 2, 64, 16, 48, 8, 40
    prompts = [50, 3, 20]
    g = torch.Generator().manual_seed(11)
    c = Cache(fqkv, [0, 0, 0], Hkv, D, page, int8, room=budget + page, seed=2)
    cos, sin = _tables(256, D)
    axes = fqkv.rope_axes([16, 8, 8], interleaved=True)
    T = sum(prompts)
    seqs = torch.repeat_interleave(torch.arange(B), torch.tensor(prompts)).to(torch.int32).cuda()
    slots = torch.cat([torch.arange(n) for n in prompts]).to(torch.int32).cuda()
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, generator=g).bfloat16().cuda()
    pos = torch.stack([slots, slots // 4, slots % 4]).contiguous()
    q_out = torch.empty(T, Hq, D, dtype=torch.float16, device="cuda")
    fqkv.rope_qkv_append_paged(qkv, cos, sin, pos, slots, c.table, q_out, c.K, c.V, c.Ks, c.Vs, axes=axes, seq_ids=seqs)
    c.lens.copy_(torch.tensor(prompts))
    w = torch.zeros(B, Hkv, c.cap, device="cuda")

    x = torch.empty(B, (Hq + 2 * Hkv) * D, dtype=torch.bfloat16, device="cuda")
    step_pos = torch.tensor([prompts] * 3, dtype=torch.int32).cuda()
    q = torch.empty(B, Hq, D, dtype=torch.float16, device="cuda")
    out = torch.empty(B, Hq, D, dtype=torch.bfloat16, device="cuda")
    one = torch.ones(B, dtype=torch.int32, device="cuda")

    def append_and_attend():
        fqkv.rope_qkv_append_paged(x, cos, sin, step_pos, c.lens, c.table, q, c.K, c.V, c.Ks, c.Vs, axes=axes)
        c.lens.add_(one)
        step_pos.add_(1)
        c.attend(fqkv, q, out=out, weights=w)

    def evict():
        fqkv.evict_kvcache_paged(c.K, c.V, c.table, c.lens, w, budget, recent, c.Ks, c.Vs, lens_out=c.lens)

    state = [t for t in (c.K, c.V, c.Ks, c.Vs, c.lens, w, step_pos) if t is not None]
    saved = [t.clone() for t in state]
    x.copy_(torch.randn(x.shape, generator=g))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        append_and_attend()
        evict()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for fn in (append_and_attend, evict):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            fn()
        graphs.append(graph)
    for t, s in zip(state, saved):
        t.copy_(s)
    lens = list(prompts)
    for i in range(steps):
        x.copy_(torch.randn(x.shape, generator=g))
        before = w.clone()
        graphs[0].replay()
        lens = [n + 1 for n in lens]
        assert c.lens.tolist() == lens
        for b, n in enumerate(lens):
            assert (before[b, :, n - 1] == 0).all()  # a new token's weight starts at zero
        c.check(fqkv, q, out, before, w)
        if i % 4 == 3:
            K0, V0 = c.values()
            w0 = w.cpu().numpy()
            graphs[1].replay()
            K1, V1 = c.values()
            t = c.table.cpu().numpy()
            for b in range(B):
                if lens[b] <= budget:
                    continue
                for h in range(Hkv):
                    keep = op.kept_tokens(w0[b, h, :lens[b]], budget, recent)
                    for a0, a1 in ((K0, K1), (V0, V1)):
                        np.testing.assert_array_equal(op.gather(a1, t[b], budget)[h], op.gather(a0, t[b], lens[b])[h][keep])
                    np.testing.assert_array_equal(w[b, h, :budget].cpu().numpy(), w0[b, h][keep])
                    assert (w[b, h, budget:] == 0).all()
            lens = [min(n, budget) for n in lens]
            assert c.lens.tolist() == lens
    assert max(lens) == budget
    _clean(fqkv)
