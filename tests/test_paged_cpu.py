"""Paged-cache operators, the host side without a GPU: refusals of the C entries before any CUDA call, the
descriptor's layout, the rotary axis map, and the float64 definitions on cases worked out by hand."""
from __future__ import annotations

import ctypes
import re

import numpy as np
import pytest
import torch

from conftest import ROOT
from oracle import paged as op

A16, A2 = 16, 18  # a 16-byte aligned dummy address (never followed), and one that is not


def _kv(fqkv, **kw):
    f = dict(fmt=0, page=16, P=10, max_pages=4, B=2, Hkv=2, D=64, k=A16, v=A16, ks=0, vs=0, k_strides=None, v_strides=None,
             ks_strides=(32, 16), vs_strides=(32, 16), table=A16, table_stride=4, lens=A16)
    f.update(kw)
    st = (f["Hkv"] * f["page"] * f["D"], f["page"] * f["D"], f["D"])
    ks, vs = f["k_strides"] or st, f["v_strides"] or st
    return fqkv.native.PAGED_KV.pack(f["fmt"], 0, f["page"], f["P"], f["max_pages"], f["B"], f["Hkv"], f["D"], f["k"], f["v"],
                                     f["ks"], f["vs"], *ks, *vs, *f["ks_strides"], *f["vs_strides"], f["table"],
                                     f["table_stride"], f["lens"])


def _attn(fqkv, desc, out_dtype=0, q=A16, o=A16, Hq=4, weights=None, ws=None, nb=0):
    rc = fqkv.native.lib().fqkv_decode_attn_paged(desc, out_dtype, q, o, Hq, weights, ws, nb, None)
    return rc, fqkv.native.last_error()


def test_descriptor_matches_the_header(fqkv):
    """Field by field: fqkv_paged_kv_t has no padding and the packed order is the header's."""
    text = (ROOT / "include" / "fqkv_b200.h").read_text()
    body = re.search(r"typedef struct fqkv_paged_kv \{(.*?)\} fqkv_paged_kv_t;", text, re.S).group(1)
    body = re.sub(r"/\*.*?\*/", "", body, flags=re.S)
    order = []
    for decl in body.split(";"):
        decl = " ".join(decl.split())
        if not decl:
            continue
        kind = "i" if decl.startswith("int32_t ") and "*" not in decl else "q" if decl.startswith("int64_t ") else "Q"
        for name in re.sub(r"^(const )?\w+ ?\*? ?", "", decl).split(","):
            n = re.search(r"\[(\d+)\]", name)
            order += [kind] * (int(n.group(1)) if n else 1)
    fmt = fqkv.native.PAGED_KV.format.lstrip("=")
    packed = [k for n, k in re.findall(r"(\d*)([iqQ])", fmt) for _ in range(int(n or 1))]
    assert packed == order


BAD, MIS = 1, 2


@pytest.mark.parametrize("kw,code,word", [
    (dict(fmt=2), BAD, "kv_format"), (dict(D=96), BAD, "D"), (dict(page=0), BAD, "page_size"), (dict(page=24), BAD, "page_size"),
    (dict(page=-16), BAD, "page_size"), (dict(P=0), BAD, "zero size"), (dict(Hkv=0), BAD, "zero size"),
    (dict(max_pages=0), BAD, "zero size"), (dict(B=-1), BAD, "zero size"), (dict(B=40000), BAD, "index range"),
    (dict(max_pages=2 ** 28), BAD, "index range"), (dict(P=2 ** 31), BAD, "index range"),
    (dict(k=0), BAD, "null"), (dict(table=0), BAD, "null"), (dict(lens=0), BAD, "null"), (dict(fmt=1), BAD, "null"),
    (dict(v=A2), MIS, "aligned"), (dict(fmt=1, ks=A2, vs=A16), MIS, "aligned"), (dict(lens=A2), MIS, "aligned"),
    (dict(table_stride=3), BAD, "block_table"), (dict(k_strides=(2048, 1024, 0)), BAD, "strides"),
    (dict(k_strides=(2048, 1024, 68)), MIS, "strides"), (dict(v_strides=(2048, 1020, 64)), MIS, "strides"),
    (dict(v_strides=(2 ** 40, 1024, 64)), BAD, "strides"), (dict(fmt=1, ks=A16, vs=A16, ks_strides=(32, 8)), BAD, "scale strides"),
    (dict(fmt=1, ks=A16, vs=A16, vs_strides=(36, 16)), MIS, "scale strides"),
])
def test_bad_descriptors_rejected_by_every_entry(fqkv, kw, code, word):
    desc = _kv(fqkv, **kw)
    rc, msg = _attn(fqkv, desc)
    assert rc == code and word in msg, msg
    lib = fqkv.native.lib()
    rc = lib.fqkv_evict_paged(desc, A16, A16, A16, 8, 2, A16, 1 << 30, None)
    assert rc == code and word in fqkv.native.last_error()
    if "lens" not in kw:
        rc = lib.fqkv_rope_append_paged(desc, 0, A16, 8 * 64, A16, A16, 10, A16, 2, 1, None, None, A16, A16, 2, 4, None)
        assert rc == code and word in fqkv.native.last_error()


def test_attention_arguments_rejected(fqkv):
    ok = _kv(fqkv)
    lib = fqkv.native.lib()
    assert lib.fqkv_decode_attn_paged(None, 0, A16, A16, 4, None, None, 0, None) == BAD
    for kw, code, word in ((dict(out_dtype=2), BAD, "out_dtype"), (dict(Hq=5), BAD, "multiple"), (dict(Hq=0), BAD, "multiple"),
                           (dict(q=None), BAD, "null"), (dict(o=None), BAD, "null"), (dict(q=A2), MIS, "aligned"),
                           (dict(weights=A2), MIS, "aligned")):
        rc, msg = _attn(fqkv, ok, **kw)
        assert rc == code and word in msg
    rc, _ = _attn(fqkv, _kv(fqkv, B=0, table=0, lens=0))
    assert rc == 0  # no sequences: nothing to do
    assert lib.fqkv_paged_workspace_bytes(2, 1, 1, 1, 64, 100, 0) == 0
    assert lib.fqkv_paged_workspace_bytes(0, 1, 3, 2, 64, 100, 0) == 0


def test_append_arguments_rejected(fqkv):
    ok = _kv(fqkv)
    lib = fqkv.native.lib()

    def call(model=0, qkv=A16, stride=8 * 64, cos=A16, rows=10, pos=A16, pos_stride=2, axes=1, amap=None, seqs=None, slots=A16,
             q=A16, T=2, Hq=4, desc=ok):
        rc = lib.fqkv_rope_append_paged(desc, model, qkv, stride, cos, A16, rows, pos, pos_stride, axes, amap, seqs, slots, q,
                                        T, Hq, None)
        return rc, fqkv.native.last_error()

    for kw, code, word in ((dict(model=2), BAD, "model_dtype"), (dict(stride=8 * 64 - 8), BAD, "qkv_row_stride"),
                           (dict(stride=8 * 64 + 4), MIS, "aligned"), (dict(qkv=A2), MIS, "aligned"), (dict(cos=A2), MIS, "aligned"),
                           (dict(q=A2), MIS, "aligned"), (dict(rows=0), BAD, "sizes"), (dict(T=-1), BAD, "sizes"),
                           (dict(axes=0), BAD, "axes"), (dict(axes=9), BAD, "axes"), (dict(axes=3), BAD, "null"),
                           (dict(axes=3, amap=A16, pos_stride=1), BAD, "positions"), (dict(T=3), BAD, "seq_ids"),
                           (dict(Hq=3), BAD, "multiple"), (dict(pos=None), BAD, "null"), (dict(slots=None), BAD, "null"),
                           (dict(slots=A2), MIS, "aligned"), (dict(desc=_kv(fqkv, B=0)), BAD, "no sequences")):
        rc, msg = call(**kw)
        assert rc == code and word in msg, (kw, rc, msg)
    assert call(T=0, qkv=None, q=None)[0] == 0


def test_evict_arguments_rejected(fqkv):
    ok = _kv(fqkv)
    lib = fqkv.native.lib()
    need = lib.fqkv_evict_workspace_bytes(2, 2, 64, 8)
    assert need >= 4 * (8 + 8 * 4) and lib.fqkv_evict_workspace_bytes(2, 2, 64, 1000) < 4 * (8 + 64 * 4) + 512 + 1
    assert lib.fqkv_evict_workspace_bytes(0, 2, 64, 8) == 0 and lib.fqkv_evict_workspace_bytes(2, 2, 64, 0) == 0
    far = A16 + 4 * 2 * 2 * 64

    def call(w=A16, wo=far, lens=A16, budget=8, recent=2, ws=A16, nb=need):
        rc = lib.fqkv_evict_paged(ok, w, wo, lens, budget, recent, ws, nb, None)
        return rc, fqkv.native.last_error()

    for kw, code, word in ((dict(budget=0), BAD, "budget"), (dict(recent=-1), BAD, "recent"), (dict(recent=9), BAD, "recent"),
                           (dict(w=None), BAD, "null"), (dict(lens=None), BAD, "null"), (dict(w=A2), MIS, "aligned"),
                           (dict(wo=far - 16), BAD, "overlap"), (dict(w=far, wo=A16 + 16), BAD, "overlap"),
                           (dict(nb=need - 1), BAD, "workspace"), (dict(ws=None), BAD, "workspace"), (dict(ws=A2), MIS, "workspace")):
        rc, msg = call(**kw)
        assert rc == code and word in msg, (kw, rc, msg)


def test_one_pool_for_keys_and_values_is_not_written(fqkv):
    """Reading it is fine; an append or an eviction would write one over the other."""
    lib = fqkv.native.lib()
    need = lib.fqkv_evict_workspace_bytes(2, 2, 64, 8)
    assert lib.fqkv_evict_paged(_kv(fqkv), A16, A16, A16, 8, 2, A16, need, None) == BAD
    assert "different pools" in fqkv.native.last_error()
    assert lib.fqkv_rope_append_paged(_kv(fqkv), 0, A16, 8 * 64, A16, A16, 10, A16, 2, 1, None, None, A16, A16, 2, 4, None) == BAD
    assert "different pools" in fqkv.native.last_error()


def test_sizes_past_the_index_range_have_no_workspace(fqkv):
    lib = fqkv.native.lib()
    assert lib.fqkv_paged_workspace_bytes(0, 1, 1, 1, 64, 2 ** 30 + 16, 1) == 0
    assert lib.fqkv_evict_workspace_bytes(1, 1, 2 ** 30 + 16, 2 ** 40) == 0
    # 16384 x 4 heads in groups of 16, of 2^30 tokens: the tiles have no 32-bit numbers
    rc, msg = _attn(fqkv, _kv(fqkv, B=16384, Hkv=4, max_pages=2 ** 26, table_stride=2 ** 26), Hq=4 * 17)
    assert rc == BAD and "index range" in msg


def test_python_layer_refuses_cpu_tensors(fqkv):
    K = torch.zeros(2, 1, 16, 64, dtype=torch.float16)
    i = torch.zeros(1, 2, dtype=torch.int32)
    q = torch.zeros(1, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="^cuda"):
        fqkv.decode_attn_gqa_paged(q, K, K, i, i[0])
    with pytest.raises(RuntimeError, match="^cuda"):
        fqkv.evict_kvcache_paged(K, K, i, i[0], torch.zeros(1, 1, 32), 4, 1)
    with pytest.raises(RuntimeError, match="^cuda"):
        fqkv.rope_qkv_append_paged(q[0], q[0].float(), q[0].float(), i[0], i[0], i, q, K, K)


def test_binding_of_another_torch_is_refused(fqkv, monkeypatch):
    assert fqkv.native.binding().built_for_torch == torch.__version__
    monkeypatch.setattr(fqkv.native, "_binding", None)
    monkeypatch.setattr(torch, "__version__", "0.0")
    with pytest.raises(fqkv.native.NativeLibraryError, match="built for torch"):
        fqkv.native.binding()


def test_rope_axes(fqkv):
    assert fqkv.rope_axes([4], device="cpu").tolist() == [0] * 4
    assert fqkv.rope_axes([2, 3, 1], device="cpu").tolist() == [0, 0, 1, 1, 1, 2]
    # pairs 0..8 in turn, then axis 0 takes what is left
    assert fqkv.rope_axes([6, 3, 3], interleaved=True, device="cpu").tolist() == [0, 1, 2, 0, 1, 2, 0, 1, 2, 0, 0, 0]
    for sec in ([32, 16, 16], [16, 24, 24], [24, 20, 20]):
        ids = fqkv.rope_axes(sec, device="cpu")
        assert torch.bincount(ids, minlength=3).tolist() == sec and ids.dtype == torch.int32
    with pytest.raises(ValueError):
        fqkv.rope_axes([])
    with pytest.raises(ValueError):
        fqkv.rope_axes([4, -1])


def test_device_status_words_of_the_paged_operators(fqkv):
    assert "page" in fqkv.ops.DEVICE_STATUS[65] and "token" in fqkv.ops.DEVICE_STATUS[66]


# ------------------------------------------------------------------ the definitions
def test_definition_kept_tokens():
    w = np.array([1.0, np.nan, 3.0, np.inf, 3.0, -0.0, 0.0, 9.0])
    assert op.kept_tokens(w, 4, 1).tolist() == [1, 2, 3, 7]      # NaN, inf, the first of the two threes; the newest
    assert op.kept_tokens(w, 3, 0).tolist() == [1, 3, 7]
    assert op.kept_tokens(np.zeros(6), 3, 1).tolist() == [0, 1, 5]
    assert op.kept_tokens(np.arange(6.0), 2, 2).tolist() == [4, 5]


def test_definition_attention_and_rope():
    K = np.zeros((3, 1, 16, 2))
    V = np.arange(3 * 16 * 2, dtype=np.float64).reshape(3, 1, 16, 2)
    r = op.paged_attention(np.ones((2, 2, 2)), K, V, np.array([[2, 0], [1, 9]]), [17, 0])
    # zero keys: the mean of page 2's rows and row 0 of page 0
    np.testing.assert_allclose(r["out"][0, 0], (V[2, 0].sum(0) + V[0, 0, 0]) / 17)
    assert (r["out"][1] == 0).all()
    y, _ = op.rope(np.array([[[1.0, 2.0, 3.0, 4.0]]]), np.array([[1.0, 1.0], [0.0, 0.0]]), np.array([[0.0, 0.0], [1.0, 1.0]]),
                   np.array([[0], [1]]), np.array([0, 1]))
    # pair (1, 3) is not turned; pair (2, 4) by a quarter: (2, 4) -> (-4, 2)
    np.testing.assert_allclose(y[0, 0], [1.0, -4.0, 3.0, 2.0])


def test_packed_descriptor_is_accepted_as_a_pointer(fqkv):
    """bytes go to the C entry as they are."""
    assert fqkv.native.SIGNATURES["fqkv_decode_attn_paged"][1][0] is ctypes.c_void_p
    assert len(_kv(fqkv)) == fqkv.native.PAGED_KV.size == 192
