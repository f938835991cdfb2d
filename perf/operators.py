"""Measured cases of the paged-cache decode operators.

Three operators work on one paged KV cache: pools of pages ``[P, Hkv, page, D]`` (fp16, or int8 codes
with one fp16 scale per token and KV head), a block table ``[B, max_pages]`` that names each sequence's
pages, and the sequences' lengths.

* ``attn``: attention of one new token per sequence over its pages (grouped query heads), optionally
  adding each cached token's attention weight to a running sum.
* ``append``: rotary embedding of a fused q/k/v projection with one or several position axes, the fp16
  cast of q, and the write of k and v (quantized for an int8 cache) into their pages.
* ``evict``: eviction down to a budget: the newest tokens and those of the largest accumulated weight
  stay, in order, moved to the front of the sequence's pages.

``own`` false: each operator in elementary torch operations.  ``own`` true: the package's operators.
"""
import importlib
import math

import torch

own = False

PACKAGE = "fused-quantized-kv-decode-attention_b200"
ROPE_BASE = 500000.0
TABLE_ROWS = 32768


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One request of the 1B decoder (32 query heads, 8 KV heads, D = 64) at its 640-token context: latency.
        _attn("attn_fp16_b1_640", B=1, Hq=32, Hkv=8, D=64, page=16, max_len=640),
        # A serving batch in full churn: lengths from an empty slot to 8K in 16-token pages, bf16 model.
        _attn("attn_fp16_b16_ragged_8k", B=16, Hq=32, Hkv=8, D=128, page=16, max_len=8192, ragged=True, out="bf16"),
        # The headline decode size (batch 64, 16K tokens, D = 128) in a paged cache: bandwidth.
        _attn("attn_fp16_b64_16k", B=64, Hq=32, Hkv=8, D=128, page=64, max_len=16384),
        # Odd everything: 7 query heads per KV head, 48-token pages, tokens outside heads in memory.
        _attn("attn_int8_b5_odd", kv="int8", B=5, Hq=28, Hkv=4, D=128, page=48, max_len=3001, ragged=True, nhd=True),
        # The headline decode size with an int8 cache.
        _attn("attn_int8_b64_16k", kv="int8", B=64, Hq=32, Hkv=8, D=128, page=32, max_len=16384),
        # Decode that also keeps the eviction statistics of an 8K context.
        _attn("attn_fp16_b8_8k_weights", B=8, Hq=32, Hkv=8, D=128, page=16, max_len=8192, weights=True),
        # One decode step of one request: the smallest append, three position axes.
        _append("append_fp16_b1", B=1, Hq=32, Hkv=8, D=64, page=16, model="bf16", max_len=640, axes=3),
        # One decode step of a batch, the plain one-axis embedding.
        _append("append_fp16_b64", B=64, Hq=32, Hkv=8, D=128, page=16, model="bf16", max_len=1000, axes=1),
        # Prefill of packed prompts with image tokens (height and width positions) into an int8 cache.
        _append("append_int8_prefill_8k", kv="int8", B=3, T=8191, Hq=32, Hkv=8, D=128, page=32, model="bf16", max_len=3000,
                axes=3, interleaved=True),
        # A request that ran 64 tokens past its 2048-token budget.
        _evict("evict_fp16_b1_2k", B=1, Hkv=8, D=64, page=16, max_len=2112, budget=2048, recent=256),
        # Long prompts of a ragged batch brought down to a quarter after their prefill.
        _evict("evict_fp16_b16_16k", B=16, Hkv=8, D=128, page=64, max_len=16384, budget=4096, recent=512, ragged=True),
        # An int8 cache with odd sizes.
        _evict("evict_int8_b6_5k", kv="int8", B=6, Hkv=4, D=128, page=48, max_len=5001, budget=1501, recent=333),
    ]


def _attn(name, B, Hq, Hkv, D, page, max_len, kv="fp16", ragged=False, nhd=False, weights=False, out="fp16"):
    return dict(name=name, op="attn", kv=kv, B=B, Hq=Hq, Hkv=Hkv, D=D, page=page, max_len=max_len, ragged=ragged, nhd=nhd,
                weights=weights, out=out)


def _append(name, B, Hq, Hkv, D, page, model, max_len, axes, T=None, kv="fp16", interleaved=False, nhd=False):
    # T None: one token for each of the B sequences, at the end of what they hold; else T tokens in all
    # (the last ones padding), which fill the B sequences from their start.
    return dict(name=name, op="append", kv=kv, B=B, T=B if T is None else T, decode=T is None, Hq=Hq, Hkv=Hkv, D=D, page=page,
                model=model, max_len=max_len, axes=axes, interleaved=interleaved, nhd=nhd)


def _evict(name, B, Hkv, D, page, max_len, budget, recent, kv="fp16", ragged=False, nhd=False):
    return dict(name=name, op="evict", kv=kv, B=B, Hkv=Hkv, D=D, page=page, max_len=max_len, budget=budget, recent=recent,
                ragged=ragged, nhd=nhd)


def draw(rng):
    log = lambda lo, hi: math.exp(rng.uniform(math.log(lo), math.log(hi)))  # noqa: E731
    op = rng.choice(["attn", "attn", "append", "evict"])
    kv, D, nhd = rng.choice(["fp16", "int8"]), rng.choice([64, 128]), rng.random() < 0.3
    Hkv, page = rng.choice([1, 2, 4, 5, 8]), rng.choice([16, 16, 32, 48, 64, 128, 256])
    B = int(log(1, 65))
    Hq = Hkv * rng.choice([1, 2, 3, 4, 4, 7, 8, 16])
    max_len = int(min(16384, max(1, log(2 ** 14, 2 ** 28) / (B * Hkv * D)))) + rng.randrange(7)
    if op == "attn":
        c = _attn("", B, Hq, Hkv, D, page, max_len, kv, rng.random() < 0.5, nhd, rng.random() < 0.3, rng.choice(["fp16", "bf16"]))
    elif op == "append":
        axes, model = rng.choice([1, 3]), rng.choice(["fp16", "bf16"])
        T = None if rng.random() < 0.5 else min(int(log(B, 8192)) + 1, B * max_len) + rng.randrange(3)
        if T is not None:
            max_len = -(-T // B)
        c = _append("", B, Hq, Hkv, D, page, model, min(max_len, 4096), axes, T, kv, rng.random() < 0.5, nhd)
    else:
        budget = max(1, int(max_len * rng.uniform(0.1, 1.0)))
        c = _evict("", B, Hkv, D, page, max_len, budget, int(budget * rng.uniform(0, 0.5)), kv, rng.random() < 0.5, nhd)
    del c["name"]
    return c


def _lens(c):
    """The sequences' lengths: the case's alone, so that work() is exact; prepare() deals them out by the seed."""
    B, n = c["B"], c["max_len"]
    if c["op"] == "append":
        if c["decode"]:
            return [n - i * (n // 2) // B for i in range(B)]  # tokens held before the append
        left, lens = c["T"] - c["T"] // 64, []  # one token in 64 is padding behind the last sequence
        for i in range(B):
            take = min(left // (B - i) + (left % (B - i) > 0), n)
            lens.append(take)
            left -= take
        return lens
    if c["ragged"] and B > 1:
        return [n * i // (B - 1) for i in range(B)]  # an empty slot among them
    return [n - i * (n // 4) // B for i in range(B)]


def work(case):
    c, lens = case, _lens(case)
    D, Hkv, n = c["D"], c["Hkv"], sum(_lens(case))
    code = 1 if c["kv"] == "int8" else 2
    row = D * code + (2 if c["kv"] == "int8" else 0)  # one token of one KV head in K (or V), with its scale
    pages = sum(-(-x // c["page"]) for x in lens)
    if c["op"] == "attn":
        b = 2 * n * Hkv * row + 2 * 2 * c["B"] * c["Hq"] * D + 4 * (pages + c["B"])
        return {"bytes": b + (8 * n * Hkv if c["weights"] else 0), "flops": 4.0 * c["Hq"] * D * n}
    if c["op"] == "append":
        t = c["B"] if c["decode"] else n
        angles = min(t, TABLE_ROWS) * D * 4  # the cos and sin rows of the tokens' positions
        return {"bytes": t * (c["Hq"] + 2 * Hkv) * D * 2 + t * c["Hq"] * D * 2 + 2 * t * Hkv * row + angles
                + 4 * t * (c["axes"] + 2), "flops": 3.0 * t * (c["Hq"] + Hkv) * D}
    moved = sum(c["budget"] for x in lens if x > c["budget"])
    return {"bytes": 4 * n * Hkv + 2 * 2 * moved * Hkv * row + 4 * n * Hkv + 8 * (pages + c["B"]), "flops": 1.0 * n * Hkv}


# ------------------------------------------------------------------ inputs
def _quantize(x):
    """Per-token symmetric int8: fp16 scale amax / 127, codes round(fp16(x / scale)) half to even, of fp16 x."""
    s = (x.abs().amax(-1).float() / 127).half()
    r = (x.float() / s.float()[..., None]).half().float().round().clamp(-127, 127)
    return torch.nan_to_num(r, nan=0.0).to(torch.int8), s


def _pool(c, pages, g):
    shape = (pages, c["page"], c["Hkv"], c["D"]) if c["nhd"] else (pages, c["Hkv"], c["page"], c["D"])
    if c["kv"] == "fp16":
        x = torch.empty(shape, dtype=torch.float16, device="cuda").normal_(generator=g)
        return (x.transpose(1, 2) if c["nhd"] else x), None
    codes = torch.empty(shape, dtype=torch.int8, device="cuda")
    scales = torch.empty(pages, c["Hkv"], c["page"], dtype=torch.float16, device="cuda")
    view = codes.transpose(1, 2) if c["nhd"] else codes
    step = max(1, (1 << 26) // (c["page"] * c["Hkv"] * c["D"]))
    for i in range(0, pages, step):
        x = torch.empty(view[i:i + step].shape, dtype=torch.float16, device="cuda").normal_(generator=g)
        view[i:i + step], scales[i:i + step] = _quantize(x)
    return view, scales


def prepare(case, seed):
    c = case
    g = torch.Generator("cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed)
    lens = [_lens(c)[i] for i in torch.randperm(c["B"], generator=h).tolist()]
    B, page, D, Hq = c["B"], c["page"], c["D"], c.get("Hq")
    # Each sequence has the pages of its tokens (of one more in a decode append, one at least); the pool's pages
    # are dealt out in no order, and the table's other entries name none.
    held = [max(1, -(-(n + (c["op"] == "append" and c["decode"])) // page)) for n in lens]
    pages = sum(held) + 3
    order = torch.randperm(pages, generator=h, dtype=torch.int64).to(torch.int32)
    table = torch.full((B, max(held) + 1), -1, dtype=torch.int32)
    at = 0
    for b, m in enumerate(held):
        table[b, :m] = order[at:at + m]
        at += m
    s = dict(case=c, table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"))
    s["K"], s["Ks"] = _pool(c, pages, g)
    s["V"], s["Vs"] = _pool(c, pages, g)
    cap = table.shape[1] * page
    new = lambda *shape: torch.empty(shape, device="cuda")  # noqa: E731
    valid = torch.arange(cap, device="cuda") < s["lens"][:, None, None]
    if c["op"] == "attn":
        s["q"] = (2.0 * new(B, Hq, D).normal_(generator=g)).half()  # peaked attention, as trained heads have
        if c["weights"]:
            s["weights"] = new(B, c["Hkv"], cap).exponential_(generator=g) * valid
    elif c["op"] == "append":
        model = torch.float16 if c["model"] == "fp16" else torch.bfloat16
        T = c["T"]
        s["qkv"] = new(T, (Hq + 2 * c["Hkv"]) * D).normal_(generator=g).to(model)
        inv = ROPE_BASE ** (-torch.arange(0, D, 2, dtype=torch.float64, device="cuda") / D)
        angle = torch.arange(TABLE_ROWS, dtype=torch.float64, device="cuda")[:, None] * inv
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        if c["decode"]:
            slots, seqs = s["lens"].clone(), torch.arange(B, dtype=torch.int32, device="cuda")
        else:
            pad = T - sum(lens)
            slots = torch.cat([torch.arange(n) for n in lens] + [torch.full((pad,), -1)]).to(torch.int32).cuda()
            seqs = torch.repeat_interleave(torch.arange(B + 1), torch.tensor(lens + [pad])).clamp(max=B - 1).to(torch.int32).cuda()
        s["slots"], s["seqs"] = slots, seqs
        first = torch.randint(TABLE_ROWS // 2, (B,), generator=h, dtype=torch.int32).cuda()[seqs.long()]
        if c["axes"] == 1:
            s["pos"] = (first + slots.clamp(min=0))[None]
        else:  # an image 37 patches wide: time stands still, height and width run
            p = slots.clamp(min=0)
            s["pos"] = torch.stack([first, first + p // 37, first + p % 37]).to(torch.int32).contiguous()
        s["axis"] = _axis_map(c).cuda()
        s["q"] = torch.zeros(T, Hq, D, dtype=torch.float16, device="cuda")
    else:
        # accumulated weights: heavy-tailed, with many ties
        w = (new(B, c["Hkv"], cap).normal_(generator=g).mul_(1.5).exp_() * 64).floor_() / 64
        s["weights"] = w * valid
        s["weights_out"] = torch.zeros_like(w)
        s["lens_out"] = torch.zeros_like(s["lens"])
    return s


def _sections(c):
    half = c["D"] // 2
    return (half,) if c["axes"] == 1 else (half // 4, half * 3 // 8, half * 3 // 8)


def _axis_map(c):
    """The position axis of each rotary pair: contiguous sections, or axes 1 and 2 interleaved into axis 0's."""
    sec, half = _sections(c), c["D"] // 2
    if len(sec) == 1:
        return torch.zeros(half, dtype=torch.int32)
    if not c["interleaved"]:
        return torch.repeat_interleave(torch.arange(3), torch.tensor(sec)).to(torch.int32)
    i = torch.arange(half)
    a = i % 3
    return torch.where(i < 3 * torch.tensor(sec)[a], a, torch.zeros_like(a)).to(torch.int32)


# ------------------------------------------------------------------ passes
def run(state):
    return {"attn": _run_attn, "append": _run_append, "evict": _run_evict}[state["case"]["op"]](state)


def _ops():
    return importlib.import_module(PACKAGE)


def _values(x, scales):
    """A pool's values: an int8 pool as codes times scales."""
    return x if scales is None else x * scales[..., None]


def _rows(pool, scales, table):
    """A pool's pages in sequence order, [B, Hkv, cap, D] in fp32."""
    t = table.clamp(min=0).long()
    x = pool[t].transpose(1, 2).float()
    x = x.reshape(x.shape[0], x.shape[1], -1, x.shape[-1])
    if scales is not None:
        sc = scales[t].transpose(1, 2).float()
        x = x * sc.reshape(x.shape[0], x.shape[1], -1, 1)
    return x


def _run_attn(s):
    c = s["case"]
    if own:
        m = _ops()
        out = None
        if c["out"] == "bf16":
            out = torch.empty(s["q"].shape, dtype=torch.bfloat16, device="cuda")
        if c["kv"] == "fp16":
            o = m.decode_attn_gqa_paged(s["q"], s["K"], s["V"], s["table"], s["lens"], out=out, weights=s.get("weights"))
        else:
            o = m.decode_attn_gqa_int8_paged(s["q"], s["K"], s["V"], s["Ks"], s["Vs"], s["table"], s["lens"], out=out,
                                             weights=s.get("weights"))
        return {"out": o, "weights": s["weights"]} if c["weights"] else {"out": o}
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    q = s["q"].float().view(B, Hkv, Hq // Hkv, D)
    z = torch.matmul(q, _rows(s["K"], s["Ks"], s["table"]).transpose(2, 3)) * (1.0 / math.sqrt(D))  # [B, Hkv, G, cap]
    live = torch.arange(z.shape[-1], device="cuda") < s["lens"][:, None, None, None]
    z = z.masked_fill(~live, -math.inf)
    e = torch.where(live, torch.exp(z - z.amax(-1, keepdim=True)), 0.0)
    p = e / e.sum(-1, keepdim=True).clamp(min=1e-30)  # an empty sequence has no weights
    o = torch.matmul(p, _rows(s["V"], s["Vs"], s["table"])).reshape(B, Hq, D)
    o = o.to(torch.float16 if c["out"] == "fp16" else torch.bfloat16)
    if not c["weights"]:
        return {"out": o}
    s["weights"] += p.sum(2)
    return {"out": o, "weights": s["weights"]}


def _run_append(s):
    c = s["case"]
    if own:
        m = _ops()
        axes = None if c["axes"] == 1 else s["axis"]
        m.rope_qkv_append_paged(s["qkv"], s["cos"], s["sin"], s["pos"], s["slots"], s["table"], s["q"], s["K"], s["V"],
                                s["Ks"], s["Vs"], axes=axes, seq_ids=None if c["decode"] else s["seqs"])
    else:
        T, Hq, Hkv, D = c["T"], c["Hq"], c["Hkv"], c["D"]
        x = s["qkv"].float().view(T, Hq + 2 * Hkv, D)
        at = s["pos"].long()[s["axis"].long()].t()  # [T, D/2]: each pair's position
        pair = torch.arange(D // 2, device="cuda")
        cos, sin = s["cos"][at, pair][:, None], s["sin"][at, pair][:, None]
        lo, hi = x[:, :Hq + Hkv, :D // 2], x[:, :Hq + Hkv, D // 2:]
        qk = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1).half()
        live = s["slots"] >= 0
        s["q"][live] = qk[live, :Hq]
        slot = s["slots"][live].long()
        pg, off = s["table"][s["seqs"][live].long(), slot // c["page"]].long(), slot % c["page"]
        k, v = qk[live, Hq:], x[live, Hq + Hkv:].half()
        if c["kv"] == "int8":
            k, ks = _quantize(k)
            v, vs = _quantize(v)
            s["Ks"][pg, :, off], s["Vs"][pg, :, off] = ks, vs
        s["K"][pg, :, off], s["V"][pg, :, off] = k, v
    return {"q": s["q"], "K": _values(s["K"], s["Ks"]), "V": _values(s["V"], s["Vs"])}


def _run_evict(s):
    c = s["case"]
    if own:
        m = _ops()
        m.evict_kvcache_paged(s["K"], s["V"], s["table"], s["lens"], s["weights"], c["budget"], c["recent"], s["Ks"], s["Vs"],
                              weights_out=s["weights_out"], lens_out=s["lens_out"])
    else:
        w, n = s["weights"], s["lens"][:, None, None]
        cap, budget = w.shape[-1], min(c["budget"], w.shape[-1])
        j = torch.arange(cap, device="cuda").expand_as(w)
        key = torch.where(j >= n - c["recent"], math.inf, w).masked_fill(j >= n, -math.inf)
        best = key.sort(dim=-1, descending=True, stable=True)[1][..., :budget]  # ties: the lowest index first
        src = best.sort(dim=-1)[0]
        dst = j[..., :budget]
        src = torch.where(n > budget, src, torch.where(dst < n, dst, 0))  # short sequences stay as they are
        dst = torch.where(n > budget, dst, src)
        t = s["table"].clamp(min=0).long()
        head = torch.arange(c["Hkv"], device="cuda")[None, :, None].expand_as(src)
        row = torch.arange(c["B"], device="cuda")[:, None, None].expand_as(src)
        here = (t[row, src // c["page"]], head, src % c["page"])
        there = (t[row, dst // c["page"]], head, dst % c["page"])
        pools = (s["K"], s["V"]) if c["kv"] == "fp16" else (s["K"], s["V"], s["Ks"], s["Vs"])
        moved = [p[here] for p in pools]
        [p.index_put_(there, m) for p, m in zip(pools, moved)]
        kept = torch.zeros_like(w)
        kept[..., :budget] = w.gather(-1, src)
        kept = kept * (j < n.clamp(max=budget))
        s["weights_out"].copy_(torch.where(j < n, kept, s["weights_out"]))
        s["lens_out"].copy_(s["lens"].clamp(max=budget))
    return {"K": _values(s["K"], s["Ks"]), "V": _values(s["V"], s["Vs"]), "weights": s["weights_out"], "lens": s["lens_out"]}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"attn": _exact_attn, "append": _exact_append, "evict": _exact_evict}[case["op"]](case, s)


def _exact_rows(c, pool, scales, ids, n):
    """Tokens [0, n) of the sequence with pages `ids`: [Hkv, n, D] in 64 bits."""
    pages = [pool[int(i)].double() if scales is None else pool[int(i)].double() * scales[int(i)].double()[..., None] for i in ids]
    return torch.cat(pages, 1)[:, :n]


def _exact_attn(c, s):
    B, Hq, Hkv, D = c["B"], c["Hq"], c["Hkv"], c["D"]
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device="cuda")
    acc = s["weights"].double() if c["weights"] else None
    for b, n in enumerate(s["lens"].tolist()):
        if n == 0:
            continue
        ids = s["table"][b, :-(-n // c["page"])].tolist()
        K, V = _exact_rows(c, s["K"], s["Ks"], ids, n), _exact_rows(c, s["V"], s["Vs"], ids, n)
        for h in range(Hkv):
            heads = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            z = s["q"][b, heads].double() @ K[h].T / math.sqrt(D)
            p = torch.exp(z - torch.logsumexp(z, -1, keepdim=True))
            out[b, heads] = p @ V[h]
            if acc is not None:
                acc[b, h, :n] += p.sum(0)
    return {"out": out} if acc is None else {"out": out, "weights": acc}


def _exact_append(c, s):
    T, Hq, Hkv, D = c["T"], c["Hq"], c["Hkv"], c["D"]
    half, page = D // 2, c["page"]
    x = s["qkv"].double().view(T, -1, D)
    q = s["q"].double()
    K, V = s["K"].double(), s["V"].double()
    axis, pos = s["axis"].tolist(), s["pos"].long()
    cos = torch.stack([s["cos"].double()[pos[a], i] for i, a in enumerate(axis)], 1)
    sin = torch.stack([s["sin"].double()[pos[a], i] for i, a in enumerate(axis)], 1)
    z = torch.complex(x[..., :half], x[..., half:]) * torch.complex(cos, sin)[:, None]
    y = torch.cat([z.real, z.imag], -1)
    slots, seqs, table = s["slots"].cpu(), s["seqs"].cpu(), s["table"].cpu()
    tokens = torch.nonzero(slots >= 0)[:, 0]
    slot = slots[tokens].long()
    pg, off = table[seqs[tokens].long(), torch.div(slot, page, rounding_mode="floor")].long().cuda(), (slot % page).cuda()
    tokens = tokens.cuda()
    q[tokens] = y[tokens, :Hq]
    if c["kv"] == "int8":  # codes next to a rounding border have no value of their own
        return {"q": q, "K": None, "V": None}
    K[pg, :, off], V[pg, :, off] = y[tokens, Hq:Hq + Hkv], x[tokens, Hq + Hkv:]
    return {"q": q, "K": K, "V": V}


def _exact_evict(c, s):
    page, budget, recent = c["page"], c["budget"], c["recent"]
    pools = [p for p in (s["K"], s["V"], s["Ks"], s["Vs"]) if p is not None]
    w_all, lens = s["weights"].double().cpu().numpy(), s["lens"].tolist()
    out_w, out_n = s["weights_out"].double().cpu().numpy(), []
    for b, n in enumerate(lens):
        out_n.append(min(n, budget))
        ids = s["table"][b].long()
        for h in range(c["Hkv"]):
            if n <= budget:
                out_w[b, h, :n] = w_all[b, h, :n]
                continue
            old = w_all[b, h, :n - recent]
            heavy = sorted(range(n - recent), key=lambda j: (-old[j], j))[:budget - recent]
            keep = torch.tensor(sorted(heavy) + list(range(n - recent, n)), device="cuda")
            to = torch.arange(budget, device="cuda")
            for p in pools:
                p[ids[to // page], h, to % page] = p[ids[keep // page], h, keep % page]
            out_w[b, h, :n] = 0
            out_w[b, h, :budget] = w_all[b, h, keep.cpu().numpy()]
    value = lambda p, sc: p.double() if sc is None else p.double() * sc.double()[..., None]  # noqa: E731
    return {"K": value(s["K"], s["Ks"]), "V": value(s["V"], s["Vs"]), "weights": torch.from_numpy(out_w),
            "lens": torch.tensor(out_n, dtype=torch.int32)}
