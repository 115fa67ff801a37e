"""The operators of a decoding step on the quantized layers, as cases that can be prepared, run and compared.

A text model on the library's 4-bit layers produces one token (or a few) at a time: its projections are products of a stored
weight with a handful of rows, its keys and values live in a paged cache of 8-bit values, and every step appends to that cache
and attends over all of it. Kinds of case:

  matvec     ``linear_matvec``: y = act(W x + b) for few rows, W as stored (NVFP4 or NF4), bias, GELU, SwiGLU
  append     ``KvCache.append``: head norm and rotation of q and k, k and v into the pages in e4m3 with a power-of-two scale
             for each (page, head)
  attention  ``KvCache.attention``: softmax(q K^T / sqrt(128)) V over that cache, causal among a sequence's new tokens

``listed()`` holds the fixed cases, ``draw(rng)`` gives one more of the same ranges. ``run(state)`` calls the library where
``own`` is true, and otherwise computes the same in elementary torch operations in 32 bits. ``exact`` is the definition in 64.
"""
from __future__ import annotations

import math

import torch

own = False

HIDDEN, FFN, HEAD_DIM = 5120, 13824, 128
E4M3_TOP = 448.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
EPS = 1e-6


# ---------------------------------------------------------------- the cases

def _matvec(fmt, rows, k, n, act="none", bias=False):
    return {"kind": "matvec", "fmt": fmt, "rows": rows, "k": k, "n": n, "act": act, "bias": bias}


def _append(batch, new, past, heads, kv_heads, page, norm, rotary):
    return {"kind": "append", "batch": batch, "new": new, "past": past, "heads": heads, "kv_heads": kv_heads, "page": page,
            "norm": norm, "rotary": rotary}


def _attention(batch, new, length, heads, kv_heads, page, ragged):
    return {"kind": "attention", "batch": batch, "new": new, "length": length, "heads": heads, "kv_heads": kv_heads, "page": page,
            "ragged": ragged}


def listed():
    return [
        # The smallest layer: one token through the 1024-wide Linear of the benchmark's first configuration. Latency.
        dict(_matvec("nvfp4", 1, 1024, 1024, bias=True), name="matvec_nvfp4_1_1024"),
        # One token through a fused q / k / v projection.
        dict(_matvec("nvfp4", 1, HIDDEN, 3 * HIDDEN), name="matvec_nvfp4_1_qkv"),
        # Eight sequences' tokens through the [gate | up] layer with SwiGLU.
        dict(_matvec("nvfp4", 8, HIDDEN, 2 * FFN, act="swiglu"), name="matvec_nvfp4_8_swiglu"),
        # Three sequences through an NF4 down-projection: long rows, an odd number of them.
        dict(_matvec("nf4", 3, FFN, HIDDEN, bias=True), name="matvec_nf4_3_down"),
        # Sixteen sequences through an NF4 up-projection with GELU.
        dict(_matvec("nf4", 16, HIDDEN, FFN, act="gelu"), name="matvec_nf4_16_up"),
        # A step of one sequence: one token, grouped heads, head norm and a rotation over the whole head.
        dict(_append(1, 1, 999, 40, 8, 64, True, 128), name="append_1x1"),
        # A step of a batch, each sequence at its own place in its page.
        dict(_append(64, 1, 2000, 40, 8, 64, False, 128), name="append_64x1"),
        # A prompt that is stored at once, behind a cached prefix that ends inside a page; 96 rotated channels.
        dict(_append(1, 4747, 77, 40, 10, 64, True, 96), name="append_prompt_4747"),
        # The first tokens of an answer: one sequence, a short cache. Latency.
        dict(_attention(1, 1, 333, 40, 8, 64, False), name="attention_1x333"),
        # A batch being served, each sequence of its own length.
        dict(_attention(32, 1, 4096, 40, 8, 64, True), name="attention_32x4096"),
        # One long document: work has to be split along the sequence.
        dict(_attention(1, 1, 131072, 40, 8, 64, False), name="attention_1x131072"),
        # Several tokens a sequence (drafted tokens being checked), small pages.
        dict(_attention(16, 5, 3001, 40, 10, 16, True), name="attention_16x5_drafts"),
    ]


def _spread(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choices(("matvec", "append", "attention"), (5, 3, 4))[0]
    if kind == "matvec":
        fmt = rng.choice(("nvfp4", "nf4"))
        k, n = 64 * _spread(rng, 4, FFN // 64), 128 * _spread(rng, 2, 2 * FFN // 128)
        if fmt == "nf4":
            n += rng.choice((0, 0, 8, 34))
        act = rng.choice(("none", "none", "gelu", "swiglu"))
        if k * n > 2 * HIDDEN * FFN:
            n = 128 * max(2, 2 * HIDDEN * FFN // k // 128)
        return _matvec(fmt, _spread(rng, 1, 16), k, n, act, rng.random() < 0.4)
    kv_heads = rng.choice((1, 2, 4, 8, 10, 40))
    heads = kv_heads * (rng.choice((1, 2, 4, 5, 8)) if kv_heads < 40 else 1)
    page = rng.choice((16, 32, 64, 64, 128))
    if kind == "append":
        batch = _spread(rng, 1, 64)
        new = 1 if rng.random() < 0.5 else _spread(rng, 2, max(2, 4747 // batch))
        return _append(batch, new, _spread(rng, 1, 4000) - 1, heads, kv_heads, page, rng.random() < 0.5, rng.choice((0, 64, 96, 128)))
    batch = _spread(rng, 1, 64)
    most = 32 * 4096 * 8 // (batch * kv_heads)  # cached tokens of a sequence, by the largest listed case
    length = _spread(rng, 16, max(16, min(131072, most)))
    new = 1 if rng.random() < 0.6 else min(length, _spread(rng, 2, 64))
    if new > 1:  # several queries read the same keys
        batch = max(1, min(batch, 32 * 4096 * 8 * 40 // (length * heads * new)))
        length = max(new, min(length, 32 * 4096 * 8 * 40 // (batch * heads * new)))
    return _attention(batch, new, length, heads, kv_heads, page, rng.random() < 0.5)


# ---------------------------------------------------------------- inputs

def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _pack_high_even(codes):
    return ((codes[:, 0::2] << 4) | codes[:, 1::2]).contiguous()


def _encode_nvfp4(w):
    """Bytes (even element in the high nibble), e4m3 scales of 16 elements in the 128 x 4 tiling, and the fp32 tensor scale."""
    n, k = w.shape
    top = float(w.abs().max()) / (6 * 448)
    blocks = (w / top).view(n, k // 16, 16)
    scale = (blocks.abs().amax(-1) / 6).clamp(max=448).to(torch.float8_e4m3fn)
    s = scale.float().unsqueeze(-1)
    v = torch.where(s > 0, blocks / s, torch.zeros_like(blocks))
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=w.device)
    codes = torch.bucketize(v.abs(), edges, out_int32=True).to(torch.uint8) | ((v < 0).to(torch.uint8) << 3)
    tiled = scale.view(torch.uint8).view(n // 128, 4, 32, k // 64, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)
    return _pack_high_even(codes.view(n, k)), tiled, top


def _encode_nf4(w, block=64, nested=256):
    table = torch.special.ndtri(torch.linspace(0.02, 0.98, 16, device=w.device))
    table = (table / table.abs().max()).float()
    flat = w.reshape(-1, block)
    top = flat.abs().amax(1)
    offset = float(top.mean())
    rest = top - offset
    pad = (-rest.numel()) % nested
    outer = torch.nn.functional.pad(rest, (0, pad)).view(-1, nested).abs().amax(1).clamp(min=1e-12)
    inner = rest / outer.repeat_interleave(nested)[: rest.numel()]
    absmax = torch.round((inner + 1) * 127.5).clamp(0, 255).to(torch.uint8)
    codes = torch.bucketize(flat / top.unsqueeze(1), (table[1:] + table[:-1]) / 2, out_int32=True).to(torch.uint8)
    return {"data": _pack_high_even(codes.view(w.shape)), "absmax": absmax, "map": table,
            "nested_map": torch.linspace(-1, 1, 256, device=w.device).float(), "nested_absmax": outer.float(), "offset": offset}


def _scale_for(amax):
    """The smallest power of two s (2^-100 at least) with amax <= 448 s."""
    m, e = torch.frexp(amax.float() / E4M3_TOP)
    e = torch.where(m > 0.5, e, e - 1).clamp(min=-100)
    e = torch.where(amax > 0, e, torch.full_like(e, -100))
    return torch.ldexp(torch.ones_like(m), e)


def _to_codes(values, scale):
    return (values / scale).clamp(-E4M3_TOP, E4M3_TOP).to(torch.float8_e4m3fn).view(torch.uint8)


def _lengths(g, batch, length, new, ragged):
    """Cached tokens of each sequence, the new ones among them; the first has them all."""
    lens = torch.full((batch,), length, dtype=torch.int32)
    if ragged and batch > 1:
        share = 0.25 + 0.75 * torch.rand(batch - 1, device="cuda", generator=g).cpu()
        lens[1:] = (share * length).to(torch.int32).clamp(min=new)
    return lens


def _cache(g, lens, most, kv_heads, page):
    """A pool with room for `most` tokens of each sequence, whose pages lie in any order, as an allocator leaves them. The slots
    behind a sequence's end hold what an earlier owner left."""
    batch = len(lens)
    per = -(-most // page)
    pages = batch * per + 3
    order = torch.randperm(pages, device="cuda", generator=g)[: batch * per].to(torch.int32)
    k = torch.randn((pages, kv_heads, page, HEAD_DIM), device="cuda", generator=g, dtype=torch.bfloat16)
    k *= torch.exp(0.7 * torch.randn((kv_heads, 1, HEAD_DIM), device="cuda", generator=g)).to(torch.bfloat16)  # loud channels
    v = torch.randn((pages, kv_heads, HEAD_DIM, page), device="cuda", generator=g, dtype=torch.bfloat16)
    ks, vs = (_scale_for(t.abs().amax((2, 3))) for t in (k, v))
    return {"k": _to_codes(k, ks[:, :, None, None].to(torch.bfloat16)), "v": _to_codes(v, vs[:, :, None, None].to(torch.bfloat16)),
            "k_scale": ks, "v_scale": vs, "table": order.view(batch, per).contiguous(), "lens": lens.cuda(), "page": page}


def _ragged_rows(counts):
    """Row starts, and for a padded [batch, most] arrangement of the rows their indices and which of them exist."""
    start = torch.zeros(len(counts) + 1, dtype=torch.int32)
    start[1:] = torch.cumsum(counts, 0)
    most = int(counts.max())
    i = torch.arange(most)
    live = i[None, :] < counts[:, None]
    index = torch.where(live, start[:-1, None] + i[None, :], torch.zeros(1, dtype=torch.int64))
    return start.cuda(), index.cuda(), live.cuda()


def prepare(case, seed):
    g = _generator(seed)
    s = {"kind": case["kind"], "case": case}
    if case["kind"] == "matvec":
        k, n, rows = case["k"], case["n"], case["rows"]
        w = torch.randn((n, k), device="cuda", generator=g).mul_(0.02)
        if case["fmt"] == "nvfp4":
            data, scale, top = _encode_nvfp4(w)
            s["weight"] = {"data": data, "scale": scale, "global": top}
        else:
            s["weight"] = _encode_nf4(w)
        x = torch.randn((rows, k), device="cuda", generator=g, dtype=torch.bfloat16)
        s["x"] = torch.where(torch.rand((rows, k), device="cuda", generator=g) < 1e-3, x * 20, x)
        s["bias"] = 0.01 * torch.randn(n, device="cuda", generator=g) if case["bias"] else None
        s["y"] = torch.empty((rows, n // 2 if case["act"] == "swiglu" else n), dtype=torch.bfloat16, device="cuda")
        return s
    heads, kv_heads, page, batch, new = case["heads"], case["kv_heads"], case["page"], case["batch"], case["new"]
    if case["kind"] == "append":
        counts = torch.full((batch,), new, dtype=torch.int64)
        past = (torch.rand(batch, device="cuda", generator=g).cpu() * (case["past"] + 1)).to(torch.int32) if batch > 1 else torch.tensor([case["past"]], dtype=torch.int32)
        lens = (past + new).to(torch.int32)
    else:
        counts = torch.full((batch,), new, dtype=torch.int64)
        lens = _lengths(g, batch, case["length"], new, case["ragged"])
        if case["ragged"] and new > 1:
            counts[1::2] = torch.clamp(counts[1::2] // 2, min=1)
    most = case["past"] + new if case["kind"] == "append" else case["length"]
    s.update(_cache(g, lens, most, kv_heads, page))
    s["row_start"], s["rows_at"], s["live"] = _ragged_rows(counts)
    s["rows"], s["max_new"], s["max_len"] = int(counts.sum()), int(counts.max()), most
    s["heads"], s["kv_heads"] = heads, kv_heads
    if case["kind"] == "append":
        s["qkv"] = torch.randn((s["rows"], (heads + 2 * kv_heads) * HEAD_DIM), device="cuda", generator=g, dtype=torch.bfloat16)
        s["q_out"] = torch.empty((s["rows"], heads * HEAD_DIM), dtype=torch.bfloat16, device="cuda")
        s["rotary"], s["norm"] = None, None
        if case["rotary"]:
            half = case["rotary"] // 2
            inverse = 1e6 ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
            angle = torch.arange(s["max_len"], device="cuda", dtype=torch.float64)[:, None] * inverse
            s["rotary"] = (torch.cos(angle).float(), torch.sin(angle).float())
        if case["norm"]:
            s["norm"] = (1 + 0.05 * torch.randn((2, HEAD_DIM), device="cuda", generator=g)).to(torch.bfloat16)
    else:
        s["q"] = torch.randn((s["rows"], heads * HEAD_DIM), device="cuda", generator=g, dtype=torch.bfloat16)
        s["out"] = torch.empty((s["rows"], heads * HEAD_DIM), dtype=torch.bfloat16, device="cuda")
    return s


# ---------------------------------------------------------------- the library

def _handles(s):
    """What a program keeps beside its tensors: the weight's descriptor, or the cache and its sequences."""
    import slopfab_b200 as sfq

    if s["kind"] == "matvec":
        w, case = s["weight"], s["case"]
        f = {"out_features": case["n"], "in_features": case["k"], "data": sfq.ptr(w["data"]), "bias_format": sfq.F32}
        if s["bias"] is not None:
            f["bias"] = sfq.ptr(s["bias"])
        if case["fmt"] == "nvfp4":
            f.update(format=sfq.NVFP4, block_scale=sfq.ptr(w["scale"]), global_scale=w["global"])
        else:
            f.update(format=sfq.NF4, nf4_absmax=sfq.ptr(w["absmax"]), nf4_quant_map=sfq.ptr(w["map"]), nf4_nested_quant_map=sfq.ptr(w["nested_map"]),
                     nf4_nested_absmax=sfq.ptr(w["nested_absmax"]), nf4_nested_offset=w["offset"], nf4_block_size=64, nf4_nested_block_size=256)
        act = {"none": sfq.ACT_NONE, "gelu": sfq.ACT_GELU_TANH, "swiglu": sfq.ACT_SWIGLU}[case["act"]]
        return sfq.linear_matvec, sfq.new_weight(**f), act
    from slopfab_b200.kv_cache import KvCache, Rotary, Sequences

    cache = KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    seqs = Sequences(s["table"], s["lens"], s["row_start"], s["max_new"], s["max_len"])
    if s["kind"] == "attention":
        return cache, seqs, None
    cos, sin = s["rotary"] or (None, None)
    q_norm, k_norm = s["norm"] if s["norm"] is not None else (None, None)
    return cache, seqs, Rotary(cos, sin, q_norm=q_norm, k_norm=k_norm, eps=EPS)


def _own(s):
    if "handles" not in s:
        s["handles"] = _handles(s)
    if s["kind"] == "matvec":
        matvec, w, act = s["handles"]
        return matvec(w, s["x"], s["y"], activation=act)
    cache, seqs, rotary = s["handles"]
    if s["kind"] == "attention":
        return cache.attention(seqs, s["q"], s["heads"], out=s["out"])
    cache.append(seqs, s["qkv"], s["heads"], q_out=s["q_out"], rotary=rotary)
    return _appended(s)


def _appended(s):
    """q, and the pool: e4m3 values and their scales."""
    return {"q": s["q_out"], "k": s["k"].view(torch.float8_e4m3fn), "v": s["v"].view(torch.float8_e4m3fn), "k_scale": s["k_scale"],
            "v_scale": s["v_scale"]}


# ---------------------------------------------------------------- the plain form

def _stored_weight(s, dtype):
    """The weight that the stored bytes stand for, [n, k]."""
    w, n, k = s["weight"], s["case"]["n"], s["case"]["k"]
    codes = torch.stack((w["data"] >> 4, w["data"] & 15), dim=-1).view(n, k).long()
    if s["case"]["fmt"] == "nvfp4":
        scale = w["scale"].view(n // 128, k // 64, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(n, k // 16)
        scale = scale.contiguous().view(torch.float8_e4m3fn).to(dtype)
        values = torch.tensor(E2M1, dtype=dtype, device="cuda")[codes]
        return (values.view(n, k // 16, 16) * scale.unsqueeze(-1)).view(n, k) * w["global"]
    absmax = w["nested_map"].to(dtype)[w["absmax"].long()]
    absmax = absmax * w["nested_absmax"].to(dtype).repeat_interleave(256)[: absmax.numel()] + w["offset"]
    return (w["map"].to(dtype)[codes].view(-1, 64) * absmax.unsqueeze(1)).view(n, k)


def _activated(z, act):
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z * z * z)))
    if act == "swiglu":
        gate, up = z.chunk(2, dim=1)
        return gate / (1 + torch.exp(-gate)) * up
    return z


def _normed_and_rotated(s, x, norm, at, dtype):
    """x [..., tokens, heads, 128]: RMSNorm over the head, then the rotation by the angles at positions `at` [..., tokens]."""
    x = x.to(dtype)
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * norm.to(dtype)
    if s["rotary"] is not None:
        half = s["rotary"][0].shape[1]
        cos, sin = (t.to(dtype)[at].unsqueeze(-2) for t in s["rotary"])
        a, b = x[..., :half], x[..., half: 2 * half]
        x = torch.cat((a * cos - b * sin, b * cos + a * sin, x[..., 2 * half:]), dim=-1)
    return x


def _plain_append(s):
    heads, kv_heads, page = s["heads"], s["kv_heads"], s["page"]
    counts = s["row_start"][1:] - s["row_start"][:-1]
    first = (s["lens"] - counts).long()  # position of a sequence's first new token
    position = torch.arange(s["rows"], device="cuda") - torch.repeat_interleave(s["row_start"][:-1].long() - first, counts.long(), output_size=s["rows"])
    owner = torch.repeat_interleave(torch.arange(len(counts), device="cuda"), counts.long(), output_size=s["rows"])
    rows = s["qkv"].view(s["rows"], heads + 2 * kv_heads, HEAD_DIM)
    q_norm, k_norm = s["norm"] if s["norm"] is not None else (None, None)
    s["q_out"].copy_(_normed_and_rotated(s, rows[:, :heads], q_norm, position, torch.float32).view(s["rows"], -1))
    k = _normed_and_rotated(s, rows[:, heads: heads + kv_heads], k_norm, position, torch.float32)
    v = rows[:, heads + kv_heads:].float()
    at = s["table"].long()[owner, position // page]  # page of each new token
    slot = position % page
    fresh = torch.zeros(s["k"].shape[0], dtype=torch.bool, device="cuda").index_fill_(0, at[slot == 0], True)
    touched = torch.unique(at)
    kept = torch.arange(page, device="cuda")
    for_page = torch.full((s["k"].shape[0],), page, device="cuda").scatter_reduce(0, at, slot, "amin")  # tokens that were there
    old = (kept[None, :] < for_page[touched][:, None])[:, None, :]
    for name, values in (("k", k), ("v", v)):
        scale = s[name + "_scale"]
        amax = torch.zeros_like(scale).index_reduce_(0, at, values.abs().amax(-1), "amax")[touched]
        new = torch.maximum(_scale_for(amax), torch.where(fresh[touched][:, None], torch.zeros_like(amax), scale[touched]))
        codes = s[name][touched]
        again = _to_codes(codes.view(torch.float8_e4m3fn).float() * (scale[touched] / new)[:, :, None, None], 1.0)
        mask = old.unsqueeze(-1) if name == "k" else old.unsqueeze(-2)
        s[name][touched] = torch.where(mask, again, codes)
        scale[touched] = new
        mine = _to_codes(values, scale[at].unsqueeze(-1))
        if name == "k":
            s["k"][at, :, slot] = mine
        else:
            s["v"][at, :, :, slot] = mine
    return _appended(s)


def _gathered(s, name, dtype):
    """K or V of each sequence, [batch, kv_heads, tokens, 128], from its pages."""
    t = s["table"].long()
    batch, per = t.shape
    x = s[name][t].view(torch.float8_e4m3fn).to(dtype) * s[name + "_scale"][t].to(dtype)[..., None, None]
    x = x if name == "k" else x.transpose(-1, -2)
    return x.permute(0, 2, 1, 3, 4).reshape(batch, x.shape[2], per * s["page"], HEAD_DIM)


def _plain_attention(s):
    heads, kv_heads = s["heads"], s["kv_heads"]
    batch, most = s["rows_at"].shape
    k, v = _gathered(s, "k", torch.float32), _gathered(s, "v", torch.float32)
    q = s["q"].float()[s["rows_at"].view(-1)].view(batch, most, kv_heads, heads // kv_heads, HEAD_DIM).permute(0, 2, 1, 3, 4)
    counts = (s["row_start"][1:] - s["row_start"][:-1])[:, None]
    sees = s["lens"][:, None] - counts + torch.arange(most, device="cuda")[None, :] + 1  # keys that a query sees
    keys = torch.arange(k.shape[2], device="cuda")
    v = torch.where((keys[None, :] < s["lens"][:, None])[:, None, :, None], v, torch.zeros_like(v))
    scores = (q.reshape(batch, kv_heads, -1, HEAD_DIM) @ k.transpose(-1, -2)).view(batch, kv_heads, most, -1, k.shape[2]) / math.sqrt(HEAD_DIM)
    hidden = (keys[None, None, :] >= sees[:, :, None])[:, None, :, None, :]
    scores = scores.masked_fill(hidden, float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p.view(batch, kv_heads, -1, k.shape[2]) @ v).view(batch, kv_heads, most, -1, HEAD_DIM)
    o = o.permute(0, 2, 1, 3, 4).reshape(batch, most, heads * HEAD_DIM)
    s["out"][s["rows_at"][s["live"]]] = o[s["live"]].to(torch.bfloat16)
    return s["out"]


def run(s):
    if own:
        return _own(s)
    if s["kind"] == "matvec":
        z = s["x"].float() @ _stored_weight(s, torch.float32).t()
        if s["bias"] is not None:
            z = z + s["bias"]
        s["y"].copy_(_activated(z, s["case"]["act"]))
        return s["y"]
    return _plain_append(s) if s["kind"] == "append" else _plain_attention(s)


# ---------------------------------------------------------------- the definition in 64 bits

def _nearest_e4m3(x):
    """The e4m3 value nearest to x (even on a tie), 448 at most: x = m 2^e in steps of 2^(e - 3), of 2^-9 below 2^-6."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(x), e - 4)
    return (torch.round(x / step) * step).clamp(-E4M3_TOP, E4M3_TOP)


def _exact_append(s):
    heads, kv_heads, page = s["heads"], s["kv_heads"], s["page"]
    starts, lens, table = s["row_start"].tolist(), s["lens"].tolist(), s["table"].tolist()
    pool = {n: s[n].view(torch.float8_e4m3fn).double() for n in ("k", "v")}
    scale = {n: s[n + "_scale"].double() for n in ("k", "v")}
    rows = s["qkv"].double().view(s["rows"], heads + 2 * kv_heads, HEAD_DIM)
    norms = s["norm"].double() if s["norm"] is not None else None
    q_all = torch.empty((s["rows"], heads * HEAD_DIM), dtype=torch.float64, device="cuda")

    def turned(x, weight, positions):
        if weight is not None:
            x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + EPS) * weight
        if s["rotary"] is None:
            return x
        cos, sin = (t.double()[positions][:, None, :] for t in s["rotary"])
        half = cos.shape[-1]
        out = x.clone()
        out[..., :half] = x[..., :half] * cos - x[..., half: 2 * half] * sin
        out[..., half: 2 * half] = x[..., :half] * sin + x[..., half: 2 * half] * cos
        return out

    for b, length in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        p0 = length - (r1 - r0)
        positions = torch.arange(p0, length, device="cuda")
        q_all[r0:r1] = turned(rows[r0:r1, :heads], norms[0] if norms is not None else None, positions).reshape(r1 - r0, -1)
        fresh = {"k": turned(rows[r0:r1, heads: heads + kv_heads], norms[1] if norms is not None else None, positions),
                 "v": rows[r0:r1, heads + kv_heads:]}
        at = p0
        while at < length:  # page by page
            end = min(length, (at // page + 1) * page)
            i, o, e = table[b][at // page], at % page, at % page + end - at
            for n in ("k", "v"):
                x = fresh[n][at - p0: end - p0].transpose(0, 1)  # [kv_heads, tokens, 128]
                amax = x.abs().amax((1, 2))
                wanted = 2.0 ** torch.ceil(torch.log2(amax / E4M3_TOP).clamp(min=-100))
                new = torch.maximum(wanted, scale[n][i]) if o else wanted
                page_values = pool[n][i] if n == "k" else pool[n][i].transpose(1, 2)
                if o:
                    page_values[:, :o] = _nearest_e4m3(page_values[:, :o] * (scale[n][i] / new)[:, None, None])
                page_values[:, o:e] = _nearest_e4m3(x / new[:, None, None])
                scale[n][i] = new
            at = end
    return {"q": q_all, "k": pool["k"], "v": pool["v"], "k_scale": scale["k"], "v_scale": scale["v"]}


def _exact_attention(s):
    heads, kv_heads, page = s["heads"], s["kv_heads"], s["page"]
    group = heads // kv_heads
    starts, lens = s["row_start"].tolist(), s["lens"].tolist()
    out = torch.empty((s["rows"], heads, HEAD_DIM), dtype=torch.float64, device="cuda")
    for b, length in enumerate(lens):
        r0, r1 = starts[b], starts[b + 1]
        ids = s["table"][b, : -(-length // page)].long()
        for h in range(kv_heads):
            k = (s["k"][ids, h].view(torch.float8_e4m3fn).double() * s["k_scale"][ids, h].double()[:, None, None]).reshape(-1, HEAD_DIM)[:length]
            v = (s["v"][ids, h].view(torch.float8_e4m3fn).double() * s["v_scale"][ids, h].double()[:, None, None]).transpose(1, 2).reshape(-1, HEAD_DIM)[:length]
            q = s["q"][r0:r1].double().view(r1 - r0, heads, HEAD_DIM)[:, h * group: (h + 1) * group]
            scores = torch.einsum("tgd,sd->tgs", q, k) / HEAD_DIM ** 0.5
            last = torch.arange(length - (r1 - r0), length, device="cuda")
            scores[(torch.arange(length, device="cuda")[None, :] > last[:, None])[:, None, :].expand_as(scores)] = -math.inf
            out[r0:r1, h * group: (h + 1) * group] = torch.softmax(scores, -1) @ v
    return out.view(s["rows"], -1)


def _exact_weight(s):
    """[n, k] in 64 bits, each element from the address of its nibble and of its scale."""
    w, n, k = s["weight"], s["case"]["n"], s["case"]["k"]
    col, row = torch.arange(k, device="cuda")[None, :], torch.arange(n, device="cuda")[:, None]
    nibble = w["data"].long()[:, torch.arange(k, device="cuda") // 2]
    nibble = torch.where(col % 2 == 0, nibble // 16, nibble % 16)
    if s["case"]["fmt"] == "nvfp4":
        block = col // 16
        at = ((row // 128) * (k // 64) + block // 4) * 512 + (row % 32) * 16 + (row % 128) // 32 * 4 + block % 4
        return torch.tensor(E2M1, dtype=torch.float64, device="cuda")[nibble] * w["scale"].view(torch.float8_e4m3fn).double()[at] * w["global"]
    block = (row * k + col) // 64
    absmax = w["nested_map"].double()[w["absmax"].long()[block]] * w["nested_absmax"].double()[block // 256] + w["offset"]
    return w["map"].double()[nibble] * absmax


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        return _exact_append(s)
    if case["kind"] == "attention":
        return _exact_attention(s)
    z = torch.einsum("rk,nk->rn", s["x"].double(), _exact_weight(s))
    if s["bias"] is not None:
        z = z + s["bias"].double()
    if case["act"] == "gelu":
        return z / 2 * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if case["act"] == "swiglu":
        half = z.shape[1] // 2
        return z[:, :half] * torch.sigmoid(z[:, :half]) * z[:, half:]
    return z


# ---------------------------------------------------------------- what a pass cannot do without

def work(case):
    if case["kind"] == "matvec":
        rows, k, n = case["rows"], case["k"], case["n"]
        stored = n * k / 2 + (n * k / 16 if case["fmt"] == "nvfp4" else n * k / 64 + n * k / 64 / 256 * 4)
        out = n // 2 if case["act"] == "swiglu" else n
        return {"bytes": stored + 2 * rows * k + 2 * rows * out + (4 * n if case["bias"] else 0), "flops": 2.0 * rows * n * k}
    heads, kv_heads, batch, new = case["heads"], case["kv_heads"], case["batch"], case["new"]
    if case["kind"] == "append":
        rows = batch * new
        pages = rows // case["page"] + batch
        tables = 4.0 * case["rotary"] * rows if batch == 1 else 4.0 * case["rotary"] * min(rows, case["past"] + new)
        per_row = 2 * (heads + 2 * kv_heads) * HEAD_DIM + 2 * heads * HEAD_DIM + 2 * kv_heads * HEAD_DIM
        return {"bytes": rows * per_row + tables + pages * kv_heads * 8, "flops": 6.0 * rows * (heads + kv_heads) * HEAD_DIM}
    # ragged lengths are a quarter to all of the longest one
    share = 0.625 if case["ragged"] and batch > 1 else 1.0
    tokens = case["length"] * (1 + (batch - 1) * share)
    queries = new * (0.75 if case["ragged"] and new > 1 and batch > 1 else 1.0)
    kv = tokens * kv_heads * 2 * (HEAD_DIM + 4.0 / case["page"] / HEAD_DIM * HEAD_DIM)
    return {"bytes": kv + batch * queries * heads * HEAD_DIM * 4, "flops": 4.0 * HEAD_DIM * heads * tokens * queries}
