"""The paged 8-bit cache: sfq_kv_cache_append and sfq_kv_cache_attention against their definitions in 64 bits.

Bounds. q: fp32 norm and rotation (a sum of 128 squares, a root, a few products: within 2^-16 of the magnitudes that are added),
one rounding to bf16, 2^-8. Codes: the nearest e4m3 of value / scale; k's value is known to 2^-16, so where it lies that near to the
middle between two codes either is right, and a scale may be the next power of two only where the largest magnitude lies that near to
448 s. v and requantised codes come from bf16 and from codes: exact.
Attention: a score is a sum of 128 fp32 products and the scale, off by 130 2^-24 of the sum of the magnitudes (d below); a weight
exp(s - m) is then off by d of itself plus 2^-20, and 2^-11 for its rounding to fp16 in front of the second product; weights and their sum
together twice that, of sum p |v|; sums of T terms in fp32 T 2^-24 at worst; one rounding to bf16, 2^-8."""
import ctypes as C
import math
import os
import subprocess
import sys

import pytest
import torch

import slopfab_b200 as sfq
from slopfab_b200.kv_cache import KvCache, Rotary, Sequences

pytestmark = pytest.mark.gpu
D = 128


def gen(seed):
    return torch.Generator("cuda").manual_seed(seed)


def values_of(codes):
    return codes.view(torch.float8_e4m3fn).double()


def nearest_e4m3(x):
    """The nearest e4m3 value of x (64 bits), ties to even, 448 at most."""
    _, e = torch.frexp(x.abs().clamp(min=2.0 ** -6))
    step = torch.ldexp(torch.ones_like(x), e - 4)
    return (torch.round(x / step) * step).clamp(-448, 448)


def scale_for(amax):
    return 2.0 ** torch.ceil(torch.log2(amax.double() / 448).clamp(min=-100))


class Case:
    """Sequences of given cached lengths (new tokens included) and new tokens, in a pool whose pages lie in any order; every slot that
    holds no token of theirs is filled with bytes of all kinds, NaN among them, and so are the table's entries behind the last page."""

    def __init__(self, counts, lens, kv_heads, group, page, seed=0, fused_pad=0):
        g = gen(seed)
        self.counts, self.lens, self.kv_heads, self.heads, self.page = counts, lens, kv_heads, kv_heads * group, page
        self.max_pages = max(-(-n // page) for n in lens) + 2
        need = [-(-n // page) for n in lens]
        pages = sum(need) + 3
        order = torch.randperm(pages, device="cuda", generator=g).tolist()
        table = torch.full((len(lens), self.max_pages), 1 << 30, dtype=torch.int32)
        table[:, -1] = -7
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = torch.tensor(order[at: at + n], dtype=torch.int32)
            at += n
        rand = lambda *s: torch.randint(0, 256, s, device="cuda", generator=g, dtype=torch.int64).to(torch.uint8)  # noqa: E731
        self.cache = KvCache(rand(pages, kv_heads, page, D), rand(pages, kv_heads, D, page),
                             *(torch.full((pages, kv_heads), float("nan"), device="cuda") for _ in range(2)))
        self.k = torch.zeros((len(lens), kv_heads, max(lens + [1]), D), dtype=torch.float64, device="cuda")  # what the cache stands for
        self.v = torch.zeros_like(self.k)
        self.table = table.cuda()
        self.rows = sum(counts)
        start = [0]
        for n in counts:
            start.append(start[-1] + n)
        self.start = start
        self.seqs = Sequences(self.table, torch.tensor(lens, dtype=torch.int32, device="cuda"), torch.tensor(start, dtype=torch.int32, device="cuda"),
                              max(counts + [1]), max(lens + [1]))
        self.g = g

    def fill(self, tokens, spread=1.0):
        """Stores `tokens[b]` tokens of each sequence directly: random codes and scales of pages."""
        for b, n in enumerate(tokens):
            for p in range(-(-n // self.page)):
                i, m = int(self.table[b, p]), min(self.page, n - p * self.page)
                for name, pool, scale in (("k", self.cache.k, self.cache.k_scale), ("v", self.cache.v, self.cache.v_scale)):
                    s = torch.exp2(torch.randint(-2, 3, (self.kv_heads,), device="cuda", generator=self.g).float() * spread - 7)
                    x = torch.randn((self.kv_heads, m, D), device="cuda", generator=self.g) * 60
                    codes = x.clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
                    scale[i] = s
                    if name == "k":
                        pool[i, :, :m] = codes
                    else:
                        pool[i, :, :, :m] = codes.transpose(1, 2)
                    getattr(self, name)[b, :, p * self.page: p * self.page + m] = values_of(codes) * s.double()[:, None, None]
        return self

    def q(self, sigma=1.0):
        return (sigma * torch.randn((self.rows, self.heads * D), device="cuda", generator=self.g)).to(torch.bfloat16)

    def want_attention(self, q, scale=None):
        """(out, bound) in 64 bits."""
        scale = scale or 1 / math.sqrt(D)
        out = torch.zeros((self.rows, self.heads, D), dtype=torch.float64, device="cuda")
        off = torch.zeros_like(out)
        group = self.heads // self.kv_heads
        for b, n in enumerate(self.counts):
            for i in range(n):
                r, sees = self.start[b] + i, self.lens[b] - n + i + 1
                for h in range(self.kv_heads):
                    k, v = self.k[b, h, :sees], self.v[b, h, :sees]
                    x = q[r].double().view(self.heads, D)[h * group: (h + 1) * group]
                    s = x @ k.T * scale
                    d = 130 * 2.0 ** -24 * (x.abs() @ k.abs().T) * scale
                    p = torch.softmax(s, -1)
                    rel = 2 * (d + 2.0 ** -20 + 2.0 ** -11 + sees * 2.0 ** -24)
                    o = p @ v
                    out[r, h * group: (h + 1) * group] = o
                    off[r, h * group: (h + 1) * group] = (p * rel) @ v.abs() + (p * rel).sum(-1, keepdim=True) * o.abs()
        out, off = out.view(self.rows, -1), off.view(self.rows, -1)
        return out, off + 2.0 ** -8 * (out.abs() + off) + 1e-30

    def check_attention(self, q, scale=0.0, out=None):
        got = self.cache.attention(self.seqs, q, self.heads, out=out, scale=scale)
        want, off = self.want_attention(q, scale)
        assert bool(((got.double() - want).abs() <= off).all()), float(((got.double() - want).abs() - off).max())
        if self.rows:
            assert float((got.double() - want).norm()) <= 2.0 ** -8 * float(want.norm()) + 1e-30
        assert sfq.device_status() == 0
        return got


# ------------------------------------------------------------------------------------------------ attention

@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 5), (3, 8), (1, 13), (8, 2)])
def test_attention_single_tokens(page, kv_heads, group):
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 127, 130, 257, 600]
    c = Case([1] * len(lens), lens, kv_heads, group, page, seed=page + group).fill(lens)
    c.check_attention(c.q())


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("kv_heads,group", [(2, 1), (1, 4), (2, 5), (1, 24)])
def test_attention_several_tokens(page, kv_heads, group):
    """Causal among the new tokens, sequences of no new token, of nothing but new tokens, of nothing at all."""
    counts, lens = [1, 3, 0, 17, 8, 0, 40, 64, 2], [1, 3, 50, 17, 300, 0, 77, 64, 511]
    c = Case(counts, lens, kv_heads, group, page, seed=page + group).fill(lens)
    c.check_attention(c.q())


@pytest.mark.parametrize("length,batch", [(5000, 1), (3333, 3), (20011, 1)])
def test_attention_long(length, batch):
    """Long enough for the sequence to be divided."""
    lens = [length - 1111 * b for b in range(batch)]
    c = Case([1] + [2] * (batch - 1), lens, 2, 5, 64, seed=length).fill(lens)
    c.check_attention(c.q(3.0))


@pytest.mark.parametrize("max_new,max_len", [(1, 1), (1, 10 ** 6), (64, 1), (500, 400)])
def test_estimates_only_size_the_launch(max_new, max_len):
    counts, lens = [9, 1, 30], [700, 100, 30]
    c = Case(counts, lens, 2, 4, 32, seed=5).fill(lens)
    c.seqs.max_new, c.seqs.max_len = max_new, max_len
    c.check_attention(c.q())


def test_attention_scale_pitch_and_rows_behind():
    counts, lens = [1, 4], [90, 200]
    c = Case(counts, lens, 2, 3, 64, seed=6).fill(lens)
    wide = torch.randn((9, 6 * D + 64), device="cuda").to(torch.bfloat16)
    out = torch.full((9, 6 * D + 8), 7.0, dtype=torch.bfloat16, device="cuda")
    c.cache.attention(c.seqs, wide[:, 32: 32 + 6 * D], 6, out=out[:, : 6 * D], scale=0.031)
    want, off = c.want_attention(wide[:5, 32: 32 + 6 * D], 0.031)
    assert bool(((out[:5, : 6 * D].double() - want).abs() <= off).all())
    assert bool((out[5:] == 7).all()) and bool((out[:, 6 * D:] == 7).all())  # rows of no sequence, columns of no head


def test_attention_peaked_and_shifted_scores():
    """One key that takes all the weight, at either end and where a step begins; scores far below and above zero."""
    n = 700
    c = Case([1], [n], 1, 4, 64, seed=7).fill([n])
    for at in (0, 63, 64, 255, 256, n - 1):
        q = c.q(0.1)
        q[0, :D] = (c.k[0, 0, at] * 40).to(torch.bfloat16)
        q[0, D: 2 * D] = (c.k[0, 0, at] * -40).to(torch.bfloat16)
        c.check_attention(q)
    c.check_attention(c.q(100.0))
    c.check_attention(torch.zeros_like(c.q()))


def test_attention_page_scales_far_apart():
    """Pages whose scales lie far apart: tiny and huge values side by side."""
    lens = [400]
    c = Case([2], lens, 1, 2, 16, seed=8).fill(lens, spread=6.0)
    c.check_attention(c.q(0.01))
    i = int(c.table[0, 3])
    for s in (2.0 ** -100, 2.0 ** 60):
        c.v[0, 0, 48:64] *= s / float(c.cache.v_scale[i, 0])
        c.cache.v_scale[i, 0] = s
        c.check_attention(c.q(0.01))


@pytest.mark.parametrize("shift", [-120, -40, 0, 40, 90])
def test_queries_of_every_size(shift):
    lens = [130]
    c = Case([1], lens, 1, 3, 64, seed=9).fill(lens)
    q = c.q().double() * 2.0 ** shift
    q[0, 5] *= 2.0 ** -30
    q[0, D + 7] *= 2.0 ** -60
    c.cache.k_scale *= 2.0 ** min(100, max(-100, -shift))
    c.k *= 2.0 ** min(100, max(-100, -shift))
    c.check_attention(q.to(torch.bfloat16))


def test_nan_and_infinity():
    lens = [100, 100, 100]
    c = Case([1, 1, 1], lens, 1, 2, 64, seed=10).fill(lens)
    q = c.q()
    clean = c.check_attention(q)
    bad = q.clone()
    bad[0, 3], bad[1, D + 3] = float("nan"), float("inf")
    got = c.cache.attention(c.seqs, bad, 2)
    assert bool(got[0, :D].isnan().all()) and bool(got[1, D:].isnan().all())
    assert torch.equal(got[0, D:], clean[0, D:]) and torch.equal(got[1, :D], clean[1, :D]) and torch.equal(got[2], clean[2])
    c.cache.v[int(c.table[2, 1]), 0, 9, 3] = 0x7F  # channel 9 of token 67
    got = c.cache.attention(c.seqs, q, 2)
    nan = got[2].view(2, D).isnan()
    assert bool(nan[:, 9].all()) and int(nan.sum()) == 2 and torch.equal(got[:2], clean[:2])
    c.cache.k[int(c.table[1, 0]), 0, 8, 3] = 0xFF  # a key of sequence 1: NaN scores
    got = c.cache.attention(c.seqs, q, 2)
    assert bool(got[1].isnan().all()) and torch.equal(got[0], clean[0])


def test_nan_of_a_later_token_stays_hidden():
    """Among a sequence's new tokens, a NaN in one's k or v reaches it and those behind it, in that channel, and none in front."""
    counts, lens = [40, 9], [100, 200]
    c = Case(counts, lens, 1, 3, 32, seed=21).fill(lens)
    q = c.q()
    clean = c.check_attention(q)
    t = 85  # the 26th of sequence 0's new tokens
    i, o = int(c.table[0, t // 32]), t % 32
    was = c.cache.v[i, 0, 77, o].clone()
    c.cache.v[i, 0, 77, o] = 0xFF
    got = c.cache.attention(c.seqs, q, 3).view(-1, 3, D)
    want = clean.view(-1, 3, D).clone()
    want[25:40, :, 77] = float("nan")
    assert torch.equal(got.nan_to_num(1e4), want.nan_to_num(1e4))
    c.cache.v[i, 0, 77, o] = was
    c.cache.k[i, 0, o, 5] = 0x7F
    got = c.cache.attention(c.seqs, q, 3)
    assert bool(got[25:40].isnan().all()) and torch.equal(got[:25], clean[:25]) and torch.equal(got[40:], clean[40:])


def test_entries_that_make_no_sense_are_reported_and_not_followed():
    counts, lens = [1, 2, 1, 1], [100, 70, 40, 90]
    c = Case(counts, lens, 2, 2, 32, seed=11).fill(lens)
    q = c.q()
    clean = c.check_attention(q)
    keep = c.table.clone()
    for bad in (-1, c.cache.k.shape[0], 1 << 30, -(1 << 31)):
        c.table[1, 1] = bad
        got = c.cache.attention(c.seqs, q, 4)
        torch.cuda.synchronize()
        assert sfq.device_status() == 41
        assert torch.equal(got[[0, 3, 4]], clean[[0, 3, 4]]) and bool(got.isfinite().all())
        k, v = c.k.clone(), c.v.clone()  # as if sequence 1 had no tokens 32 .. 63
        c.k[1, :, 32:], c.v[1, :, 32:] = torch.cat((k[1, :, 64:], k[1, :, :32]), 1), torch.cat((v[1, :, 64:], v[1, :, :32]), 1)
        c.lens[1] -= 32
        want, off = c.want_attention(q)
        assert bool(((got.double() - want).abs() <= off).all())
        c.lens[1] += 32
        c.k, c.v = k, v
        c.table.copy_(keep)
    c.table[1] = -1  # no key at all: zeros
    assert bool((c.cache.attention(c.seqs, q, 4)[1:3] == 0).all()) and sfq.device_status() == 41
    c.table.copy_(keep)
    good = c.seqs.seq_len.clone()
    for bad in (0, -5, c.max_pages * 32 + 1, 2 ** 31 - 1):
        c.seqs.seq_len[2] = bad
        got = c.cache.attention(c.seqs, q, 4)
        assert sfq.device_status() in (40, 41) and torch.equal(got[[0, 1, 2, 4]], clean[[0, 1, 2, 4]])
        if bad <= 0:
            assert bool((got[3] == 0).all())
    c.seqs.seq_len.copy_(good)
    starts = c.seqs.row_start.clone()
    for bad in ([0, 1, 3, 4, 9], [-2, 1, 3, 4, 5], [0, 1, 0, 4, 5], [0, 100, 3, 4, 5]):
        c.seqs.row_start.copy_(torch.tensor(bad))
        c.cache.attention(c.seqs, q, 4)
        assert sfq.device_status() == 40, bad
    c.seqs.row_start.copy_(starts)
    assert torch.equal(c.check_attention(q), clean)


def test_attention_offsets_past_32_bits():
    """A pool of more than 2^32 bytes whose last pages are used."""
    pages, kv_heads = 16 * 1024 + 40, 32  # 8 KB a page and head: 4.3 GB each for K and V
    k = torch.empty((pages, kv_heads, 64, D), dtype=torch.uint8, device="cuda")
    v = torch.empty((pages, kv_heads, D, 64), dtype=torch.uint8, device="cuda")
    big = KvCache(k, v, *(torch.zeros((pages, kv_heads), device="cuda") for _ in range(2)))
    lens = [150, 64]
    c = Case([1, 1], lens, kv_heads, 1, 64, seed=12).fill(lens)
    table = torch.full_like(c.table, -1)
    used = 0
    for b, n in enumerate(lens):
        for p in range(-(-n // 64)):
            to, at = pages - 1 - used, int(c.table[b, p])
            used += 1
            table[b, p] = to
            for name in ("k", "v", "k_scale", "v_scale"):
                getattr(big, name)[to] = getattr(c.cache, name)[at]
    q = c.q()
    want = c.check_attention(q)
    seqs = Sequences(table, c.seqs.seq_len, c.seqs.row_start, 1, 150)
    assert torch.equal(big.attention(seqs, q, c.heads), want)
    qkv = torch.randn((2, 3 * kv_heads * D), device="cuda").to(torch.bfloat16)
    big.append(seqs, qkv, kv_heads)
    c.cache.append(c.seqs, qkv, kv_heads)
    for b, n in enumerate(lens):
        to, at = int(table[b, (n - 1) // 64]), int(c.table[b, (n - 1) // 64])
        slots = (n - 1) % 64 + 1
        assert torch.equal(big.k[to, :, :slots], c.cache.k[at, :, :slots]) and torch.equal(big.v[to, :, :, :slots], c.cache.v[at, :, :, :slots])
    assert sfq.device_status() == 0


def test_attention_repeats_streams_and_graphs():
    counts, lens = [1, 5, 1], [3000, 900, 64]
    c, d = (Case(counts, lens, 2, 5, 64, seed=s).fill(lens) for s in (13, 14))
    q = c.q()
    a, b = c.check_attention(q), d.check_attention(q)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append((c.cache.attention(c.seqs, q, 10), d.cache.attention(d.seqs, q, 10)))
    torch.cuda.synchronize()
    assert all(torch.equal(x, a) and torch.equal(y, b) for x, y in outs)
    # two captured graphs that are replayed beside each other, with sequences that grow between replays
    graphs, results = [], []
    for case in (c, d):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            results.append(case.cache.attention(case.seqs, q, 10))
    for shorter in (0, 37, 64):
        for case in (c, d):
            case.lens[0] = 3000 - shorter
            case.seqs.seq_len[0] = 3000 - shorter
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
                g.replay()
        torch.cuda.synchronize()
        for case, r in ((c, results[0]), (d, results[1])):
            assert torch.equal(r, case.check_attention(q))


# ------------------------------------------------------------------------------------------------ append

def tables(rows, half, seed):
    angle = torch.rand((rows, half), device="cuda", generator=gen(seed), dtype=torch.float64) * 6.28
    return torch.cos(angle).float(), torch.sin(angle).float()


def turned(x, norm, cos, sin, at, eps):
    """(value, magnitude that its fp32 error is relative to) of head vectors x [n, heads, 128] at positions `at`."""
    x = x.double()
    if norm is not None:
        x = x / torch.sqrt((x ** 2).mean(-1, keepdim=True) + eps) * norm.double()
    mag = x.abs()
    if cos is not None:
        c, s = cos.double()[at][:, None, :], sin.double()[at][:, None, :]
        h = c.shape[-1]
        a, b = x[..., :h], x[..., h: 2 * h]
        mag = torch.cat((a.abs() + b.abs(), a.abs() + b.abs(), x[..., 2 * h:].abs()), -1)
        x = torch.cat((a * c - b * s, b * c + a * s, x[..., 2 * h:]), -1)
    return x, mag


def check_append(c, qkv, rotary_dim=0, norm=False, position=None, eps=1e-6, in_place=False, seed=0):
    """Appends the last counts[b] tokens of each sequence to what is cached, and compares every byte of the pool."""
    heads, kv_heads, page = c.heads, c.kv_heads, c.page
    most = max(c.lens + [1])
    cos, sin = tables(most if position is None else int(position.max()) + 1, rotary_dim // 2, seed) if rotary_dim else (None, None)
    norms = (1 + 0.1 * torch.randn((2, D), device="cuda", generator=gen(seed + 1))).to(torch.bfloat16) if norm else (None, None)
    before = {n: getattr(c.cache, n).clone() for n in ("k", "v", "k_scale", "v_scale")}
    rotary = Rotary(cos, sin, position, norms[0], norms[1], eps) if rotary_dim or norm else None
    original = qkv.clone()
    q = c.cache.append(c.seqs, qkv, heads, q_out=qkv[:, : heads * D] if in_place else None, rotary=rotary)
    torch.cuda.synchronize()
    assert sfq.device_status() == 0
    rows = original.view(original.shape[0], heads + 2 * kv_heads, D)
    after = {n: getattr(c.cache, n) for n in before}
    untouched = {n: torch.ones_like(before[n], dtype=torch.bool) for n in ("k", "v")}
    scale_untouched = torch.ones_like(before["k_scale"], dtype=torch.bool)
    for b, n in enumerate(c.counts):
        if n == 0:
            continue
        r0, p0 = c.start[b], c.lens[b] - n
        at = torch.arange(p0, p0 + n, device="cuda") if position is None else position[r0: r0 + n].long()
        if heads:
            want, mag = turned(rows[r0: r0 + n, :heads], norms[0], cos, sin, at, eps)
            off = 2.0 ** -8 * want.abs() + 2.0 ** -15 * mag + 1e-38
            assert bool(((q[r0: r0 + n].view(n, heads, D).double() - want).abs() <= off).all())
        fresh = {"k": turned(rows[r0: r0 + n, heads: heads + kv_heads], norms[1], cos, sin, at, eps), "v": (rows[r0: r0 + n, heads + kv_heads:].double(), None)}
        t = p0
        while t < p0 + n:
            end = min(p0 + n, (t // page + 1) * page)
            i, o, e = int(c.table[b, t // page]), t % page, t % page + end - t
            scale_untouched[i] = False
            untouched["k"][i, :, :e], untouched["v"][i, :, :, :e] = False, False
            for name in ("k", "v"):
                x, mag = fresh[name]
                x = x[t - p0: end - p0].transpose(0, 1)
                slack = 2.0 ** -16 * mag[t - p0: end - p0].transpose(0, 1) if mag is not None else torch.zeros_like(x)
                old = before[name + "_scale"][i].double() if o else torch.zeros(kv_heads, dtype=torch.float64, device="cuda")
                got = after[name + "_scale"][i].double()
                finite = torch.where(x.isfinite(), x.abs(), 0.0)
                low, high = (torch.maximum(old, scale_for((finite + f * slack).amax((1, 2)))) for f in (-1, 1))
                assert bool(((got == low) | (got == high)).all()), (b, t, name)
                codes = after[name][i] if name == "k" else after[name][i].transpose(1, 2)
                have = values_of(codes)
                if o:  # what was there: rounded again where the scale has grown, untouched where it has not
                    was = values_of(before[name][i] if name == "k" else before[name][i].transpose(1, 2))[:, :o]
                    want_old = torch.where((got == old)[:, None, None], was, nearest_e4m3(was * (old / got)[:, None, None]))
                    assert torch.equal(have[:, :o].nan_to_num(500.0), want_old.nan_to_num(500.0))
                mine, y, d = have[:, o:e], x / got[:, None, None], slack / got[:, None, None]
                ok = (mine == nearest_e4m3(y)) | (mine == nearest_e4m3(y - d)) | (mine == nearest_e4m3(y + d)) | (mine.isnan() & y.isnan())
                assert bool(ok.all()), (b, t, name, int((~ok).sum()))
            t = end
    for name in ("k", "v"):
        assert torch.equal(after[name][untouched[name]], before[name][untouched[name]])
        s, w = after[name + "_scale"][scale_untouched], before[name + "_scale"][scale_untouched]
        assert torch.equal(s.nan_to_num(-1.0), w.nan_to_num(-1.0))
    if heads:
        assert torch.equal(q[c.rows:], original[c.rows:, : heads * D] if in_place else q[c.rows:])
    assert torch.equal(qkv[:, heads * D:], original[:, heads * D:])
    return q


def new_qkv(c, extra=0, sigma=1.0):
    n = (c.heads + 2 * c.kv_heads) * D
    return (sigma * torch.randn((c.rows + extra, n), device="cuda", generator=c.g)).to(torch.bfloat16)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("kv_heads,group", [(1, 1), (2, 5), (3, 8), (1, 13)])
@pytest.mark.parametrize("rotary,norm", [(0, False), (128, False), (96, True), (16, True), (64, False)])
def test_append_single_tokens(page, kv_heads, group, rotary, norm):
    lens = [1, 2, 16, 17, 33, 64, 65, 128, 129, 256, 257, 300]
    c = Case([1] * len(lens), lens, kv_heads, group, page, seed=page).fill([n - 1 for n in lens])
    check_append(c, new_qkv(c), rotary, norm)


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("kv_heads,group", [(1, 4), (2, 3)])
@pytest.mark.parametrize("rotary,norm", [(0, True), (96, False), (128, True)])
def test_append_prompts(page, kv_heads, group, rotary, norm):
    """Several tokens: from an empty sequence, inside one page, over page borders, none at all; rows behind the last sequence."""
    counts, lens = [1, 3, 0, 17, 100, 0, 64, 200, 5, 129], [1, 3, 50, 40, 100, 0, 77, 331, 260, 129]
    c = Case(counts, lens, kv_heads, group, page, seed=page).fill([n - m for n, m in zip(lens, counts)])
    check_append(c, new_qkv(c, extra=4), rotary, norm, in_place=True)


def test_append_without_queries_and_with_positions():
    counts, lens = [4, 1], [9, 30]
    c = Case(counts, lens, 2, 2, 16, seed=3).fill([5, 29])
    position = torch.tensor([700, 3, 3, 0, 41], dtype=torch.int32, device="cuda")
    check_append(c, new_qkv(c), 96, True, position)
    kv = new_qkv(c)[:, 4 * D:].contiguous()
    c.heads = 0
    check_append(c, kv, 96, False, position)


def test_scales_grow_and_start_anew():
    """A page that is filled token by token with values that grow, shrink, vanish: every step against the definition, so that codes are
    rounded again exactly where the scale has grown."""
    page = 16
    c = Case([1], [3 * page], 2, 1, page, seed=4)
    for t in range(3 * page):
        c.lens[0] = t + 1
        c.seqs.seq_len[0] = t + 1
        sigma = [1.0, 0.0, 3.0, 2.0 ** -9, 100.0, 2.0 ** -60, 2.0 ** 40, 1e-30, 0.0, 2.0 ** 90][t % 10] if t >= page else 1.0 + 0.1 * t
        check_append(c, new_qkv(c, sigma=sigma), 0, False)


def test_a_zero_page_and_values_at_the_border():
    c = Case([1], [1], 1, 1, 16, seed=5)
    qkv = new_qkv(c)
    qkv[:, D:] = 0
    check_append(c, qkv)
    assert float(c.cache.k_scale[int(c.table[0, 0]), 0]) == 2.0 ** -100
    for top, scale in ((448.0, 1.0), (450.0, 2.0), (447.0, 1.0), (3.5, 2.0 ** -7), (3.3e38, 2.0 ** 120), (1e-33, 2.0 ** -100)):
        qkv[:, D:] = (torch.rand((1, 2 * D), device="cuda") * top * 0.5).to(torch.bfloat16)
        qkv[0, D + 5], qkv[0, 2 * D + 9] = top, -top
        check_append(c, qkv)
        i = int(c.table[0, 0])
        assert float(c.cache.k_scale[i, 0]) == scale == float(c.cache.v_scale[i, 0])


def test_append_infinity_and_nan():
    """The scale follows the finite values; infinities are stored as the largest code, NaN as NaN."""
    c = Case([2], [2], 1, 1, 16, seed=6)
    qkv = new_qkv(c)
    qkv[0, D + 1], qkv[1, D + 2], qkv[0, 2 * D + 3] = float("inf"), float("nan"), float("-inf")
    c.cache.append(c.seqs, qkv, 1)
    i = int(c.table[0, 0])
    k, v = values_of(c.cache.k[i, 0, :2]), values_of(c.cache.v[i, 0, :, :2])
    assert float(k[0, 1]) == 448 and bool(k[1, 2].isnan()) and float(v[3, 0]) == -448
    assert float(c.cache.k_scale[i, 0]) <= 2.0 ** -5 and int(k.isnan().sum()) == 1 and int(v.isnan().sum()) == 0


def test_append_entries_that_make_no_sense():
    counts, lens = [1, 20, 1], [40, 50, 10]
    c = Case(counts, lens, 2, 2, 16, seed=7).fill([39, 30, 9])
    qkv = new_qkv(c)
    keep = {n: getattr(c.cache, n).clone() for n in ("k", "v", "k_scale", "v_scale")}
    table = c.table.clone()
    for bad in (-1, c.cache.k.shape[0], 1 << 30):
        c.table[1, 1:4] = bad
        c.table[0, 2] = bad
        q = c.cache.append(c.seqs, qkv, 4)
        torch.cuda.synchronize()
        assert sfq.device_status() == 41 and torch.equal(q, qkv[:, : 4 * D])
        mine = int(table[2, 0])
        for n, t in keep.items():  # nothing but sequence 2's page is written
            now = getattr(c.cache, n).clone()
            now[mine] = t[mine]
            assert torch.equal(now.nan_to_num(-1.0) if now.is_floating_point() else now, t.nan_to_num(-1.0) if t.is_floating_point() else t)
        c.table.copy_(table)
    cos, sin = tables(20, 48, 1)
    c.cache.append(c.seqs, qkv, 4, rotary=Rotary(cos, sin))
    torch.cuda.synchronize()
    assert sfq.device_status() == 42
    for name, bad in (("seq_len", [40, 19, 10]), ("seq_len", [0, 50, 10]), ("seq_len", [40, 50, 10 ** 9]), ("row_start", [0, 1, 500, 22]), ("row_start", [5, 1, 21, 22])):
        t = getattr(c.seqs, name)
        good = t.clone()
        t.copy_(torch.tensor(bad))
        c.cache.append(c.seqs, qkv, 4)
        torch.cuda.synchronize()
        assert sfq.device_status() in (40, 41)
        t.copy_(good)


@pytest.mark.parametrize("max_new", [1, 7, 1000])
def test_append_estimates_only_size_the_launch(max_new):
    counts, lens = [100, 1, 33], [140, 100, 33]
    c = Case(counts, lens, 2, 2, 16, seed=8).fill([40, 99, 0])
    c.seqs.max_new = max_new
    check_append(c, new_qkv(c), 128, True)


def test_append_in_a_graph_and_beside_others():
    """A step captured once and replayed as the sequences grow; other caches are written beside it."""
    lens = [10, 60, 128]
    c, d = (Case([1] * 3, [n + 20 for n in lens], 2, 2, 64, seed=s).fill(lens) for s in (9, 9))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    qkv = new_qkv(c)
    steps = [new_qkv(c) for _ in range(20)]
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    cos, sin = tables(200, 64, 3)
    rotary = Rotary(cos, sin)
    graph = torch.cuda.CUDAGraph()
    c.seqs.seq_len.copy_(length)
    with torch.cuda.graph(graph):
        q = c.cache.append(c.seqs, qkv, 4, rotary=rotary)
        o = c.cache.attention(c.seqs, q, 4)
    torch.cuda.synchronize()
    for t, x in enumerate(steps):
        with torch.cuda.stream(streams[0]):
            qkv.copy_(x)
            c.seqs.seq_len.copy_(length + t + 1)
            graph.replay()
        with torch.cuda.stream(streams[1]):
            d.seqs.seq_len.copy_(length + t + 1)
            p = d.cache.append(d.seqs, x, 4, rotary=rotary)
            r = d.cache.attention(d.seqs, p, 4)
        torch.cuda.synchronize()
        assert torch.equal(q, p) and torch.equal(o, r)
    assert torch.equal(c.cache.k, d.cache.k) and torch.equal(c.cache.v, d.cache.v)
    assert sfq.device_status() == 0


# ------------------------------------------------------------------------------------------------ together

@pytest.mark.parametrize("fmt", ["nvfp4", "nf4"])
def test_decoding_steps(fmt):
    """A layer of a small model, as a program would use the operators: a prompt of several tokens, then single ones. Each step's input to
    an operator is what the one before it gave, and each result is compared with its definition on that input."""
    from test_gpu_matvec import Weight, check

    heads, kv_heads, batch = 6, 2, 3
    hidden = heads * D
    wqkv, wo, w1, w2 = (Weight(fmt, n, k, i) for i, (n, k) in enumerate((((heads + 2 * kv_heads) * D, hidden), (hidden, hidden), (1024, hidden), (hidden, 512))))
    prompts, steps = [5, 1, 33], 4
    total = [n + steps for n in prompts]
    c = Case(prompts, total, kv_heads, heads // kv_heads, 16, seed=20)
    x = None
    norm_x = lambda t: (t.float() * torch.rsqrt((t.float() ** 2).mean(-1, keepdim=True) + 1e-6)).to(torch.bfloat16)  # noqa: E731
    for step in range(steps + 1):
        counts = prompts if step == 0 else [1] * batch
        c.counts, c.rows = counts, sum(counts)
        c.start = [sum(counts[:b]) for b in range(batch + 1)]
        c.lens = [n + step for n in prompts]
        c.seqs = Sequences(c.table, torch.tensor(c.lens, dtype=torch.int32, device="cuda"), torch.tensor(c.start, dtype=torch.int32, device="cuda"),
                           max(counts), max(c.lens))
        x = norm_x(torch.randn((c.rows, hidden), device="cuda", generator=c.g)) if x is None or step == 0 else norm_x(x[-batch:])
        qkv = norm_x(check(wqkv, x))
        q = check_append(c, qkv, 96, True, seed=20)
        for b, n in enumerate(c.lens):
            for t in range(n):  # what the cache now stands for
                i, o = int(c.table[b, t // 16]), t % 16
                c.k[b, :, t] = values_of(c.cache.k[i, :, o]) * c.cache.k_scale[i].double()[:, None]
                c.v[b, :, t] = values_of(c.cache.v[i, :, :, o].contiguous()) * c.cache.v_scale[i].double()[:, None]
        o = check(wo, norm_x(c.check_attention(q)))
        h = check(w1, norm_x(o + x), "swiglu")
        x = check(w2, norm_x(h))
    assert sfq.device_status() == 0


FIRST_CALL = """
import torch
import slopfab_b200 as sfq
from slopfab_b200.kv_cache import KvCache, Sequences
i32 = lambda *v: torch.tensor(v, dtype=torch.int32, device="cuda")
cache = KvCache.empty(4, 2, 64)
seqs = Sequences(i32(2, 0).view(1, 2), i32(3), i32(0, 3), 3, 3)
qkv = torch.randn((3, 8 * 128), device="cuda").to(torch.bfloat16)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = cache.attention(seqs, cache.append(seqs, qkv, 4), 4)
graph.replay()
torch.cuda.synchronize()
assert torch.equal(out, cache.attention(seqs, cache.append(seqs, qkv, 4), 4)) and sfq.device_status() == 0
print("same")
"""


def test_first_call_of_a_process_inside_a_capture():
    out = subprocess.run([sys.executable, "-c", FIRST_CALL], capture_output=True, text=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
    assert out.returncode == 0 and out.stdout.strip() == "same", out.stderr


def test_out_beside_q_in_one_buffer():
    """q and out are columns of the same rows, q_out is q's place in the projection."""
    c = Case([2, 1], [40, 33], 2, 2, 16, seed=31).fill([38, 32])
    wide = torch.randn((3, 4 * D + 2 * D * 2 + 4 * D), device="cuda", generator=c.g).to(torch.bfloat16)
    n = (4 + 2 * 2) * D
    fused = wide[:, :n].contiguous()
    q = c.cache.append(c.seqs, wide[:, :n], 4, q_out=wide[:, : 4 * D])
    out = c.cache.attention(c.seqs, q, 4, out=wide[:, n:])
    assert torch.equal(q, fused[:, : 4 * D]) and torch.equal(wide[:, 4 * D: n], fused[:, 4 * D:])
    assert torch.equal(out, c.cache.attention(c.seqs, fused[:, : 4 * D], 4))
    with pytest.raises(sfq.SfqError, match="overlap"):
        c.cache.attention(c.seqs, wide[:, : 4 * D], 4, out=wide[:, D: 5 * D])
    with pytest.raises(sfq.SfqError, match="apart"):
        c.cache.append(c.seqs, wide[:, :n], 4, q_out=wide[:, D: 5 * D])


@pytest.mark.parametrize("lens", [[2100, 64, 0, 1, 700, 65, 1300], [2000] * 7, [2000, 1990, 1950, 2000, 1900, 1980, 1970], [3000, 0, 0, 0, 0, 0, 5], [1, 0, 1, 1, 0, 1, 1]])
@pytest.mark.parametrize("max_len", [None, 64, 100000])
@pytest.mark.parametrize("news", [1, 5])
def test_sequences_of_all_lengths_in_parts(lens, max_len, news):
    """Even and ragged batches, divided as the host's and the device's idea of the lengths has it."""
    counts = [min(news, n) for n in lens]
    c = Case(counts, lens, 2, 4, 64, seed=41).fill(lens)
    c.seqs.max_len = max_len or max(lens)
    c.check_attention(c.q())


@pytest.mark.parametrize("most", [1, 2, 5, 16, 17, 40])
@pytest.mark.parametrize("page", [16, 64, 256])
@pytest.mark.parametrize("norm", [False, True])
def test_append_some_tokens(most, page, norm):
    """Each form of the launch, with sequences of fewer tokens and of none, over page borders."""
    counts = [most, 1, 0, max(most - 1, 1), most, (most + 1) // 2]
    past = [0, page - 1, 7, page - 2, 3 * page - most // 2, page]
    c = Case(counts, [a + b for a, b in zip(counts, past)], 2, 3, page, seed=51).fill(past)
    check_append(c, new_qkv(c), 96, norm)


@pytest.mark.parametrize("even", [False, True])
def test_more_sequences_than_lanes(even):
    lens = [700 if even else (37 * i * i) % 900 for i in range(70)]
    c = Case([min(1, n) for n in lens], lens, 1, 4, 64, seed=61).fill(lens)
    c.check_attention(c.q())


def test_a_row_of_a_buffer_of_odd_width():
    """One token whose q, k, v, q_out and out are rows of buffers with pitches that several rows could not have."""
    c = Case([1], [90], 2, 2, 64, seed=71).fill([89])
    d = Case([1], [90], 2, 2, 64, seed=71).fill([89])
    qkv = new_qkv(c)
    rows = [torch.full((2, n * D + 10), 3.0, dtype=torch.bfloat16, device="cuda") for n in (8, 4, 4)]
    rows[0][0, : 8 * D] = qkv[0]
    q = c.cache.append(c.seqs, rows[0][:1, : 8 * D], 4, q_out=rows[1][:1, : 4 * D])
    out = c.cache.attention(c.seqs, q, 4, out=rows[2][:1, : 4 * D])
    want = d.cache.append(d.seqs, qkv, 4)
    assert torch.equal(q, want) and torch.equal(out, d.cache.attention(d.seqs, want, 4))
    for r in rows[1:]:
        assert bool((r[0, 4 * D:] == 3).all()) and bool((r[1] == 3).all())
    assert sfq.device_status() == 0


@pytest.mark.parametrize("size", [2.0 ** 15, 2.0 ** 21, 2.0 ** 24, 2.0 ** 25])
@pytest.mark.parametrize("shift", [-60, 0, 60])
def test_scores_whose_last_place_is_an_octave_and_more(size, shift):
    """Scores of up to `size` octaves, in fp32 steps of 2^-24 of that: the key with all the weight is the result, whatever its page's scale."""
    n = 200
    c = Case([1], [n], 1, 2, 16, seed=82).fill([n])
    page = c.table[0, : -(-n // 16)].long()
    c.cache.v_scale[page] *= 2.0 ** shift
    c.v *= 2.0 ** shift
    c.cache.k_scale[page] = 1.0
    c.cache.k[page] = 0
    one = torch.tensor([1.0, 0.875]).to(torch.float8_e4m3fn).view(torch.uint8).tolist()
    for at in range(0, n, 7):  # this key is alone at the top
        c.cache.k[page[:, None], 0, torch.arange(16, device="cuda"), 0] = one[1]
        c.cache.k[page[at // 16], 0, at % 16, 0] = one[0]
        q = torch.zeros_like(c.q())
        q[0, 0], q[0, D] = 1.0, 1.0
        got = c.cache.attention(c.seqs, q, 2, scale=size * math.log(2))
        want = c.v[0, 0, at].to(torch.bfloat16)
        assert torch.equal(got.view(2, D), want.expand(2, D)), at


@pytest.mark.parametrize("news,group", [(1, 5), (3, 4), (40, 5)])
def test_heads_and_tokens_stand_for_themselves(news, group):
    """An infinite or NaN query, and one whose scores lie far from the others', changes no bit of the queries beside it, which share
    its tile."""
    c = Case([news] * 8, [100 + i for i in range(8)], 8, group, 32, seed=83).fill([100 + i for i in range(8)])
    for seed in range(8):
        q = c.q()
        clean = c.check_attention(q).view(-1, 8, group, D)
        for bad in (float("inf"), float("nan"), 3e4, -3e4):
            other = q.clone()
            other.view(-1, 8, group, D)[:, :, seed % group, 9] = bad
            got = c.cache.attention(c.seqs, other, c.heads).view(-1, 8, group, D)
            got[:, :, seed % group] = clean[:, :, seed % group]
            assert torch.equal(got, clean), (seed, bad, int((got != clean).sum()))


@pytest.mark.parametrize("octaves", [14.7, 18.3, 22.3, 24.5, 25.5, 28.6])
@pytest.mark.parametrize("news,group,n", [(1, 5, 700), (3, 4, 700), (6, 4, 700), (1, 4, 20000)])
def test_a_key_that_takes_the_weight_and_has_no_value(octaves, news, group, n):
    """The first key has nearly all the weight, and its value is zero: the output is what the others leave, each of them 2^-octaves of
    the first one's weight. The bound is the file's: every weight is good to 2^-11 of itself."""
    c = Case([news], [n], 1, group, 64, seed=81).fill([n])
    page = c.table[0, : -(-n // 64)].long()
    c.cache.k[page] = 0
    c.cache.k[page[0], 0, 0, 0] = torch.tensor(1.0).to(torch.float8_e4m3fn).view(torch.uint8).item()
    c.cache.v[page] &= 0x7F  # magnitudes
    c.cache.v[page[0], 0, :, 0] = 0
    c.k.zero_()
    c.k[0, 0, 0, 0] = float(c.cache.k_scale[page[0], 0])
    c.v.abs_()
    c.v[0, 0, 0] = 0
    q = torch.zeros_like(c.q())
    q.view(-1, group, D)[..., 0] = 1.0
    c.check_attention(q, scale=octaves * math.log(2) / float(c.k[0, 0, 0, 0]))


def test_values_near_the_smallest_scale():
    """The same weights over values 2^-90 as large give a result 2^-90 as large, though it comes from small weights: the key that has
    all but 2^-8 of the weight has no value, and each of the others 2^-18 of its weight. All values are positive: a rounding of each
    result, and as much for the weights."""
    n = 900
    c = Case([1], [n], 1, 4, 16, seed=84).fill([n])
    page = c.table[0, : -(-n // 16)].long()
    c.cache.k[page] = 0
    c.cache.k_scale[page] = 1.0
    c.cache.k[page[3], 0, 9, 0] = 0x38  # 1.0
    c.cache.v[page] &= 0x7F
    c.cache.v[page[3], 0, :, 9] = 0
    q = torch.zeros((1, 4 * D), dtype=torch.bfloat16, device="cuda")
    q[0, ::D] = 1.0
    c.cache.v_scale[page] = 2.0 ** -7
    want = c.cache.attention(c.seqs, q, 4, scale=18 * math.log(2)).double()
    c.cache.v_scale[page] = 2.0 ** -97
    got = c.cache.attention(c.seqs, q, 4, scale=18 * math.log(2)).double() * 2.0 ** 90
    assert float(want.min()) > 0 and bool(((got - want).abs() <= 2.0 ** -7 * want).all())


@pytest.mark.parametrize("counts,past", [([1, 0, 1, 1], [0, 5, 63, 64]), ([5, 0, 16, 1], [0, 5, 60, 64]), ([5, 0, 40, 130], [0, 5, 60, 63])])
def test_append_writes_no_row_or_column_beyond_its_own(counts, past):
    """A q_out of its own, wider than the heads and longer than the sequences' rows, in each form of the launch: what is written is what a
    plain call gives, and the rest of the buffer keeps what it held."""
    lens = [a + b for a, b in zip(counts, past)]
    c, d = (Case(counts, lens, 2, 3, 64, seed=91).fill(past) for _ in range(2))
    qkv = new_qkv(c, extra=7)
    cos, sin = tables(max(lens), 48, 5)
    norms = (1 + 0.1 * torch.randn((2, D), device="cuda", generator=gen(6))).to(torch.bfloat16)
    rotary = Rotary(cos, sin, None, norms[0], norms[1])
    buffer = torch.full((c.rows + 7, c.heads * D + 24), -9.0, dtype=torch.bfloat16, device="cuda")
    q = c.cache.append(c.seqs, qkv, c.heads, q_out=buffer[:, 8: 8 + c.heads * D], rotary=rotary)
    rows = qkv[: c.rows].view(c.rows, -1, D)[:, : c.heads]
    at = torch.cat([torch.arange(p, n, device="cuda") for p, n in zip(past, lens)])
    want, mag = turned(rows, norms[0], cos, sin, at, rotary.eps)
    got = q[: c.rows].reshape(c.rows, c.heads, D).double()
    assert bool(((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -15 * mag + 1e-38).all())
    keep = buffer.clone()
    keep[: c.rows, 8: 8 + c.heads * D] = -9.0
    assert bool((keep == -9.0).all())
    assert torch.equal(d.cache.append(d.seqs, qkv, d.heads, rotary=rotary)[: c.rows], q[: c.rows])
    for name in ("k", "v"):
        assert torch.equal(getattr(c.cache, name), getattr(d.cache, name))
    assert sfq.device_status() == 0


def test_a_position_outside_the_tables_stands_for_the_first():
    """It is reported, and the token is stored as if it stood at position 0."""
    counts, lens = [1, 6], [9, 30]
    c, d = (Case(counts, lens, 2, 2, 16, seed=92).fill([8, 24]) for _ in range(2))
    qkv = new_qkv(c)
    cos, sin = tables(50, 48, 7)
    good = torch.tensor([4, 0, 2, 0, 49, 0, 7], dtype=torch.int32, device="cuda")
    bad = torch.tensor([4, -1, 2, 50, 49, -(1 << 31), 7], dtype=torch.int32, device="cuda")
    q = c.cache.append(c.seqs, qkv, 4, rotary=Rotary(cos, sin, good))
    assert sfq.device_status() == 0
    r = d.cache.append(d.seqs, qkv, 4, rotary=Rotary(cos, sin, bad))
    assert sfq.device_status() == 42
    assert torch.equal(q, r) and all(torch.equal(getattr(c.cache, n), getattr(d.cache, n)) for n in ("k", "v"))


@pytest.mark.parametrize("pad", [0, 64, 10])
def test_one_token_in_place(pad):
    c = Case([1], [70], 2, 3, 64, seed=93).fill([69])
    d = Case([1], [70], 2, 3, 64, seed=93).fill([69])
    qkv = new_qkv(c)
    wide = torch.full((2, 10 * D + pad), 5.0, dtype=torch.bfloat16, device="cuda")
    wide[0, : 10 * D] = qkv[0]
    cos, sin = tables(70, 64, 8)
    q = c.cache.append(c.seqs, wide[:1, : 10 * D], 6, q_out=wide[:1, : 6 * D], rotary=Rotary(cos, sin))
    assert q.data_ptr() == wide.data_ptr() and torch.equal(q, d.cache.append(d.seqs, qkv, 6, rotary=Rotary(cos, sin)))
    assert torch.equal(wide[0, 6 * D: 10 * D], qkv[0, 6 * D:]) and bool((wide[1] == 5).all()) and bool((wide[0, 10 * D:] == 5).all())
    assert torch.equal(c.cache.k, d.cache.k) and torch.equal(c.cache.v, d.cache.v)


@pytest.mark.parametrize("shift", [-130, -128, -126, -124])
def test_the_smallest_queries_over_the_largest_keys(shift):
    """Scores of an ordinary size from queries near the end of bf16's range and keys near the other end of the scales'."""
    c = Case([1], [300], 1, 4, 64, seed=94).fill([300])
    c.cache.k_scale *= 2.0 ** 125
    c.k *= 2.0 ** 125
    q = (c.q().clamp(-4, 4).double() * 2.0 ** shift).to(torch.bfloat16)
    c.check_attention(q)
    c.check_attention(q, scale=0.3)


@pytest.mark.parametrize("size", [2.0 ** -9, 1.0, 4.0, 2.0 ** 40])
def test_negative_scales(size):
    """A page whose scale of V, or of K, is negative stands for the negative of its codes' values."""
    c = Case([2], [200], 2, 3, 32, seed=95).fill([200])
    for name, t in (("v_scale", c.v), ("k_scale", c.k)):
        for p in (0, 3, 6):
            i = int(c.table[0, p])
            was = getattr(c.cache, name)[i].clone()
            now = -(torch.full_like(was, size) if name == "v_scale" else was)
            t[0, :, 32 * p: 32 * p + 32] *= (now / was).double()[:, None, None]
            getattr(c.cache, name)[i] = now
        c.check_attention(c.q())
