"""sfq_linear_matvec against the stored weight and x in 64 bits.

Bounds. Sums: a sum of K products in fp32 in any order is off by K 2^-24 of the sum S of the products' magnitudes at most; the
products themselves are exact or rounded once more (NVFP4: 8 + 6 significant bits; two more roundings where a scale is applied), so
(K + 4) 2^-24 S. NF4: the 16 table entries may be held as fp16, 2^-11 of S. Output: one rounding to bf16, 2^-8 of the value. GELU
has a slope of 1.13 at most, silu of 1.1 and |silu(z)| <= |z|; tanhf and __expf are good to 2^-20 of values of at most 1."""
import ctypes as C

import numpy as np
import pytest
import torch

import slopfab_b200 as sfq
from helpers import dev, pack_nvfp4

pytestmark = pytest.mark.gpu

E2M1 = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6, -0., -.5, -1, -1.5, -2, -3, -4, -6], dtype=torch.float64)
ACTS = {"none": sfq.ACT_NONE, "gelu": sfq.ACT_GELU_TANH, "swiglu": sfq.ACT_SWIGLU}


class Weight:
    """A stored weight of random bytes, its descriptor and its values in 64 bits."""

    def __init__(self, fmt, n, k, seed, bias=None, block=64, nested=256):
        g = torch.Generator("cuda").manual_seed(seed)
        rand = lambda lo, hi, *shape: torch.randint(lo, hi, shape, device="cuda", generator=g, dtype=torch.int64).to(torch.uint8)  # noqa: E731
        self.fmt, self.n, self.k = fmt, n, k
        self.data = rand(0, 256, n, k // 2)
        codes = torch.stack((self.data >> 4, self.data & 15), -1).view(n, k).long()
        f = dict(data=sfq.ptr(self.data), out_features=n, in_features=k)
        if fmt == "nvfp4":
            self.scale = rand(0, 0x7F, n * k // 16)  # every scale but NaN: subnormals, zero and 448 among them
            f.update(format=sfq.NVFP4, block_scale=sfq.ptr(self.scale), global_scale=0.003)
            s = self.scale.view(n // 128, k // 64, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(n, k // 16).contiguous()
            s = s.view(torch.float8_e4m3fn).double().repeat_interleave(16, 1)
            self.values = E2M1.cuda()[codes] * s * float(np.float32(0.003))
        else:
            blocks = -(-n * k // block)
            self.scale = rand(0, 256, blocks)
            self.map = torch.sort(torch.randn(16, device="cuda", generator=g)).values
            self.nested_map = torch.linspace(-1, 1, 256, device="cuda")
            self.nested_absmax = 0.01 + 0.01 * torch.rand(-(-blocks // nested), device="cuda", generator=g)
            f.update(format=sfq.NF4, nf4_absmax=sfq.ptr(self.scale), nf4_quant_map=sfq.ptr(self.map), nf4_nested_quant_map=sfq.ptr(self.nested_map),
                     nf4_nested_absmax=sfq.ptr(self.nested_absmax), nf4_block_size=block, nf4_nested_block_size=nested, nf4_nested_offset=0.02)
            b = torch.arange(n * k, device="cuda") // block
            absmax = self.nested_map.double()[self.scale.long()[b]] * self.nested_absmax.double()[b // nested] + float(np.float32(0.02))
            self.values = self.map.double()[codes] * absmax.view(n, k)
        self.bias = None
        if bias is not None:
            self.bias = torch.randn(n, device="cuda", generator=g).to(bias)
            f.update(bias=sfq.ptr(self.bias), bias_format=sfq.F32 if bias == torch.float32 else sfq.BF16)
        self.desc = sfq.new_weight(**f)

    def want(self, x, act):
        """(values, how far a result may be off) of act(x W^T + b)."""
        xd = x.double()
        z, mag = xd @ self.values.T, xd.abs() @ self.values.abs().T
        if self.bias is not None:
            z, mag = z + self.bias.double(), mag + self.bias.double().abs()
        off = mag * ((self.k + 4) * 2.0 ** -24 + (2.0 ** -11 if self.fmt == "nf4" else 0.0))
        if act == "gelu":
            y = 0.5 * z * (1 + torch.tanh(0.7978845608028654 * (z + 0.044715 * z ** 3)))
            off = 1.13 * off + 2.0 ** -20 * z.abs()
        elif act == "swiglu":
            a, b, c, d = z[:, : self.n // 2], z[:, self.n // 2:], off[:, : self.n // 2], off[:, self.n // 2:]
            y = a * torch.sigmoid(a) * b
            off = 1.1 * c * b.abs() + (a.abs() + 1.1 * c) * d + 2.0 ** -20 * (a * b).abs()
        else:
            y = z
        return y, off + 2.0 ** -8 * (y.abs() + off) + 1e-38


def draw_x(rows, k, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    x = torch.randn((rows, k), device="cuda", generator=g).to(torch.bfloat16)
    return torch.where(torch.rand((rows, k), device="cuda", generator=g) < 1e-3, x * 20, x)


def check(w, x, act="none"):
    y = torch.full((x.shape[0], w.n // 2 if act == "swiglu" else w.n), float("nan"), dtype=torch.bfloat16, device="cuda")
    got = sfq.linear_matvec(w.desc, x, y, ACTS[act])
    assert got is y
    want, off = w.want(x, act)
    assert bool(((y.double() - want).abs() <= off).all())
    # And far nearer on the whole than at worst: a rounding of 2^-8 of each value, or of 2^-134 where bf16 is subnormal (its steps are
    # 2^-133 there), with as much again for the sum.
    far, size = float((y.double() - want).norm()), float(want.norm())
    assert far <= 2.0 ** -8 * size + 2.0 ** -133 * y.numel() ** 0.5
    return y


@pytest.mark.parametrize("fmt,n,k", [("nvfp4", 128, 64), ("nvfp4", 256, 192), ("nvfp4", 384, 1024), ("nvfp4", 1152, 4160), ("nvfp4", 640, 13824),
                                     ("nf4", 2, 64), ("nf4", 34, 128), ("nf4", 7, 192), ("nf4", 250, 1088), ("nf4", 1025, 4160), ("nf4", 514, 13824)])
@pytest.mark.parametrize("rows", [1, 2, 3, 8, 9, 16, 17, 37])
def test_shapes(fmt, n, k, rows):
    check(Weight(fmt, n, k, n + k), draw_x(rows, k, rows))


@pytest.mark.parametrize("fmt,n,k", [("nvfp4", 384, 704), ("nvfp4", 128, 5120), ("nf4", 42, 192), ("nf4", 1026, 2048)])
@pytest.mark.parametrize("rows", [1, 5, 12])
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("bias", [None, torch.float32, torch.bfloat16])
def test_activations_and_bias(fmt, n, k, rows, act, bias):
    check(Weight(fmt, n, k, n, bias), draw_x(rows, k, rows) * (0.05 if fmt == "nvfp4" else 0.5), act)


@pytest.mark.parametrize("block,nested", [(64, 1), (64, 256), (128, 4), (4096, 256)])
def test_nf4_block_sizes(block, nested):
    check(Weight("nf4", 130, 448, block, None, block, nested), draw_x(3, 448, 1))


def test_a_packed_weight_against_the_dense_arm():
    """Beside the library's own dense arm: bf16(w) has a rounding of 2^-8 of each weight."""
    rng = np.random.default_rng(3)
    n, k = 256, 512
    data, scale, top = pack_nvfp4((0.02 * rng.standard_normal((n, k))).astype(np.float32))
    keep = dev(data), dev(scale)
    w = sfq.new_weight(format=sfq.NVFP4, data=sfq.ptr(keep[0]), block_scale=sfq.ptr(keep[1]), global_scale=top, out_features=n, in_features=k)
    x = draw_x(5, k, 1)
    dense = torch.empty((n, k), dtype=torch.bfloat16, device="cuda")
    sfq.check(sfq.lib.sfq_unpack_nvfp4_bf16(sfq.ptr(keep[0]), sfq.ptr(keep[1]), top, sfq.ptr(dense), n, k, sfq.stream_ptr()))
    want, mag = sfq.LinearRunner().forward(w, x).double(), x.double().abs() @ dense.double().abs().T
    assert bool(((sfq.linear_matvec(w, x).double() - want).abs() <= 2.0 ** -8 * (mag + 2 * want.abs()) + 1e-6).all())


@pytest.mark.parametrize("fmt", ["nvfp4", "nf4"])
def test_values_of_every_size(fmt):
    """Rows whose elements lie further apart than fp16 reaches, tiny and huge rows, zeros, subnormals; each row stands for itself."""
    n, k = 256, 1024
    w = Weight(fmt, n, k, 5)
    x = draw_x(9, k, 2).float()
    spread = torch.linspace(-60, 60, k, device="cuda")
    x[0] *= torch.exp2(spread)
    x[1] *= 2.0 ** -130
    x[2] *= 2.0 ** 100
    x[3] = 0
    x[4, 1:] = 0
    x[5, 7] = 1e30   # one element far above the others ...
    x[6] *= torch.exp2(-spread[torch.randperm(k, device="cuda")])
    x[7] *= 2.0 ** -30
    x = x.to(torch.bfloat16)
    check_rows = [check(w, x[r: r + 1]) for r in range(9)]
    assert torch.equal(torch.cat(check_rows), check(w, x))
    # ... that meets codes of zero everywhere: what is left is the sum of the others
    if fmt == "nvfp4":
        w.data[:, 3] &= 0xF0
        w.values[:, 7] = 0
        x = x.clone()
        x[5, 8:512] *= 2.0 ** -20
        check(w, x[5:6])


@pytest.mark.parametrize("fmt", ["nvfp4", "nf4"])
def test_nan_and_infinity_stay_in_their_row(fmt):
    w = Weight(fmt, 128, 512, 6)
    x = draw_x(4, 512, 3)
    clean = check(w, x)
    x[1, 100], x[2, 17] = float("nan"), float("inf")
    y = sfq.linear_matvec(w.desc, x)
    assert torch.equal(y[[0, 3]], clean[[0, 3]])
    assert bool(y[1].isnan().all())
    want = x[2:3].double() @ w.values.T  # inf times a weight of zero is NaN
    assert torch.equal(y[2:3].isnan(), want.isnan()) and torch.equal(y[2:3][~want.isnan()].double(), want[~want.isnan()])


def test_a_nan_scale_makes_its_columns_nan():
    w = Weight("nvfp4", 256, 128, 7)
    x = draw_x(2, 128, 4)
    clean = check(w, x)
    w.scale[512 + 5 * 16 + 2 * 4 + 1] = 0x7F  # row 5 + 64, elements 80 .. 95
    y = sfq.linear_matvec(w.desc, x)
    assert bool(y[:, 69].isnan().all())
    y[:, 69] = clean[:, 69]
    assert torch.equal(y, clean)


def test_repeats_streams_and_graphs():
    """The same bits on every call, whatever runs beside it, and in a captured graph whose input changes."""
    w, v = Weight("nvfp4", 1152, 2048, 8), Weight("nf4", 1000, 2048, 9)
    x = draw_x(3, 2048, 5)
    a, b = check(w, x), check(v, x)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append((sfq.linear_matvec(w.desc, x), sfq.linear_matvec(v.desc, x)))
    torch.cuda.synchronize()
    assert all(torch.equal(p, a) and torch.equal(q, b) for p, q in outs)
    y = torch.empty_like(a)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sfq.linear_matvec(w.desc, x, y)
    for seed in (6, 7):
        x.copy_(draw_x(3, 2048, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, check(w, x))


def test_a_view_of_a_fused_weight():
    """The middle third of a fused projection by sfq_weight_row_block."""
    w = Weight("nvfp4", 768, 256, 10, torch.float32)
    part = sfq.QuantWeight()
    sfq.check(sfq.lib.sfq_weight_row_block(C.byref(w.desc), 3, 1, C.byref(part)))
    x = draw_x(2, 256, 8)
    assert torch.equal(sfq.linear_matvec(part, x), check(w, x)[:, 256:512])


def test_reads_behind_a_producer_and_writes_for_a_consumer():
    """In one stream with no wait between: the input is written just before, the output read just behind, many times."""
    w = Weight("nvfp4", 2048, 2048, 11)
    x = torch.empty((2, 2048), dtype=torch.bfloat16, device="cuda")
    y = torch.empty((2, 2048), dtype=torch.bfloat16, device="cuda")
    sources = [draw_x(2, 2048, s) for s in range(4)]
    wants = [check(w, s) for s in sources]
    got = []
    for i in range(40):
        x.copy_(sources[i % 4])
        sfq.linear_matvec(w.desc, x, y)
        got.append(y.clone())
    assert all(torch.equal(g, wants[i % 4]) for i, g in enumerate(got))


# Teams that take several groups of weight rows: the ring of copies that runs on into the next group, the next group's absmax, sums whose
# place is used again, and with SwiGLU and odd remainders the rows past the end in the last group. On 148 SMs the first NVFP4 shape has
# three rounds in every form, the others two.
MANY = [("nvfp4", 40064, 192), ("nvfp4", 20096, 1088), ("nf4", 30018, 192), ("nf4", 20034, 1088), ("nf4", 9502, 2048)]


@pytest.mark.parametrize("fmt,n,k", MANY)
@pytest.mark.parametrize("rows", [1, 3, 4, 5, 8, 12, 16])
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
def test_teams_with_several_groups_of_rows(fmt, n, k, rows, act):
    bias = {"none": None, "gelu": torch.float32, "swiglu": torch.bfloat16}[act]
    check(Weight(fmt, n, k, n + rows, bias), draw_x(rows, k, rows) * (0.05 if fmt == "nvfp4" else 0.5), act)


def spanning(x, where):
    """x with elements over 100 binades in a part of K (fractions of it), and none but zeros in another."""
    x, k = x.float(), x.shape[1]
    a, b, c, d = (int(f * k) for f in where)
    x[:, a:b] *= torch.exp2(torch.linspace(-60, 40, b - a, device="cuda"))
    x[:, c:d] = 0
    return x.to(torch.bfloat16)


PARTS = [(0.0, 0.2, 0.5, 0.75), (0.8, 1.0, 0.0, 0.5), (0.3, 0.45, 0.0, 0.0), (0.0, 1.0, 0.0, 0.0)]


@pytest.mark.parametrize("fmt,n,k", [("nvfp4", 40064, 192), ("nf4", 20034, 1088)])
@pytest.mark.parametrize("rows", [1, 5, 12])
@pytest.mark.parametrize("where", PARTS)
def test_wide_x_through_several_groups_of_rows(fmt, n, k, rows, where):
    """Every group is walked once for each band of 32 binades."""
    check(Weight(fmt, n, k, n + rows), spanning(draw_x(rows, k, rows), where), "none")


# K divided over clusters, of two CTAs and (514 rows) of four; all but 514 and 2432 rows with several groups for a team.
CLUSTERS = [("nvfp4", 10240, 13824, 16), ("nvfp4", 2432, 13824, 13), ("nf4", 10274, 5120, 16), ("nf4", 514, 13824, 16), ("nf4", 5122, 13824, 5)]


@pytest.mark.parametrize("fmt,n,k,rows", CLUSTERS)
@pytest.mark.parametrize("act", ["none", "gelu", "swiglu"])
@pytest.mark.parametrize("bias", [torch.float32, torch.bfloat16])
def test_activations_and_bias_over_clusters(fmt, n, k, rows, act, bias):
    check(Weight(fmt, n, k, n, bias), draw_x(rows, k, rows) * (0.01 if fmt == "nvfp4" else 0.1), act)


@pytest.mark.parametrize("fmt,n,k,rows", CLUSTERS)
@pytest.mark.parametrize("where", PARTS)
def test_wide_x_over_clusters(fmt, n, k, rows, where):
    """The CTAs of a cluster find different exponents and different numbers of bands in their parts of K, some of them none."""
    x = spanning(draw_x(rows, k, rows), where)
    x[rows // 2] = draw_x(1, k, 99)  # and a row within one band beside them
    check(Weight(fmt, n, k, n), x)


@pytest.mark.parametrize("fmt,n,k,rows", [("nvfp4", 128, 200000, 2), ("nf4", 66, 200000, 2), ("nf4", 2402, 123008, 1)])
def test_the_largest_inputs(fmt, n, k, rows):
    """Rows of x that only the shared memory of four CTAs holds."""
    w = Weight(fmt, n, k, n)
    check(w, draw_x(rows, k, rows))
    check(w, spanning(draw_x(rows, k, rows), PARTS[1]))
    with pytest.raises(sfq.SfqError, match="too large"):
        big = sfq.QuantWeight.from_buffer_copy(w.desc)
        big.in_features = 1 << 20
        sfq.linear_matvec(big, torch.zeros((1, 1 << 20), dtype=torch.bfloat16, device="cuda"))


@pytest.mark.parametrize("fmt", ["nvfp4", "nf4"])
@pytest.mark.parametrize("rows", [1, 4, 8, 16])
@pytest.mark.parametrize("gate,up", [(1.0, 1.0), (0.2, 0.1), (6.0, 6.0)])
def test_the_output_of_swiglu_as_input(fmt, rows, gate, up):
    """What a down-projection is given, over many binades: silu(g) u in bf16. With deviations of 6 most rows need a second band."""
    k = 6912
    g = torch.Generator("cuda").manual_seed(rows)
    a, b = (s * torch.randn((rows, k), device="cuda", generator=g) for s in (gate, up))
    check(Weight(fmt, 1280, k, rows), (a * torch.sigmoid(a) * b).to(torch.bfloat16))


@pytest.mark.parametrize("rows", [1, 3, 8, 16])
@pytest.mark.parametrize("size", [-100, -30, -16, 17, 60])
def test_nf4_maps_of_every_size(rows, size):
    """A map 2^size as large over an absmax 2^-size as large is the same weight, and gives the same bits."""
    w = Weight("nf4", 130, 640, 12, torch.float32)
    x = draw_x(rows, 640, rows)
    want = check(w, x, "gelu")
    w.map *= 2.0 ** size
    w.nested_absmax *= 2.0 ** -size
    w.desc.nf4_nested_offset *= 2.0 ** -size
    assert torch.equal(check(w, x, "gelu"), want)
