"""Refusals of the decoding-step entry points: each is made on the host before anything is launched, so no GPU is needed."""
import ctypes as C

import pytest
import torch

import slopfab_b200 as sfq
from slopfab_b200.kv_cache import KvCache, Rotary, Sequences

A = 1 << 20  # stands for an aligned device address; nothing here is dereferenced


def _weight(**over):
    f = dict(format=sfq.NVFP4, data=A, block_scale=A, out_features=256, in_features=128)
    f.update(over)
    return sfq.new_weight(**f)


def _nf4(**over):
    f = dict(format=sfq.NF4, data=A, nf4_absmax=A, nf4_quant_map=A, nf4_nested_quant_map=A, nf4_nested_absmax=A, out_features=34, in_features=192)
    f.update(over)
    return sfq.new_weight(**f)


def _matvec(w, x=A, rows=2, act=0, y=2 * A):
    return sfq.lib.sfq_linear_matvec(C.byref(w) if w is not None else None, x, rows, act, y, None)


@pytest.mark.parametrize("w,text", [
    (lambda: _weight(format=sfq.W4A8), b"NVFP4 and NF4"), (lambda: _weight(format=sfq.BF16), b"NVFP4 and NF4"),
    (lambda: _weight(pre_quant_scale=A), b"pre-scale"), (lambda: _weight(convrot=1), b"ConvRot"),
    (lambda: _weight(out_features=200), b"% 128"), (lambda: _weight(in_features=96), b"% 64"), (lambda: _weight(out_features=0), b"positive"),
    (lambda: _weight(data=None), b"null"), (lambda: _weight(block_scale=None), b"block_scale"), (lambda: _weight(data=A + 8), b"aligned"),
    (lambda: _weight(block_scale=A + 2), b"aligned"), (lambda: _weight(bias=A, bias_format=sfq.F16), b"bias"),
    (lambda: _nf4(in_features=96), b"% 64"), (lambda: _nf4(nf4_block_size=48), b"powers of two"), (lambda: _nf4(nf4_block_size=32), b"powers of two"),
    (lambda: _nf4(nf4_nested_block_size=100), b"powers of two"), (lambda: _nf4(nf4_absmax=None), b"double-quant"),
])
def test_matvec_refuses_weights(w, text):
    assert _matvec(w()) == sfq.ERR_INVALID_ARGUMENT
    assert text in sfq.lib.sfq_last_error()


def test_matvec_refuses_calls():
    assert _matvec(None) == sfq.ERR_INVALID_ARGUMENT
    assert _matvec(_weight(), act=7) == sfq.ERR_INVALID_ARGUMENT
    assert _matvec(_nf4(out_features=33), act=sfq.ACT_SWIGLU) == sfq.ERR_INVALID_ARGUMENT and b"even" in sfq.lib.sfq_last_error()
    for x, y in ((None, A), (A, None), (A + 2, 2 * A), (A, 2 * A + 1), (A, A), (A, A + 2 * 2 * 128 - 2), (A + 2 * 2 * 256 - 16, A)):
        assert _matvec(_weight(), x=x, y=y) == sfq.ERR_INVALID_ARGUMENT, (x, y)
    assert _matvec(_weight(), rows=0, x=None, y=None) == sfq.OK and _matvec(_weight(), rows=-3) == sfq.OK  # no-ops


def _cache(**over):
    f = dict(d_k=A, d_v=A, d_k_scale=A, d_v_scale=A, num_pages=7, page_size=64, kv_heads=2, head_dim=128, d_page_table=A, d_seq_len=A, d_row_start=A,
             batch=3, max_pages=4, max_new=1, max_len=200)
    f.update(over)
    return sfq.KvCacheDesc(**f)


BAD_CACHES = [dict(head_dim=64), dict(page_size=8), dict(page_size=48), dict(page_size=512), dict(num_pages=0), dict(kv_heads=0), dict(batch=0),
              dict(max_pages=0), dict(max_new=0), dict(max_len=0), dict(d_k=None), dict(d_v=None), dict(d_k_scale=None), dict(d_v_scale=None),
              dict(d_page_table=None), dict(d_seq_len=None), dict(d_row_start=None), dict(d_k=A + 8), dict(d_v=A + 8), dict(kv_heads=40000)]


def _append(c, rotary=None, q=A, ld_q=512, q_out=A, ld_q_out=512, heads=4, k=2 * A, v=3 * A, ld_kv=256, rows=3):
    return sfq.lib.sfq_kv_cache_append(C.byref(c) if c is not None else None, C.byref(rotary) if rotary is not None else None, q, ld_q, q_out, ld_q_out,
                                       heads, k, v, ld_kv, rows, None)


def _attend(c, q=A, ld_q=512, out=2 * A, ld_out=512, heads=4, rows=3, ws=A, ws_bytes=1 << 40):
    return sfq.lib.sfq_kv_cache_attention(C.byref(c) if c is not None else None, q, ld_q, out, ld_out, heads, rows, 0.0, ws, ws_bytes, None)


@pytest.mark.parametrize("over", BAD_CACHES)
def test_bad_caches_are_refused(over):
    assert _append(_cache(**over)) == sfq.ERR_INVALID_ARGUMENT
    assert _attend(_cache(**over)) == sfq.ERR_INVALID_ARGUMENT
    n = C.c_size_t()
    assert sfq.lib.sfq_kv_cache_attention_workspace_bytes(C.byref(_cache(**over)), 4, 3, C.byref(n)) == sfq.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("over", [dict(q=None), dict(q_out=None), dict(k=None), dict(v=None), dict(heads=-1), dict(ld_q=504), dict(ld_q=516),
                                  dict(ld_q_out=504), dict(ld_kv=248), dict(ld_kv=260), dict(q=A + 8), dict(q_out=A + 8), dict(k=A + 8), dict(v=A + 2)])
def test_append_refuses_operands(over):
    assert _append(_cache(), **over) == sfq.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("over", [dict(d_sin=None), dict(d_cos=None), dict(rotary_dim=0), dict(rotary_dim=24), dict(rotary_dim=144), dict(table_rows=0),
                                  dict(d_cos=A + 4), dict(d_q_norm=A + 2), dict(d_k_norm=A + 2)])
def test_append_refuses_rotations(over):
    f = dict(d_cos=A, d_sin=A, table_rows=5, rotary_dim=96, d_q_norm=A, d_k_norm=A, eps=1e-6)
    f.update(over)
    assert _append(_cache(), rotary=sfq.RotaryDesc(**f)) == sfq.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("over", [dict(rows=1 << 29), dict(q=None), dict(out=None), dict(heads=0), dict(heads=3), dict(ld_q=504),
                                  dict(ld_out=516), dict(out=A), dict(q=A + 8), dict(out=2 * A + 2)])
def test_attention_refuses_operands(over):
    assert _attend(_cache(), **over) == sfq.ERR_INVALID_ARGUMENT


def test_buffers_off_their_alignment_are_refused():
    for name in ("d_k_scale", "d_v_scale", "d_page_table", "d_seq_len", "d_row_start"):
        c = _cache(**{name: A + 2})
        assert _append(c) == sfq.ERR_INVALID_ARGUMENT and _attend(c) == sfq.ERR_INVALID_ARGUMENT and b"4-byte" in sfq.lib.sfq_last_error()
    assert _append(_cache(), sfq.RotaryDesc(d_position=A + 2)) == sfq.ERR_INVALID_ARGUMENT and b"4-byte" in sfq.lib.sfq_last_error()
    for name in ("nf4_quant_map", "nf4_nested_quant_map", "nf4_nested_absmax"):
        assert _matvec(_nf4(**{name: A + 2})) == sfq.ERR_INVALID_ARGUMENT and b"4-byte" in sfq.lib.sfq_last_error()
    for at, fmt in ((A + 2, sfq.F32), (A + 1, sfq.BF16)):
        assert _matvec(_weight(bias=at, bias_format=fmt)) == sfq.ERR_INVALID_ARGUMENT and b"bias" in sfq.lib.sfq_last_error()


def test_overlapping_operands_are_refused():
    # a fused projection: q, k and v in columns of rows of 1024
    fused = dict(q=A, ld_q=1024, k=A + 512 * 2, v=A + 768 * 2, ld_kv=1024, ld_q_out=1024)
    for q_out in (A + 16, A - 16, A + 512 * 2 - 16, A + 768 * 2, A + 1024 * 2, A + 1024 * 2 + 512 * 2):
        assert _append(_cache(), **{**fused, "q_out": q_out}) == sfq.ERR_INVALID_ARGUMENT and b"apart" in sfq.lib.sfq_last_error()
    assert _append(_cache(), **{**fused, "q_out": A, "ld_q_out": 512}) == sfq.ERR_INVALID_ARGUMENT and b"apart" in sfq.lib.sfq_last_error()
    # what does not overlap goes on to the next check
    bad = sfq.RotaryDesc(d_cos=A, d_sin=A, table_rows=5, rotary_dim=24)
    for q_out, ld in ((A, 1024), (A - 3 * 1024 * 2, 1024), (A + 3 * 1024 * 2, 1024), (2 * A, 512)):
        assert _append(_cache(), bad, **{**fused, "q_out": q_out, "ld_q_out": ld}) == sfq.ERR_INVALID_ARGUMENT and b"rotary_dim" in sfq.lib.sfq_last_error()
    for out, ld in ((A + 16, 1024), (A - 16, 1024), (A, 1024), (A, 512), (A + 1024 * 2, 1024)):
        assert _attend(_cache(), ld_q=1024, out=out, ld_out=ld) == sfq.ERR_INVALID_ARGUMENT and b"overlap" in sfq.lib.sfq_last_error()
    long = _cache(max_len=100000)
    assert _attend(long, ld_q=1024, out=A + 512 * 2, ld_out=1024, ws=None) == sfq.ERR_INVALID_ARGUMENT and b"workspace" in sfq.lib.sfq_last_error()


def test_scales_that_are_not_finite_are_refused():
    for scale in (float("nan"), float("inf"), -float("inf")):
        assert sfq.lib.sfq_kv_cache_attention(C.byref(_cache()), A, 512, 2 * A, 512, 4, 3, scale, A, 1 << 40, None) == sfq.ERR_INVALID_ARGUMENT
        assert b"scale" in sfq.lib.sfq_last_error()


def test_descriptors_follow_their_tensors():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    cache = KvCache.empty(5, 2, 64, device="cpu")
    seqs = Sequences(i32(3, 4), i32(3), i32(4), 1, 100)
    d = cache._desc(seqs)
    assert C.sizeof(d) == C.sizeof(sfq.KvCacheDesc)
    want = dict(d_k=cache.k.data_ptr(), d_v=cache.v.data_ptr(), d_k_scale=cache.k_scale.data_ptr(), d_v_scale=cache.v_scale.data_ptr(), num_pages=5, page_size=64,
                kv_heads=2, head_dim=128, d_page_table=seqs.page_table.data_ptr(), d_seq_len=seqs.seq_len.data_ptr(), d_row_start=seqs.row_start.data_ptr(),
                batch=3, max_pages=4, max_new=1, max_len=100)
    assert {k: getattr(d, k) for k in want} == want
    seqs.page_table.resize_(3, 2)  # the same memory, another shape
    assert cache._desc(seqs).max_pages == 2
    seqs.page_table.resize_(2, 2)
    with pytest.raises(ValueError):
        cache._desc(seqs)
    with pytest.raises(AttributeError):  # a rotation's tensors are checked once
        Rotary(position=i32(3)).position = i32(4)
    with pytest.raises(ValueError, match="cache's device"):
        rotary = Rotary(position=i32(3))
        object.__setattr__(rotary, "device", 0)
        cache.append(seqs, torch.zeros((3, 8 * 128), dtype=torch.bfloat16), 4, rotary=rotary)


def test_attention_refuses_workspaces():
    long = _cache(max_len=100000)  # divided: parts are kept
    n = C.c_size_t()
    sfq.check(sfq.lib.sfq_kv_cache_attention_workspace_bytes(C.byref(long), 4, 3, C.byref(n)))
    assert n.value > 0
    for over in (dict(ws=None), dict(ws=A + 8), dict(ws_bytes=0), dict(ws_bytes=n.value - 1)):
        assert _attend(long, **over) == sfq.ERR_INVALID_ARGUMENT and b"workspace" in sfq.lib.sfq_last_error()
    sfq.check(sfq.lib.sfq_kv_cache_attention_workspace_bytes(C.byref(_cache()), 4, 3, C.byref(n)))
    assert n.value == 0


def test_no_rows_is_a_no_op_and_null_descriptors_are_refused():
    assert _append(_cache(), rows=0, q=None, k=None) == sfq.OK and _attend(_cache(), rows=0, q=None) == sfq.OK
    assert _append(None) == sfq.ERR_INVALID_ARGUMENT and _attend(None) == sfq.ERR_INVALID_ARGUMENT
    assert sfq.lib.sfq_kv_cache_attention_workspace_bytes(C.byref(_cache()), 4, 3, None) == sfq.ERR_INVALID_ARGUMENT


def test_python_faces_refuse_what_does_not_fit():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    cache = KvCache.empty(5, 2, 64, device="cpu")
    seqs = Sequences(i32(3, 4), i32(3), i32(4), 1, 100)
    qkv = torch.zeros((3, 8 * 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA device"):  # there is no CPU path
        cache.append(seqs, qkv, 4)
    with pytest.raises(ValueError, match="CUDA device"):
        cache.attention(seqs, qkv[:, :512], 4)
    with pytest.raises(ValueError, match="CUDA device"):
        sfq.linear_matvec(_weight(), torch.zeros((1, 128), dtype=torch.bfloat16))
    for bad in (qkv.float(), qkv[:, :-128], qkv[0], qkv.t().contiguous().t()):
        with pytest.raises(ValueError):
            cache.append(seqs, bad, 4)
    with pytest.raises(ValueError):
        cache.append(seqs, qkv, 4, q_out=torch.zeros((2, 512), dtype=torch.bfloat16))
    for bad in (torch.zeros((1, 64), dtype=torch.bfloat16), torch.zeros((1, 128)), torch.zeros(128, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            sfq.linear_matvec(_weight(), bad)
    with pytest.raises(ValueError):
        sfq.linear_matvec(_weight(), torch.zeros((1, 128), dtype=torch.bfloat16), torch.zeros((1, 128), dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        KvCache(cache.k, cache.k, cache.k_scale, cache.v_scale)
    with pytest.raises(ValueError):
        KvCache(cache.k, cache.v, cache.k_scale[:4], cache.v_scale)
    with pytest.raises(ValueError):
        Rotary(cos=torch.zeros((4, 48)))
    with pytest.raises(ValueError):
        Rotary(q_norm=torch.ones(64, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        Rotary(torch.zeros((4, 48)), torch.zeros((4, 48)), position=torch.zeros(3))


def _host_cache():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    return KvCache.empty(5, 2, 64, device="cpu"), Sequences(i32(3, 4), i32(3), i32(4), 1, 100)


def test_rows_that_overlap_are_refused():
    """A row that is repeated by a stride of 0, and windows that slide over a buffer: their pitch is less than a row."""
    cache, seqs = _host_cache()
    wide = torch.zeros(3 * 8 * 128, dtype=torch.bfloat16)
    qkv, q, out = wide.view(3, -1), wide.view(3, -1)[:, :512], torch.zeros((3, 512), dtype=torch.bfloat16)
    for n, call in ((8 * 128, lambda t: cache.append(seqs, t, 4)), (512, lambda t: cache.append(seqs, qkv, 4, q_out=t)),
                    (512, lambda t: cache.attention(seqs, t, 4)), (512, lambda t: cache.attention(seqs, q, 4, out=t))):
        for bad in (wide[:n].expand(3, n), wide.as_strided((3, n), (n // 2, 1)), wide.as_strided((3, n), (n - 8, 1))):
            with pytest.raises(ValueError, match="overlap"):
                call(bad)
    for good in (q, out):  # these go on to the next check
        with pytest.raises(ValueError, match="CUDA device"):
            cache.attention(seqs, good, 4)


def test_a_single_row_has_no_pitch():
    """The stride of one row says nothing: it may be odd, less than the row, or more than 32 bits hold."""
    cache, _ = _host_cache()
    wide = torch.zeros(2 * 2058, dtype=torch.bfloat16).view(2, 2058)
    for row in (wide[:1, :512], wide[0, :512].expand(1, 512), wide[0].as_strided((1, 512), (1, 1)), wide[0].as_strided((1, 512), (1 << 40, 1))):
        assert cache._pitch("q", row, 1, 512) == 512, row.stride()
    assert cache._pitch("q", wide[:, :512], 2, 512) == 2058


def test_pitches_of_more_than_32_bits_are_refused():
    """ctypes would pass on their low 32 bits, 512 here."""
    cache, _ = _host_cache()
    for stride in ((1 << 32) + 512, 1 << 31):
        with pytest.raises(ValueError, match="32 bits"):
            cache._pitch("q", torch.empty((2, stride), dtype=torch.bfloat16, device="meta")[:, :512], 2, 512)


def test_the_pool_follows_its_tensors():
    """A pool whose tensors are replaced, grown or given other memory: a call never goes to the memory of before, and what no longer
    fits together is refused."""
    cache, seqs = _host_cache()
    larger = KvCache.empty(9, 2, 64, device="cpu")
    tensors = lambda c: (c.k, c.v, c.k_scale, c.v_scale)  # noqa: E731
    addresses = lambda d: (d.d_k, d.d_v, d.d_k_scale, d.d_v_scale)  # noqa: E731
    cache.k = larger.k
    with pytest.raises(ValueError):  # the other three have five pages
        cache._desc(seqs)
    with pytest.raises(ValueError):
        cache.append(seqs, torch.zeros((3, 8 * 128), dtype=torch.bfloat16), 4)
    cache.v, cache.k_scale, cache.v_scale = larger.v, larger.k_scale, larger.v_scale
    d = cache._desc(seqs)
    assert addresses(d) == tuple(t.data_ptr() for t in tensors(larger)) and d.num_pages == 9
    cache.k_scale = torch.zeros((9, 2), dtype=torch.float64)
    with pytest.raises(ValueError):
        cache._desc(seqs)
    cache.k_scale = larger.k_scale
    cache.k_scale *= 2  # the same tensor
    for t in tensors(cache):  # the same tensors, other memory
        t.set_(t.clone())
        d = cache._desc(seqs)
        assert addresses(d) == tuple(u.data_ptr() for u in tensors(cache)) and d.num_pages == 9
    cache.k.resize_(11, 2, 64, 128)
    with pytest.raises(ValueError):
        cache._desc(seqs)
    cache.k.resize_(3, 2, 64, 128)  # the same memory, fewer pages than the others
    with pytest.raises(ValueError):
        cache._desc(seqs)
    few = KvCache.empty(4, 3, 16, device="cpu")
    cache.k, cache.v, cache.k_scale, cache.v_scale = tensors(few)
    assert (cache._desc(seqs).kv_heads, cache._desc(seqs).page_size) == (3, 16) and cache.kv_heads == 3
    with pytest.raises(ValueError, match="CUDA device"):  # rows of the heads that there are now
        cache.append(seqs, torch.zeros((3, 9 * 128), dtype=torch.bfloat16), 3)


def test_a_rotation_follows_its_tensors():
    """Tables, positions and norm weights that are given other memory, as a module's are when its data is replaced."""
    bf16 = lambda *s: torch.zeros(s, dtype=torch.bfloat16)  # noqa: E731
    r = Rotary(torch.zeros((40, 48)), torch.zeros((40, 48)), torch.zeros(3, dtype=torch.int32), bf16(128), bf16(128))
    names = ("cos", "sin", "position", "q_norm", "k_norm")
    assert r._desc_now() is r.desc
    for name in names:
        t = getattr(r, name)
        t.data = t.clone()
        d = r._desc_now()
        assert [getattr(d, "d_" + n) for n in names] == [getattr(r, n).data_ptr() for n in names]
    r.sin.resize_(20, 48)
    r.cos.resize_(20, 48)  # the same memory, fewer rows
    assert r._desc_now().table_rows == 20
    r.cos.resize_(60, 48)
    cache, seqs = _host_cache()
    with pytest.raises(ValueError, match="cos and sin"):
        cache.append(seqs, bf16(3, 8 * 128), 4, rotary=r)


def test_pools_that_share_memory_are_refused():
    """With pages of 128 tokens K and V have the same shape, and one tensor could be given for both; scales always have."""
    cache = KvCache.empty(5, 2, 128, device="cpu")
    both = torch.zeros((6, 2, 128, 128), dtype=torch.uint8)
    scales = torch.zeros(19)
    for bad in ((cache.k, cache.k, cache.k_scale, cache.v_scale), (cache.k, cache.v, cache.k_scale, cache.k_scale), (both[:5], both[1:], cache.k_scale, cache.v_scale),
                (cache.k, cache.v, scales[9:].view(5, 2), scales[:10].view(5, 2))):
        with pytest.raises(ValueError, match="apart"):
            KvCache(*bad)
    scales = torch.zeros(20)
    KvCache(cache.k, cache.v, scales[10:].view(5, 2), scales[:10].view(5, 2))  # side by side


def test_a_single_row_may_be_turned_in_place_with_any_pitch():
    bad = sfq.RotaryDesc(d_cos=A, d_sin=A, table_rows=5, rotary_dim=24)  # the check behind that of the operands
    fused = dict(q=A, ld_q=1024, q_out=A, ld_q_out=512, k=A + 512 * 2, v=A + 768 * 2, ld_kv=1024)
    assert _append(_cache(), bad, **fused, rows=1) == sfq.ERR_INVALID_ARGUMENT and b"rotary_dim" in sfq.lib.sfq_last_error()
    assert _append(_cache(), bad, **fused, rows=2) == sfq.ERR_INVALID_ARGUMENT and b"apart" in sfq.lib.sfq_last_error()
    assert _append(_cache(), bad, **{**fused, "q_out": A + 16}, rows=1) == sfq.ERR_INVALID_ARGUMENT and b"apart" in sfq.lib.sfq_last_error()
