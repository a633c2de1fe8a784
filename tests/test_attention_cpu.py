"""CPU: what the attention operators refuse (no kernel is launched), and the record's definition."""

import ctypes

import pytest
import torch

from rvq_b200 import _native, attention
from rvq_b200.attention import (Cache4, Cache4AttentionOp, Cache4EvictOp, Cache4ReadOp, Cache4WriteOp, PromptAttentionOp)
from rvq_b200.step import RvqVec
from tests import _attention as ref

BF = torch.bfloat16


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


def ints(*v, dtype=torch.int64):
    return torch.tensor(v, dtype=dtype)


def test_struct_layouts():
    assert ctypes.sizeof(attention.RvqCache4) == 8 + 4 * 4
    assert ctypes.sizeof(attention.RvqPromptAttnArgs) == 7 * 8 + 2 * 8 + 8 * 8 + 8 * 4
    assert ctypes.sizeof(attention.RvqCache4RowsArgs) == 24 + 4 * 8 + 8 + 4 * 8 + 2 * 4
    assert ctypes.sizeof(attention.RvqCache4AttnArgs) == 3 * 24 + 5 * 8 + 24 + 3 * 8 + 4 * 4
    assert ctypes.sizeof(attention.RvqCache4EvictArgs) == 2 * 24 + 5 * 8 + 2 * 4
    assert attention.record_bytes(128) == 160 and attention.record_bytes(64) == 80
    with pytest.raises(NotImplementedError):
        attention.record_bytes(96)


def test_record_definition():
    """The test oracle's records unpack to its held values, and those are half a step from the input."""
    g = torch.Generator().manual_seed(0)
    for hd in (64, 128):
        k, v = torch.randn(6, 2, hd, generator=g).to(BF), torch.randn(6, 2, hd, generator=g).half()
        rec = ref.records(k, v)
        assert rec.shape == (6, 2, hd * 5 // 4)
        for x, part in zip((k, v), ref.unpack(rec, hd)):
            assert torch.equal(ref.values(*part), ref.held(x))


def prompt(q=None, k=None, v=None, out=None, **kw):
    q = z(6, 4, 64) if q is None else q
    k = z(6, 2, 64) if k is None else k
    return PromptAttentionOp(q, k, z(6, 2, 64) if v is None else v, z(6, 4, 64) if out is None else out, scaling=1.0, **kw)


@pytest.mark.parametrize("error,make", [
    (ValueError, lambda: prompt(q=z(6, 256))),
    (NotImplementedError, lambda: prompt(q=z(6, 4, 64, dtype=torch.float32))),
    (ValueError, lambda: prompt(k=z(6, 2, 64, dtype=torch.float16))),
    (ValueError, lambda: prompt(out=z(6, 4, 64, dtype=torch.float16))),
    (ValueError, lambda: prompt(out=z(5, 4, 64))),
    (ValueError, lambda: prompt(k=z(6, 2, 128))),
    (ValueError, lambda: prompt(v=z(5, 2, 64))),
    (ValueError, lambda: prompt(k=z(6, 3, 64), v=z(6, 3, 64))),
    (NotImplementedError, lambda: prompt(q=z(6, 4, 136), k=z(6, 2, 136), v=z(6, 2, 136), out=z(6, 4, 136))),
    (NotImplementedError, lambda: prompt(q=z(6, 130, 64), out=z(6, 130, 64))),
    (ValueError, lambda: prompt(q=z(6, 4, 12), k=z(6, 2, 12), v=z(6, 2, 12), out=z(6, 4, 12))),
    (ValueError, lambda: prompt(q=z(6, 4, 128)[:, :, ::2])),
    (ValueError, lambda: prompt(q=z(6 * 4 * 64 + 8)[1:1 + 6 * 256].view(6, 4, 64))),
    (ValueError, lambda: prompt(k=z(6, 1, 64).expand(6, 2, 64))),
    (ValueError, lambda: prompt(out=z(1, 4, 64).expand(6, 4, 64))),
    (ValueError, lambda: prompt(cu_k=ints(0, 6, dtype=torch.int32))),
    (ValueError, lambda: prompt(cu_q=ints(0, 6))),
    (ValueError, lambda: prompt(cu_q=ints(0, dtype=torch.int32))),
    (ValueError, lambda: prompt(cu_q=ints(0, 3, 6, dtype=torch.int32), cu_k=ints(0, 6, dtype=torch.int32))),
    (ValueError, lambda: prompt(lse=z(6, 4, dtype=torch.float32))),
    (ValueError, lambda: prompt(lse=z(4, 6))),
    (ValueError, lambda: prompt()),                                            # not on a GPU
])
def test_prompt_refuses(error, make):
    with pytest.raises(error):
        make()


def test_prompt_refuses_overlap():
    wide = z(6, 9, 64)
    with pytest.raises(ValueError, match="overlap"):
        prompt(q=wide[:, :4], out=wide[:, 3:7])
    with pytest.raises(ValueError, match="CUDA"):                               # columns apart: only the device is wrong
        prompt(q=wide[:, :4], out=wide[:, 4:8])
    with pytest.raises(ValueError, match="overlap"):
        q = z(6, 4, 64)
        prompt(q=q, out=q)


def test_refuses_outputs_that_overlap_themselves():
    buf = z(4096)
    for st in ((64, 8, 1), (8, 64, 1), (256, 56, 1), (200, 64, 1)):
        with pytest.raises(ValueError, match="overlap"):
            prompt(out=torch.as_strided(buf, (6, 4, 64), st))
        with pytest.raises(ValueError, match="overlap"):
            Cache4ReadOp(Cache4(1, 4, 8, 64), torch.as_strided(buf, (6, 4, 64), st), z(6, 4, 64))
    for st in ((256, 64, 1), (64, 384, 1), (264, 64, 1)):
        with pytest.raises(ValueError, match="CUDA"):
            prompt(out=torch.as_strided(buf, (6, 4, 64), st))


def test_interleaved_views():
    """Against the elements themselves, over many pairs of views of one buffer."""
    buf = torch.arange(4000)
    g = torch.Generator().manual_seed(1)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    said = [0, 0]
    for _ in range(3000):
        hd, s1 = 8, 8 * r(1, 4)
        s0 = s1 * r(1, 5) if r(0, 1) else 8 * r(1, 20)
        st = (s0, s1, 1) if r(0, 1) else (s1, s0, 1)
        views = []
        for _ in range(2):
            n = (r(1, 5), r(1, 5), hd)
            at = 4 * r(0, 60)
            views.append(torch.as_strided(buf, n, st, at))
        share = bool(set(views[0].flatten().tolist()) & set(views[1].flatten().tolist()))
        if attention._interleaved(*views):
            assert not share
            said[0] += 1
        else:
            said[1] += not share
    assert said[0] > 300                                                        # it does find views that are apart


def test_tensors_in_the_gaps_of_views():
    """Against the bytes themselves, over many pairs."""
    buf = torch.zeros(8192, dtype=torch.uint8)
    g = torch.Generator().manual_seed(2)
    r = lambda lo, hi: int(torch.randint(lo, hi + 1, (1,), generator=g))
    said = [0, 0]
    for _ in range(3000):
        n0, n1, hd = r(1, 5), r(1, 5), 8
        s1 = 8 * r(1, 5)
        s0 = s1 * n1 + 8 * r(0, 4)
        n, st = ((n0, n1), (s0, s1)) if r(0, 1) else ((n1, n0), (s1, s0))
        view = torch.as_strided(buf.view(BF), (*n, hd), (*st, 1), 8 * r(0, 30))
        t = buf.view(torch.int32)[r(0, 500):][:r(1, 12)]
        bytes_of = lambda x: {x.storage_offset() * x.element_size() + b
                              for i in torch.cartesian_prod(*(torch.arange(m) for m in x.shape)).view(-1, x.dim())
                              for b in range(int((i * torch.tensor(x.stride())).sum()) * x.element_size(),
                                             int((i * torch.tensor(x.stride())).sum()) * x.element_size() + x.element_size())}
        if said[0] + said[1] >= 600:
            break
        (a0, a1), (b0, b1) = attention._span(view), attention._span(t)
        if a0 >= b1 or b0 >= a1:
            continue
        share = bool(bytes_of(view) & bytes_of(t))
        assert attention._in_gaps(view, t) is not share
        said[share] += 1
    assert min(said) > 30


def test_refuses_to_write_over_other_operands():
    """One buffer for what is written and anything else of the call, of every operator."""
    words = z(4096, dtype=torch.float32)
    as_int = lambda n: words.view(torch.int32)[:n]
    as_long = lambda n: words.view(torch.int64)[:n]
    over = lambda *shape: words.view(BF)[:int(torch.tensor(shape).prod())].view(shape)
    data = words.view(torch.uint8)[:2 * 2 * 8 * 80].view(2, 2, 8, 80)
    stored = Cache4(2, 2, 8, 64, data=data)
    w = words[:32].view(2, 2, 8)
    two = dict(cu=ints(0, 3, 6, dtype=torch.int32))
    for make in (lambda: prompt(out=over(6, 4, 64), cu_q=as_int(3)),
                 lambda: prompt(lse=words[:24].view(4, 6), cu_q=ints(0, 3, 6, dtype=torch.int32), cu_k=as_int(3)),
                 lambda: Cache4WriteOp(stored, z(6, 2, 64), z(6, 2, 64), cu=as_int(3)),
                 lambda: Cache4WriteOp(stored, z(6, 2, 64), z(6, 2, 64), start=as_long(2), **two),
                 lambda: Cache4ReadOp(cache(), over(6, 2, 64), z(6, 2, 64), cu=as_int(3)),
                 lambda: Cache4ReadOp(cache(), z(6, 2, 64), over(6, 2, 64), start=as_long(2), **two),
                 lambda: step(out=over(2, 4, 64), rows=as_long(2)),
                 lambda: step(c=stored, rows=as_long(2)),
                 lambda: step(weights=w, q_norm=over(64), k_norm=z(64)),
                 lambda: step(out=over(2, 4, 64), cos=z(9, 64), sin=z(9, 64), pos=as_long(2)),
                 lambda: step(out=over(2, 4, 64), cos=over(9, 64), sin=z(9, 64), pos=ints(0, 0)),
                 lambda: evict(w=w, kept=as_int(16).view(2, 2, 4)),
                 lambda: evict(c=stored, kept=as_int(16).view(2, 2, 4)),
                 lambda: evict(rows=as_long(2), kept=as_int(16).view(2, 2, 4)),
                 lambda: evict(kept=as_int(16).view(2, 2, 4), new_rows=as_long(2)),
                 lambda: evict(out=cache(max_len=4), out_weights=words[:16].view(2, 2, 4), kept=as_int(16).view(2, 2, 4)),
                 lambda: evict(w=w, new_rows=as_long(2))):
        with pytest.raises(ValueError, match="overlap"):
            make()


def cache(n_seq=2, n_kv=2, max_len=8, hd=64):
    return Cache4(n_seq, n_kv, max_len, hd)


@pytest.mark.parametrize("error,make", [
    (ValueError, lambda: cache(n_seq=0)),
    (ValueError, lambda: cache(max_len=0)),
    (NotImplementedError, lambda: cache(hd=80)),
    (ValueError, lambda: Cache4(1, 2, 8, 64, data=z(1, 2, 8, 79, dtype=torch.uint8))),
    (ValueError, lambda: Cache4(1, 2, 8, 64, data=z(1, 2, 8, 80, dtype=torch.int8))),
    (ValueError, lambda: Cache4(1, 2, 8, 64, data=z(1, 2, 8, 160, dtype=torch.uint8)[..., :80])),
    (ValueError, lambda: Cache4(1, 1, 1, 64, data=z(88, dtype=torch.uint8)[1:81].view(1, 1, 1, 80))),
])
def test_cache_refuses(error, make):
    with pytest.raises(error):
        make()


@pytest.mark.parametrize("op", [Cache4WriteOp, Cache4ReadOp])
@pytest.mark.parametrize("error,args,kw", [
    (ValueError, (z(4, 2, 64), z(4, 2, 64)), {}),                               # two sequences need cu
    (ValueError, (z(4, 3, 64), z(4, 3, 64)), dict(cu=ints(0, 2, 4, dtype=torch.int32))),
    (ValueError, (z(4, 2, 64), z(5, 2, 64)), dict(cu=ints(0, 2, 4, dtype=torch.int32))),
    (ValueError, (z(4, 2, 128), z(4, 2, 128)), dict(cu=ints(0, 2, 4, dtype=torch.int32))),
    (ValueError, (z(4, 2, 64), z(4, 2, 64, dtype=torch.float16)), dict(cu=ints(0, 2, 4, dtype=torch.int32))),
    (NotImplementedError, (z(4, 2, 64, dtype=torch.float32),) * 2, dict(cu=ints(0, 2, 4, dtype=torch.int32))),
    (ValueError, (z(4, 2, 64), z(4, 2, 64)), dict(cu=ints(0, 4, dtype=torch.int32))),
    (ValueError, (z(4, 2, 64), z(4, 2, 64)), dict(cu=ints(0, 2, 4))),
    (ValueError, (z(4, 2, 64), z(4, 2, 64)), dict(cu=ints(0, 2, 4, dtype=torch.int32), start=ints(0))),
    (ValueError, (z(4, 2, 64), z(4, 2, 64)), dict(cu=ints(0, 2, 4, dtype=torch.int32), start=ints(0, 0, dtype=torch.int32))),
    (ValueError, (z(4, 2, 64), z(4, 2, 64)), dict(cu=ints(0, 2, 4, dtype=torch.int32))),   # not on a GPU
])
def test_rows_refuse(op, error, args, kw):
    with pytest.raises(error):
        op(cache(), *args, **kw)


def test_read_refuses_one_output_twice():
    k = z(4, 2, 64)
    with pytest.raises(ValueError, match="overlap"):
        Cache4ReadOp(cache(1), k, k)
    with pytest.raises(ValueError, match="CUDA"):                               # written from the same tensor: allowed
        Cache4WriteOp(cache(1), k, k)


def step(q=None, k=None, v=None, c=None, rows=None, out=None, **kw):
    kw.setdefault("scaling", 1.0)
    q = z(2, 4, 64) if q is None else q
    return Cache4AttentionOp(q, z(2, 2, 64) if k is None else k, z(2, 2, 64) if v is None else v, cache() if c is None else c,
                             ints(1, 2) if rows is None else rows, z(2, 4, 64) if out is None else out, **kw)


@pytest.mark.parametrize("error,make", [
    (ValueError, lambda: step(q=z(2, 3, 64))),
    (ValueError, lambda: step(q=z(2, 256))),
    (ValueError, lambda: step(q=z(3, 4, 64))),
    (NotImplementedError, lambda: step(q=z(2, 130, 64), out=z(2, 130, 64))),
    (NotImplementedError, lambda: step(q=z(2, 4, 64, dtype=torch.float64))),
    (ValueError, lambda: step(q=z(2, 4, 128)[..., :64])),
    (ValueError, lambda: step(k=z(2, 2, 64, dtype=torch.float16))),
    (ValueError, lambda: step(q=z(2, 4, 64, dtype=torch.float16))),
    (ValueError, lambda: step(v=z(2, 1, 64))),
    (ValueError, lambda: step(q=z(3, 2, 4, 64, dtype=torch.float32), n_heads=4, q_tiles=2)),
    (ValueError, lambda: step(rows=ints(1, 2, 3))),
    (ValueError, lambda: step(rows=ints(1, 2, dtype=torch.int32))),
    (ValueError, lambda: step(out=z(2, 4, 64, dtype=torch.float16))),
    (ValueError, lambda: step(out=z(2, 2, 64))),
    (ValueError, lambda: step(weights=z(2, 2, 7, dtype=torch.float32))),
    (ValueError, lambda: step(weights=z(2, 2, 8))),
    (ValueError, lambda: step(q_norm=z(64))),
    (ValueError, lambda: step(cos=z(9, 64), sin=z(9, 64))),
    (ValueError, lambda: step(cos=z(9, 64), sin=z(8, 64), pos=ints(0, 0))),
    (ValueError, lambda: step(cos=z(9, 64), sin=z(9, 64), pos=ints(0))),
    (NotImplementedError, lambda: step(*(z(2, h, 64, dtype=torch.float16) for h in (4, 2, 2)), out=z(2, 4, 64, dtype=torch.float16),
                                       q_norm=z(64), k_norm=z(64))),
    (ValueError, lambda: step()),                                               # not on a GPU
])
def test_step_refuses(error, make):
    with pytest.raises(error):
        make()


def test_step_refuses_shared_buffers():
    q = z(2, 4, 64)
    with pytest.raises(ValueError, match="overlap"):
        step(q=q, out=q)
    with pytest.raises(ValueError, match="together"):
        Cache4AttentionOp(q, z(2, 2, 64), None, cache(), ints(1, 2), z(2, 4, 64), scaling=1.0)


def evict(c=None, w=None, rows=None, **kw):
    kw.setdefault("keep", 4)
    return Cache4EvictOp(cache() if c is None else c, z(2, 2, 8, dtype=torch.float32) if w is None else w,
                         ints(8, 8) if rows is None else rows, **kw)


@pytest.mark.parametrize("error,make", [
    (ValueError, lambda: evict(keep=0)),
    (ValueError, lambda: evict(keep=9)),
    (ValueError, lambda: evict(recent=5)),
    (ValueError, lambda: evict(recent=-1)),
    (ValueError, lambda: evict(w=z(2, 2, 9, dtype=torch.float32))),
    (ValueError, lambda: evict(w=z(2, 2, 8))),
    (ValueError, lambda: evict(rows=ints(8))),
    (ValueError, lambda: evict(out=cache(max_len=4))),
    (ValueError, lambda: evict(out=cache(max_len=3), out_weights=z(2, 2, 3, dtype=torch.float32))),
    (ValueError, lambda: evict(out=cache(n_kv=1, max_len=4), out_weights=z(2, 1, 4, dtype=torch.float32))),
    (ValueError, lambda: evict(out=cache(max_len=4), out_weights=z(2, 2, 5, dtype=torch.float32))),
    (ValueError, lambda: evict(kept=z(2, 2, 5, dtype=torch.int32))),
    (ValueError, lambda: evict(new_rows=ints(0, 0, 0))),
    (ValueError, lambda: evict()),                                              # not on a GPU
])
def test_evict_refuses(error, make):
    with pytest.raises(error):
        make()


def test_evict_refuses_shared_buffers():
    rows = ints(8, 8)
    with pytest.raises(ValueError, match="overlap"):
        evict(rows=rows, new_rows=rows)
    c = cache()
    with pytest.raises(ValueError, match="overlap"):
        evict(c=c, out=c, out_weights=z(2, 2, 8, dtype=torch.float32))


# -- the C entry points: pointers are never followed on the host ---------------------------------------------------------
def c_prompt(**kw):
    a = attention.RvqPromptAttnArgs(16, 16, 16, 16, None, None, None, 6, 6, (ctypes.c_int64 * 2)(256, 64),
                                    (ctypes.c_int64 * 2)(128, 64), (ctypes.c_int64 * 2)(128, 64),
                                    (ctypes.c_int64 * 2)(256, 64), 1, 4, 2, 64, 1.0, 1, _native.RVQ_BF16, 0)
    for name, v in kw.items():
        setattr(a, name, v)
    return attention._lib().rvq_prompt_attention(ctypes.byref(a), None, 0, None)


def test_c_prompt_checks():
    lib = attention._lib()
    assert lib.rvq_prompt_attention(None, None, 0, None) == _native.RVQ_ERR_INVALID
    INV, UNS, BIG = _native.RVQ_ERR_INVALID, _native.RVQ_ERR_UNSUPPORTED, _native.RVQ_ERR_TOO_LARGE
    assert c_prompt(q=None) == INV and c_prompt(k=None) == INV and c_prompt(v=24) == INV
    assert c_prompt(n_kv=3) == INV and c_prompt(n_kv=0) == INV and c_prompt(n_seq=0) == INV and c_prompt(n_seq=2) == INV
    assert c_prompt(head_dim=136) == UNS and c_prompt(head_dim=20) == UNS and c_prompt(kind=_native.RVQ_F32) == UNS
    assert c_prompt(n_heads=130) == UNS and c_prompt(tokens=(1 << 30) + 1) == BIG and c_prompt(keys=(1 << 30) + 1) == BIG
    assert c_prompt(q_stride=(ctypes.c_int64 * 2)(256, 68)) == INV
    assert c_prompt(out_stride=(ctypes.c_int64 * 2)(-256, 64)) == INV
    assert c_prompt(tokens=0) == _native.RVQ_OK


def c_cache(**kw):
    c = attention.RvqCache4(16, 2, 2, 8, 64)
    for name, v in kw.items():
        setattr(c, name, v)
    return c


def test_c_rows_checks():
    lib = attention._lib()
    INV, UNS, BIG = _native.RVQ_ERR_INVALID, _native.RVQ_ERR_UNSUPPORTED, _native.RVQ_ERR_TOO_LARGE
    st = (ctypes.c_int64 * 2)(128, 64)
    for fn in (lib.rvq_cache4_write, lib.rvq_cache4_read):
        def call(c=None, **kw):
            a = attention.RvqCache4RowsArgs(c_cache() if c is None else c, 16, 16, 16, None, 4, st, st, _native.RVQ_BF16, 0)
            for name, v in kw.items():
                setattr(a, name, v)
            return fn(ctypes.byref(a), None)
        assert fn(None, None) == INV
        assert call(c_cache(data=None)) == INV and call(c_cache(data=8)) == INV and call(c_cache(head_dim=32)) == UNS
        assert call(c_cache(max_len=0)) == INV and call(k=None) == INV and call(v=8) == INV and call(cu=None) == INV
        assert call(kind=_native.RVQ_F32) == UNS and call(tokens=1 << 31) == BIG and call(tokens=-1) == INV
        assert call(k_stride=(ctypes.c_int64 * 2)(128, 60)) == INV
        assert call(tokens=0) == _native.RVQ_OK


def test_c_step_checks():
    lib = attention._lib()
    INV, UNS = _native.RVQ_ERR_INVALID, _native.RVQ_ERR_UNSUPPORTED
    B = _native.RVQ_BF16

    def call(**kw):
        a = attention.RvqCache4AttnArgs(RvqVec(16, 512, 1, B), RvqVec(16, 256, 1, B), RvqVec(16, 256, 1, B), None, None,
                                        None, None, None, c_cache(), 16, 16, None, 4, 0, 1e-6, 1.0)
        for name, v in kw.items():
            setattr(a, name, v)
        return lib.rvq_cache4_attention(ctypes.byref(a), None, 0, None)
    assert lib.rvq_cache4_attention(None, None, 0, None) == INV
    assert call(cache=c_cache(data=None)) == INV and call(cache=c_cache(head_dim=80)) == UNS and call(rows=None) == INV
    assert call(n_heads=3) == INV and call(n_heads=130, q=RvqVec(16, 2 * 130 * 64, 1, B)) == UNS
    assert call(q=RvqVec(16, 511, 1, B)) == INV and call(k=RvqVec(None, 0, 0, 0)) == INV
    assert call(k=RvqVec(16, 256, 1, _native.RVQ_F16)) == INV and call(q_norm=16) == INV and call(cos=16, sin=16) == INV
    assert call(cos=16, sin=16, pos=16) == INV                                  # table_len 0
    H = _native.RVQ_F16
    assert call(q=RvqVec(16, 512, 1, H), k=RvqVec(16, 256, 1, H), v=RvqVec(16, 256, 1, H), q_norm=16, k_norm=16) == UNS


def test_c_evict_checks():
    lib = attention._lib()
    INV, UNS = _native.RVQ_ERR_INVALID, _native.RVQ_ERR_UNSUPPORTED

    def call(**kw):
        a = attention.RvqCache4EvictArgs(c_cache(), c_cache(), 16, 16, 16, None, 16, 4, 2)
        for name, v in kw.items():
            setattr(a, name, v)
        return lib.rvq_cache4_evict(ctypes.byref(a), None)
    assert lib.rvq_cache4_evict(None, None) == INV
    assert call(keep=0) == INV and call(keep=9) == INV and call(recent=5) == INV and call(recent=-1) == INV
    assert call(weights=None) == INV and call(kept=None) == INV and call(rows=None) == INV
    assert call(cache=c_cache(head_dim=96), out=c_cache(head_dim=96)) == UNS
    assert call(out=c_cache(data=32)) == INV                                    # overlaps without being the same
    assert call(out=c_cache(max_len=9)) == INV                                  # the same buffer, another length
    assert call(out=c_cache(data=1 << 20, n_kv=1)) == INV
    assert call(out_weights=32) == INV and call(new_rows=16) == INV
