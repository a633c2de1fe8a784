"""GPU: prompt attention, the 4-bit cache and eviction against plain implementations in 64 bits (tests/_attention.py,
where the tolerances are derived)."""

import ctypes

import pytest
import torch

from rvq_b200.attention import (Cache4, Cache4AttentionOp, Cache4EvictOp, Cache4ReadOp, Cache4WriteOp,
                                PromptAttentionOp, take_timeout)
from tests import _attention as ref

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(g, *shape, dtype=BF, scale=1.0):
    return (torch.randn(*shape, generator=g, device=g.device) * scale).to(dtype)


def check(got, want, tol):
    assert torch.equal(torch.isfinite(got), torch.isfinite(want)), "finite places differ"
    ok = torch.isfinite(want)
    off = (got.double() - want).abs()[ok] - tol[ok]
    assert off.numel() == 0 or float(off.max()) <= 0, float(off.max())


def offsets(lens, dev):
    return torch.tensor([0] + list(torch.tensor(lens).cumsum(0)), dtype=torch.int32, device=dev)


def prompt_case(dev, lens, nh, nkv, hd, dtype, causal, prefix=0, seed=0, tail=3, scale=1.0):
    """Runs packed sequences with rows of NaN behind the last; checks every row, and that the tail is left alone."""
    g = gen(dev, seed)
    klens = [n + prefix for n in lens]
    T, S = sum(lens), sum(klens)
    q, k, v = (randn(g, n + tail, h, hd, dtype=dtype, scale=scale) for n, h in ((T, nh), (S, nkv), (S, nkv)))
    for t, n in ((q, T), (k, S), (v, S)):
        t[n:] = float("nan")
    out = torch.full_like(q, 7.0)
    lse = torch.full((nh, T + tail), 7.0, device=dev)
    op = PromptAttentionOp(q, k, v, out, scaling=hd ** -0.5, causal=causal, cu_q=offsets(lens, dev),
                           cu_k=offsets(klens, dev) if prefix else None, lse=lse)
    op.launch()
    assert not take_timeout()
    a = b = 0
    for n, m in zip(lens, klens):
        want, wl, tol, ltol = ref.attend(q[a:a + n], k[b:b + m], v[b:b + m], hd ** -0.5, causal)
        check(out[a:a + n], want, tol)
        check(lse[:, a:a + n], wl, ltol)
        a, b = a + n, b + m
    assert bool((out[T:] == 7).all()) and bool((lse[:, T:] == 7).all())


@pytest.mark.parametrize("hd", [16, 72, 80, 128])
@pytest.mark.parametrize("tokens,prefix", [(70, 0), (9, 3000)])
def test_prompt_output_alignment(tokens, prefix, hd, cuda_device):
    """Output rows and a workspace at 16-byte steps that are no 32-byte steps get the same bits."""
    g = gen(cuda_device, tokens + hd)
    q, k, v = (randn(g, n, h, hd, dtype=BF) for n, h in ((tokens, 8), (tokens + prefix, 2), (tokens + prefix, 2)))
    want = torch.empty_like(q)
    PromptAttentionOp(q, k, v, want, scaling=0.1).launch()
    value, _, tol, _ = ref.attend(q, k, v, 0.1, True)
    check(want, value, tol)
    for lead, gap in ((8, 0), (16, 8), (0, 8), (8, 24)):
        room = torch.full((tokens, 8, lead + hd + gap), 7.0, dtype=BF, device=cuda_device)
        out = room[:, :, lead:lead + hd]
        op = PromptAttentionOp(q, k, v, out, scaling=0.1)
        if op._ws is not None:
            held = torch.zeros(op._ws.numel() + 16, dtype=torch.uint8, device=cuda_device)
            op._bind("rvq_prompt_attention", ctypes.byref(op.args), held.data_ptr() + 16, op._ws.numel())
        op.launch()
        assert torch.equal(out, want)
        assert bool((room[:, :, :lead] == 7).all()) and bool((room[:, :, lead + hd:] == 7).all())
    assert not take_timeout()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lens", [[1], [2], [63], [64], [65], [127, 1], [128], [129, 200], [300], [1, 1, 1, 0, 5, 0, 31],
                                  [517, 3, 260]])
def test_prompt_lengths(lens, causal, dtype, cuda_device):
    prompt_case(cuda_device, lens, 8, 2, 64, dtype, causal, seed=sum(lens))
    prompt_case(cuda_device, lens, 8, 2, 128, dtype, causal, seed=sum(lens) + 1)


@pytest.mark.parametrize("nh,nkv", [(1, 1), (2, 1), (3, 1), (10, 2), (6, 1), (14, 2), (16, 2), (8, 8), (64, 1), (33, 1), (24, 2)])
@pytest.mark.parametrize("hd", [8, 16, 64, 80, 128])
def test_prompt_heads(nh, nkv, hd, cuda_device):
    prompt_case(cuda_device, [150, 77], nh, nkv, hd, BF, True, seed=nh * hd)


@pytest.mark.parametrize("lens,prefix", [([1], 1), ([1], 4000), ([7, 1, 40], 1000), ([130], 129), ([5, 0, 300], 256)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_prompt_after_a_past(lens, prefix, causal, dtype, cuda_device):
    prompt_case(cuda_device, lens, 8, 2, 128, dtype, causal, prefix=prefix, seed=prefix)
    prompt_case(cuda_device, lens, 4, 4, 64, dtype, causal, prefix=prefix, seed=prefix + 1)


def test_prompt_rows_that_see_nothing(cuda_device):
    """Fewer keys than queries: the first queries see no key; sequences without keys."""
    dev = cuda_device
    g = gen(dev, 1)
    for hd in (64, 128):
        ql, kl = [200, 3, 70, 0, 5], [60, 0, 70, 9, 1]
        q, k, v = randn(g, sum(ql), 4, hd), randn(g, sum(kl), 2, hd), randn(g, sum(kl), 2, hd)
        for causal in (True, False):
            out, lse = torch.full_like(q, 7.0), torch.full((4, sum(ql)), 7.0, device=dev)
            PromptAttentionOp(q, k, v, out, scaling=0.125, causal=causal, cu_q=offsets(ql, dev),
                              cu_k=offsets(kl, dev), lse=lse).launch()
            a = b = 0
            for n, m in zip(ql, kl):
                want, wl, tol, ltol = ref.attend(q[a:a + n], k[b:b + m], v[b:b + m], 0.125, causal)
                check(out[a:a + n], want, tol)
                check(lse[:, a:a + n], wl, ltol)
                a, b = a + n, b + m
    # no keys at all
    out = torch.full((9, 4, 64), 7.0, dtype=BF, device=dev)
    PromptAttentionOp(randn(g, 9, 4, 64), randn(g, 0, 2, 64), randn(g, 0, 2, 64), out, scaling=1.0).launch()
    assert bool((out == 0).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("hd", [64, 128])
def test_prompt_hidden_values_may_be_anything(bad, hd, cuda_device):
    """A key and a value of a later token hold NaN or infinities: queries before it are as if it were not there, queries
    from it on see it.  Neighbouring sequences do not see each other."""
    dev = cuda_device
    g = gen(dev, 5)
    for where, n in ((140, 300), (0, 64), (299, 300), (127, 128), (37, 200)):
        q, k, v = randn(g, n + 50, 4, hd), randn(g, n + 50, 2, hd), randn(g, n + 50, 2, hd)
        v[where, 0, 3] = bad
        v[where, 1] = bad
        k[n:] = bad
        v[n:] = bad
        out, lse = torch.zeros_like(q), torch.zeros(4, n + 50, device=dev)
        PromptAttentionOp(q, k, v, out, scaling=0.1, causal=True, cu_q=offsets([n, 50], dev), lse=lse).launch()
        want, wl, tol, ltol = ref.attend(q[:n], k[:n], v[:n], 0.1, True)
        check(out[:n], want, tol)
        got, exp = out[:n].double(), want
        assert torch.equal(got[~torch.isfinite(exp)].nan_to_num(7, 8, 9), exp[~torch.isfinite(exp)].nan_to_num(7, 8, 9))
        check(lse[:, :n], wl, ltol)
        # a bad key
        k = randn(g, n, 2, hd)
        v = randn(g, n, 2, hd)
        k[where] = bad
        out = torch.zeros_like(q[:n])
        PromptAttentionOp(q[:n], k, v, out, scaling=0.1, causal=True).launch()
        if where:
            want, _, tol, _ = ref.attend(q[:where], k[:where], v[:where], 0.1, True)
            check(out[:where], want, tol)
        if bad != bad:
            assert bool(torch.isnan(out[where:]).all())


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tokens,prefix,first", [(64, 0, 40), (128, 0, 128), (300, 0, 230), (40, 1060, 20), (40, 9000, 40)])
def test_prompt_scores_of_minus_infinity_beside_hidden_values(tokens, prefix, first, hd, dtype, bad, cuda_device):
    """The first queries' every score is -infinity (a key channel, where they are positive): zeros, whatever the value of the
    last token holds.  The ones from `first` on, over the finite keys, are as if the others were not there."""
    g = gen(cuda_device, tokens + prefix)
    q, k, v = (randn(g, n, h, hd, dtype=dtype) for n, h in ((tokens, 4), (tokens + prefix, 2), (tokens + prefix, 2)))
    q[..., 0] = q[..., 0].abs() + 0.5
    k[:prefix + first, :, 0] = float("-inf")
    v[-1, 0, 3] = bad
    v[-1, 1] = bad
    out, lse = torch.full_like(q, 7.0), torch.full((4, tokens), 7.0, device=cuda_device)
    PromptAttentionOp(q, k, v, out, scaling=0.1, causal=True, lse=lse).launch()
    assert not take_timeout()
    assert bool((out[:first] == 0).all()) and bool(torch.isneginf(lse[:, :first]).all())
    if first < tokens:
        want, wl, tol, ltol = ref.attend(q[first:], k[prefix + first:], v[prefix + first:], 0.1, True)
        check(out[first:], want, tol)
        check(lse[:, first:], wl, ltol)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,where", [(16384, 16383), (17001, 9000)])
def test_prompt_hidden_value_far_into_a_long_prompt(n, where, hd, bad, cuda_device):
    """One value that is not finite, far into a prompt of many units a CTA: the queries before it in its key tile are summed again
    over all their keys.  The waits of the warps beside that hold on; queries elsewhere keep their bits."""
    dev = cuda_device
    g = gen(dev, n + hd)
    q, k, v = (randn(g, n, h, hd) for h in (8, 2, 2))
    clean, out = torch.empty_like(q), torch.empty_like(q)
    PromptAttentionOp(q, k, v, clean, scaling=0.1).launch()
    v[where, 0, 3] = bad
    v[where, 1] = bad
    PromptAttentionOp(q, k, v, out, scaling=0.1).launch()
    assert not take_timeout()
    first = where - 200                                      # a key tile and a tile of queries before it
    assert torch.equal(out[:first], clean[:first])
    want, _, tol, _ = ref.attend(q[first:where], k[:where], v[:where], 0.1, True)
    check(out[first:where], want, tol)
    hit = torch.zeros(8, hd, dtype=torch.bool, device=dev)
    hit[:4, 3] = True
    hit[4:] = True
    after = out[where:]
    assert torch.equal(after[:, ~hit], clean[where:][:, ~hit])
    assert not bool(torch.isfinite(after[:, hit]).any())


def test_prompt_large_and_equal_scores(cuda_device):
    """Scores far from zero (the running maximum moves by hundreds), rising and falling along the keys; all equal."""
    dev = cuda_device
    g = gen(dev, 9)
    for sign in (1, -1):
        for hd in (64, 128):
            n = 700
            q = randn(g, n, 4, hd).abs()
            k = (torch.linspace(-8, 8, n, device=dev) * sign)[:, None, None].expand(n, 2, hd).to(BF).contiguous()
            v = randn(g, n, 2, hd)
            out, lse = torch.zeros_like(q), torch.zeros(4, n, device=dev)
            for causal in (True, False):
                PromptAttentionOp(q, k, v, out, scaling=0.5, causal=causal, lse=lse).launch()
                want, wl, tol, ltol = ref.attend(q, k, v, 0.5, causal)
                check(out, want, tol)
                check(lse, wl, ltol)
    q = torch.zeros(130, 4, 64, dtype=BF, device=dev)
    k, v = randn(g, 130, 2, 64), randn(g, 130, 2, 64)
    out = torch.empty_like(q)
    PromptAttentionOp(q, k, v, out, scaling=1.0).launch()
    want, _, tol, _ = ref.attend(q, k, v, 1.0, True)
    check(out, want, tol)


@pytest.mark.parametrize("scaling", [-0.2, 0.0, 1.0, 30.0])
def test_prompt_scalings(scaling, cuda_device):
    g = gen(cuda_device, 11)
    q, k, v = (randn(g, 300, h, 128, scale=0.5) for h in (4, 2, 2))
    out, lse = torch.zeros_like(q), torch.zeros(4, 300, device=cuda_device)
    PromptAttentionOp(q, k, v, out, scaling=scaling, lse=lse).launch()
    want, wl, tol, ltol = ref.attend(q, k, v, scaling, True)
    check(out, want, tol)
    check(lse, wl, ltol)


def test_prompt_strided_views(cuda_device):
    """q, k, v as slices of one packed projection, out as a slice of a wider buffer, heads in reverse storage order."""
    dev = cuda_device
    g = gen(dev, 13)
    n, nh, nkv, hd = 210, 6, 2, 128
    qkv = randn(g, n, (nh + 2 * nkv) * hd + 8)
    q = qkv[:, :nh * hd].view(n, nh, hd)
    k = qkv[:, nh * hd:(nh + nkv) * hd].view(n, nkv, hd)
    v = qkv[:, (nh + nkv) * hd:(nh + 2 * nkv) * hd].view(n, nkv, hd)
    wide = torch.full((nh, n, hd + 16), 7.0, dtype=BF, device=dev)
    out = wide[:, :, 8:8 + hd].transpose(0, 1)
    PromptAttentionOp(q, k, v, out, scaling=0.09).launch()
    want, _, tol, _ = ref.attend(q, k, v, 0.09, True)
    check(out, want, tol)
    assert bool((wide[:, :, :8] == 7).all()) and bool((wide[:, :, 8 + hd:] == 7).all())


def test_prompt_long(cuda_device):
    """4,500 tokens, and 9 after 30,000; sums over many tiles."""
    prompt_case(cuda_device, [4500], 4, 1, 128, BF, True, seed=2)
    prompt_case(cuda_device, [9], 8, 2, 128, HF, True, prefix=30000, seed=3)
    prompt_case(cuda_device, [9], 8, 2, 64, BF, False, prefix=30000, seed=4)


def test_prompt_many_sequences(cuda_device):
    """More sequences than a warp has lanes, most of them short or empty, in front of and behind long ones."""
    lens = [1, 0, 2] * 70 + [300] + [0, 5] * 40 + [130] + [1] * 33
    prompt_case(cuda_device, lens, 4, 2, 64, BF, True, seed=6)
    prompt_case(cuda_device, [0] * 100 + [70] + [0] * 100, 16, 2, 128, HF, False, seed=7)


def test_prompt_among_millions_of_empty_sequences(cuda_device):
    """The walk from the last sequence to the first, over three million empty ones, is longer than the waits' bound may be."""
    dev = cuda_device
    g = gen(dev, 53)
    q, k, v = randn(g, 500, 2, 64), randn(g, 500, 1, 64), randn(g, 500, 1, 64)
    cu = torch.full((3_000_003,), 300, dtype=torch.int32, device=dev)
    cu[0], cu[-1] = 0, 500
    out = torch.zeros_like(q)
    PromptAttentionOp(q, k, v, out, scaling=0.1, cu_q=cu).launch()
    assert not take_timeout()
    for a, b in ((0, 300), (300, 500)):
        want, _, tol, _ = ref.attend(q[a:b], k[a:b], v[a:b], 0.1, True)
        check(out[a:b], want, tol)


def test_prompt_bad_offsets_stay_in_bounds(cuda_device):
    """Offsets beyond the tensors are cut off at them."""
    dev = cuda_device
    g = gen(dev, 3)
    q, k, v = (randn(g, 100, h, 64) for h in (4, 2, 2))
    out = torch.zeros_like(q)
    cu = torch.tensor([0, 60, 1000], dtype=torch.int32, device=dev)
    PromptAttentionOp(q, k, v, out, scaling=0.125, cu_q=cu).launch()
    for a, b in ((0, 60), (60, 100)):
        want, _, tol, _ = ref.attend(q[a:b], k[a:b], v[a:b], 0.125, True)
        check(out[a:b], want, tol)


# -- the 4-bit cache ---------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("lens,start", [([1], [0]), ([5], [3]), ([0, 1, 17, 0, 200], [4, 9, 0, 1, 31])])
def test_write_then_read(lens, start, dtype, hd, cuda_device):
    """Records are the definition's, byte for byte; the rest of the cache is left alone; read gives the held values."""
    dev = cuda_device
    g = gen(dev, hd + len(lens))
    B, nkv, T = len(lens), 3, sum(lens)
    max_len = max(n + s for n, s in zip(lens, start)) + 2
    k = randn(g, T + 2, nkv, hd, dtype=dtype)
    v = randn(g, T + 2, nkv, hd, dtype=dtype, scale=3.0)
    k[0, 0, :32] = 0.5                       # a group of equal values
    k[0, 1, :32] = 0.0
    k[0, 2, 5] = 300.0
    v[0, 0, 32:64] = torch.linspace(-1, 1, 32, device=dev).to(dtype)
    cache = Cache4(B, nkv, max_len, hd, dev)
    cache.data.fill_(0xA5)
    want = cache.data.clone()
    cu, st = offsets(lens, dev), torch.tensor(start, dtype=torch.int64, device=dev)
    Cache4WriteOp(cache, k, v, cu=cu, start=st).launch()
    ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    Cache4ReadOp(cache, ko, vo, cu=cu, start=st).launch()
    a = 0
    for b, (n, s) in enumerate(zip(lens, start)):
        want[b, :, s:s + n] = ref.records(k[a:a + n], v[a:a + n]).transpose(0, 1)
        a += n
    assert torch.equal(cache.data, want)
    assert torch.equal(ko[:T], ref.held(k[:T]).to(dtype)) and torch.equal(vo[:T], ref.held(v[:T]).to(dtype))
    assert bool((ko[T:] == 7).all()) and bool((vo[T:] == 7).all())


def test_quantisation_error_is_half_a_step(cuda_device):
    """Held values are within half a step (and the roundings of zero and step to bf16) of what was written."""
    g = gen(cuda_device, 8)
    k, v = randn(g, 500, 2, 128), randn(g, 500, 2, 128)
    cache = Cache4(1, 2, 500, 128, cuda_device)
    Cache4WriteOp(cache, k, v).launch()
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    Cache4ReadOp(cache, ko, vo).launch()
    for x, y in ((k, ko), (v, vo)):
        x = x.float().unflatten(-1, (4, 32))
        span = x.amax(-1, keepdim=True) - x.amin(-1, keepdim=True)
        # half of a step that is at most 2^-8 too wide; 15 steps that are 2^-8 too narrow miss the top by 15 2^-8 steps;
        # the read value is rounded to bf16
        tol = span / 15 * (0.5 + 15.5 * 2.0 ** -8) + x.abs() * 2.0 ** -8 + span * 2.0 ** -8
        assert bool(((x - y.float().unflatten(-1, (4, 32))).abs() <= tol).all())


def test_write_outside_the_cache_is_dropped(cuda_device):
    dev = cuda_device
    g = gen(dev, 2)
    k, v = randn(g, 10, 2, 64), randn(g, 10, 2, 64)
    cache = Cache4(2, 2, 6, 64, dev)
    cu = torch.tensor([0, 5, 10], dtype=torch.int32, device=dev)
    st = torch.tensor([-2, 3], dtype=torch.int64, device=dev)
    Cache4WriteOp(cache, k, v, cu=cu, start=st).launch()
    want = torch.zeros_like(cache.data)
    want[0, :, 0:3] = ref.records(k[2:5], v[2:5]).transpose(0, 1)
    want[1, :, 3:6] = ref.records(k[5:8], v[5:8]).transpose(0, 1)
    assert torch.equal(cache.data, want)
    ko, vo = torch.full_like(k, 7.0), torch.full_like(v, 7.0)
    Cache4ReadOp(cache, ko, vo, cu=cu, start=st).launch()
    assert bool((ko[:2] == 0).all()) and bool((vo[8:] == 0).all())
    assert torch.equal(ko[2:8], ref.held(k[2:8]).to(BF))
    huge = torch.tensor([2 ** 40, -2 ** 40], dtype=torch.int64, device=dev)
    Cache4WriteOp(cache, k, v, cu=cu, start=huge).launch()
    assert torch.equal(cache.data, want)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_non_finite_groups_are_held_as_such(bad, cuda_device):
    g = gen(cuda_device, 4)
    k, v = randn(g, 4, 1, 64), randn(g, 4, 1, 64)
    k[1, 0, 7] = bad
    cache = Cache4(1, 1, 4, 64, cuda_device)
    Cache4WriteOp(cache, k, v).launch()
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    Cache4ReadOp(cache, ko, vo).launch()
    assert not bool(torch.isfinite(ko[1, 0, :32]).any())
    rest = [0, 2, 3]
    assert torch.equal(ko[rest], ref.held(k)[rest].to(BF)) and torch.equal(ko[1, 0, 32:], ref.held(k)[1, 0, 32:].to(BF))
    assert torch.equal(vo, ref.held(v).to(BF))


def test_rows_of_strided_tensors(cuda_device):
    g = gen(cuda_device, 6)
    wide = randn(g, 20, 2 * 3 * 64 + 8)
    k, v = wide[:, :192].view(20, 3, 64), wide[:, 192:384].view(20, 3, 64)
    cache = Cache4(1, 3, 20, 64, cuda_device)
    Cache4WriteOp(cache, k, v).launch()
    assert torch.equal(cache.data[0], ref.records(k, v).transpose(0, 1))
    out = torch.full((3, 20, 2, 72), 7.0, dtype=BF, device=cuda_device)
    ko, vo = out[:, :, 0, :64].transpose(0, 1), out[:, :, 1, :64].transpose(0, 1)
    Cache4ReadOp(cache, ko, vo).launch()
    assert torch.equal(ko, ref.held(k).to(BF)) and torch.equal(vo, ref.held(v).to(BF))
    assert bool((out[..., 64:] == 7).all())


def filled(dev, g, B, nkv, max_len, hd):
    """A cache of quantised random rows."""
    k = randn(g, B * nkv * max_len, 1, hd, scale=1.5)
    v = randn(g, B * nkv * max_len, 1, hd)
    flat = Cache4(1, 1, B * nkv * max_len, hd, dev)
    Cache4WriteOp(flat, k, v).launch()
    return Cache4(B, nkv, max_len, hd, data=flat.data.view(B, nkv, max_len, -1))


def step_case(dev, rows, nh, nkv, hd, dtype, max_len, seed=0, append=True, weigh=True):
    g = gen(dev, seed)
    B, rep = len(rows), nh // nkv
    cache = filled(dev, g, B, nkv, max_len, hd)
    for b, n in enumerate(rows):
        cache.data[b, :, max(n, 0):] = 0xFF                   # NaN parameters behind the live rows
    before = cache.data.clone()
    q, k, v = randn(g, B, nh, hd, dtype=dtype), randn(g, B, nkv, hd, dtype=dtype), randn(g, B, nkv, hd, dtype=dtype)
    out = torch.full_like(q, 7.0)
    w = torch.rand(B, nkv, max_len, generator=g, device=dev) if weigh else None
    w0 = w.clone() if weigh else None
    rt = torch.tensor(rows, dtype=torch.int64, device=dev)
    Cache4AttentionOp(q, k if append else None, v if append else None, cache, rt, out, scaling=hd ** -0.5,
                      weights=w).launch()
    assert not take_timeout()
    new = ref.records(k, v)
    for b, n in enumerate(rows):
        total = n + append
        if n < 0 or total < 1 or total > max_len:
            assert bool((out[b] == (7 if n < 0 else 0)).all())
            if weigh:
                assert torch.equal(w[b], w0[b])
            continue
        if append:
            before[b, :, n] = new[b]
        for h in range(nkv):
            want, ww, tol, wtol = ref.attend_cache(q[b, h * rep:(h + 1) * rep], before[b, h], total, hd, hd ** -0.5)
            check(out[b, h * rep:(h + 1) * rep], want, tol)
            if weigh:
                base = w0[b, h, :total].double()
                if append:
                    base[n] = 0
                check(w[b, h, :total], base + ww, wtol + 2.0 ** -22 * (base + ww))
                assert torch.equal(w[b, h, total:], w0[b, h, total:])
    assert torch.equal(cache.data, before)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("rows", [[0], [1], [15], [16], [17], [31, 32, 33], [100], [300, 0, 7], [1000], [255, 256, 511]])
def test_step_lengths(rows, dtype, hd, cuda_device):
    step_case(cuda_device, rows, 8, 2, hd, dtype, max(rows) + 9, seed=sum(rows) + hd)


@pytest.mark.parametrize("weigh", [False, True])
@pytest.mark.parametrize("max_len", [128, 129, 384, 385, 640, 641, 1024, 1025])
@pytest.mark.parametrize("seqs,nh,nkv", [(1, 8, 2), (2, 9, 1), (40, 8, 8)])
def test_step_short_caches(seqs, nh, nkv, max_len, weigh, cuda_device):
    # full to the last row, and a few rows of the same cache
    rows = [max_len - 1 if b % 2 == 0 else max_len // 3 for b in range(seqs)]
    step_case(cuda_device, rows, nh, nkv, 64, BF, max_len, seed=max_len + seqs, weigh=weigh)


@pytest.mark.parametrize("nh,nkv", [(1, 1), (2, 1), (3, 1), (6, 2), (7, 1), (16, 2), (9, 1), (12, 1), (16, 1), (40, 2), (64, 1), (8, 8)])
def test_step_heads(nh, nkv, cuda_device):
    step_case(cuda_device, [130, 61], nh, nkv, 128, BF, 140, seed=nh)
    step_case(cuda_device, [130, 61], nh, nkv, 64, HF, 140, seed=nh, weigh=False)


def test_step_odd_calls(cuda_device):
    """No append, skipped sequences, no room, nothing to attend to, a full cache."""
    for weigh in (False, True):
        step_case(cuda_device, [40, -1, 0, 64, 65, 12], 4, 2, 64, BF, 64, append=False, weigh=weigh)
        step_case(cuda_device, [63, -1, 64, 0, 70, -9], 4, 2, 128, BF, 64, append=True, weigh=weigh)
        step_case(cuda_device, [2 ** 40, 3], 4, 2, 128, BF, 64, append=True, weigh=weigh)


@pytest.mark.parametrize("rows", [[5000], [20011], [3000, 1, 2999, 4096], [700] * 40])
def test_step_long_and_many(rows, cuda_device):
    step_case(cuda_device, rows, 8, 2, 128, BF, max(rows) + 1, seed=len(rows))
    step_case(cuda_device, rows, 4, 1, 64, HF, max(rows) + 5, seed=len(rows) + 1, weigh=False)


def test_step_offsets_beyond_32_bits(cuda_device):
    """A cache of more than 4 GiB; the live rows are at its far end."""
    dev = cuda_device
    B, nkv, hd, max_len = 3, 8, 128, 1_200_000                # 4.6 GB
    cache = Cache4(B, nkv, max_len, hd, dev)
    g = gen(dev, 1)
    n = 300
    k, v = randn(g, n, nkv, hd), randn(g, n, nkv, hd)
    start = max_len - n - 1
    cu = torch.tensor([0, 0, 0, n], dtype=torch.int32, device=dev)
    st = torch.tensor([0, 0, start], dtype=torch.int64, device=dev)
    Cache4WriteOp(cache, k, v, cu=cu, start=st).launch()
    assert torch.equal(cache.data[2, :, start:start + n], ref.records(k, v).transpose(0, 1))
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    Cache4ReadOp(cache, ko, vo, cu=cu, start=st).launch()
    assert torch.equal(ko, ref.held(k).to(BF))
    q, kn, vn = randn(g, B, 32, hd), randn(g, B, nkv, hd), randn(g, B, nkv, hd)
    rows = torch.tensor([-1, -1, max_len - 1], dtype=torch.int64, device=dev)
    out = torch.zeros_like(q)
    w = torch.zeros(B, nkv, max_len, device=dev)
    Cache4AttentionOp(q, kn, vn, cache, rows, out, scaling=0.1, weights=w).launch()
    assert not take_timeout()
    assert torch.equal(cache.data[2, :, max_len - 1], ref.records(kn, vn)[2])
    # rows before `start` hold zeros: score 0 and value 0
    want, ww, tol, wtol = ref.attend_cache(q[2, 28:32], cache.data[2, 7, start:], n + 1, hd, 0.1)
    lse_tail = torch.logsumexp(q[2, 28:32].double() @ ref.values(*[t.double() for t in ref.unpack(
        cache.data[2, 7, start:], hd)[0]]).T * 0.1, -1)
    share = 1 / (1 + start * torch.exp(-lse_tail))
    # sums of 1.2 million weights in fp32: relative 2^-24 times the number of additions along the longest chain
    grow = 1 + 4 * max_len * 2.0 ** -24
    check(out[2, 28:32], want * share[:, None], tol * grow + (grow - 1) * want.abs() * share[:, None] + 2.0 ** -20)
    wsum = w[2, 7].double().sum()
    assert abs(float(wsum) - 4) <= 4 * (grow - 1) + 1e-3
    assert bool((w[:2] == 0).all())


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("max_len", [50, 4000])
def test_step_operands_anywhere(max_len, dtype, cuda_device):
    """q, k, v and out at addresses of single elements: the same bits, and nothing beside out is written."""
    dev = cuda_device
    g = gen(dev, max_len)
    B, nh, nkv, hd = 2, 6, 2, 64
    data = filled(dev, g, B, nkv, max_len, hd).data
    rows = torch.tensor([max_len - 1, 17], dtype=torch.int64, device=dev)
    whole = [randn(g, B, h, hd, dtype=dtype) for h in (nh, nkv, nkv)]
    want = torch.zeros(B, nh, hd, dtype=dtype, device=dev)
    Cache4AttentionOp(*whole, Cache4(B, nkv, max_len, hd, data=data.clone()), rows, want, scaling=0.1).launch()

    def shifted(x, by):
        room = torch.full((x.numel() + 16,), 7.0, dtype=dtype, device=dev)
        room[by:by + x.numel()] = x.flatten()
        return room, room[by:by + x.numel()].view(x.shape)

    for by in (1, 3, 8):
        room, out = shifted(torch.zeros_like(want), by)
        Cache4AttentionOp(*(shifted(x, by)[1] for x in whole), Cache4(B, nkv, max_len, hd, data=data.clone()), rows, out,
                          scaling=0.1).launch()
        assert torch.equal(out, want)
        assert bool((room[:by] == 7).all()) and bool((room[by + out.numel():] == 7).all())


def rotated(x, w, eps, cos, sin):
    """Per-head RMSNorm and rotary embedding with the roundings of rvq_b200.decoder."""
    from rvq_b200.decoder import rmsnorm, rotate_half
    x = rmsnorm(x, w, eps)
    return x * cos + rotate_half(x) * sin


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tiles", [0, 5])
def test_step_with_norm_and_rotation(hd, tiles, cuda_device):
    """Raw projections (bf16 or fp32 partials) with norms and positions.  The norm's fp32 sums may round differently, by
    one bf16 step in a few values: outputs agree within bf16 noise, records almost everywhere."""
    dev = cuda_device
    g = gen(dev, hd + tiles)
    B, nh, nkv, max_len = 3, 8, 2, 90
    cache = filled(dev, g, B, nkv, max_len, hd)
    rows = torch.tensor([80, 0, 33], dtype=torch.int64, device=dev)
    pos = torch.tensor([400, 0, 77], dtype=torch.int64, device=dev)
    qn, kn = (1 + 0.1 * randn(g, hd).float()).to(BF), (1 + 0.1 * randn(g, hd).float()).to(BF)
    ang = torch.randn(500, hd // 2, generator=g, device=dev).repeat(1, 2)
    cos, sin = ang.cos().to(BF), ang.sin().to(BF)
    if tiles:
        parts = [torch.randn(tiles, B, h, hd, generator=g, device=dev) for h in (nh, nkv, nkv)]
        whole = []
        for p in parts:
            s = p[0].clone()
            for t in range(1, tiles):
                s += p[t]
            whole.append(s.to(BF))
    else:
        whole = parts = [randn(g, B, h, hd) for h in (nh, nkv, nkv)]
    before = cache.data.clone()
    out = torch.zeros(B, nh * hd, dtype=BF, device=dev)
    Cache4AttentionOp(*parts, cache, rows, out, n_heads=nh, scaling=hd ** -0.5, q_norm=qn, k_norm=kn, cos=cos, sin=sin,
                      pos=pos, eps=1e-6, q_tiles=max(tiles, 1), kv_tiles=max(tiles, 1)).launch()
    c, s = cos[pos][:, None], sin[pos][:, None]
    q, k = rotated(whole[0], qn, 1e-6, c, s), rotated(whole[1], kn, 1e-6, c, s)
    rec = ref.records(k, whole[2])
    for b in range(B):
        n = int(rows[b])
        got = cache.data[b, :, n]
        assert float((got != rec[b]).float().mean()) < 0.05
        before[b, :, n] = got                                # attention goes over what was appended
        for h in range(nkv):
            want, _, tol, _ = ref.attend_cache(q[b, 4 * h:4 * h + 4], before[b, h], n + 1, hd, hd ** -0.5)
            # a step of bf16 in a few of q's values moves scores by up to 2^-8 |q||k| scaling
            (_, kz, ks), _ = ref.unpack(before[b, h, :n + 1], hd)
            move = 2.0 ** -7 * hd ** -0.5 * float(q[b].float().abs().max()) * float((kz.abs() + 15 * ks).max()) * 8
            check(out.view(B, nh, hd)[b, 4 * h:4 * h + 4], want, tol + move * want.abs().amax())
    assert torch.equal(cache.data, before)


@pytest.mark.parametrize("norm,rotate", [(True, True), (True, False), (False, True)])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("tiles", [0, 5])
def test_step_norm_and_rotation_bit_by_bit(tiles, hd, norm, rotate, cuda_device):
    """Small whole numbers as projections: their sums of squares are exact in any order, so that norm and rotation have one
    result, and a call that does them has the bits (outputs, weights, records) of one that is given the normed and rotated q and k.
    Calls with other norms or positions do not."""
    from rvq_b200.decoder import rmsnorm, rotate_half
    dev = cuda_device
    g = gen(dev, 7 * hd + tiles)
    B, nh, nkv, max_len = 3, 8, 2, 700
    data = filled(dev, g, B, nkv, max_len, hd).data
    rows = torch.tensor([650, 1, 33], dtype=torch.int64, device=dev)
    pos = torch.tensor([400, 3, 77], dtype=torch.int64, device=dev)
    qn, kn = (torch.empty(hd, device=dev).uniform_(0.25, 2, generator=g).to(BF) for _ in range(2))
    ang = torch.randn(500, hd // 2, generator=g, device=dev).repeat(1, 2)
    cos, sin = ang.cos().to(BF), ang.sin().to(BF)
    shapes = [(B, h, hd) for h in (nh, nkv, nkv)]
    if tiles:
        parts = [torch.randint(-3, 4, (tiles, *s), generator=g, device=dev).float() for s in shapes]
        whole = [p.sum(0).to(BF) for p in parts]
    else:
        whole = parts = [torch.randint(-9, 10, s, generator=g, device=dev).to(BF) for s in shapes]

    def call(q, k, v, q_tiles=1, **kw):
        cache = Cache4(B, nkv, max_len, hd, data=data.clone())
        out, w = torch.zeros(B, nh, hd, dtype=BF, device=dev), torch.ones(B, nkv, max_len, device=dev)
        Cache4AttentionOp(q, k, v, cache, rows, out, n_heads=nh, scaling=hd ** -0.5, weights=w, q_tiles=q_tiles,
                          kv_tiles=q_tiles, **kw).launch()
        return out, w, cache.data

    def options(qn=qn, kn=kn, pos=pos):
        return dict(**(dict(q_norm=qn, k_norm=kn, eps=1e-6) if norm else {}),
                    **(dict(cos=cos, sin=sin, pos=pos) if rotate else {}))

    turned = lambda x: x * cos[pos][:, None] + rotate_half(x) * sin[pos][:, None] if rotate else x
    given = lambda x, w: turned(rmsnorm(x, w, 1e-6) if norm else x)
    want = call(given(whole[0], qn), given(whole[1], kn), whole[2])
    got = call(*parts, max(tiles, 1), **options())
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    # and that says something: the longest sequence has other bits where q's norm, its weights or a position is another, in every
    # head (without a norm, where one row may have all the weight whatever the position, in some head)
    other = [] if not norm else [call(*parts, max(tiles, 1), **options(qn=torch.ones_like(qn))),
                                 call(given(whole[0], torch.ones_like(qn)), given(whole[1], kn), whole[2])]
    if norm:
        other.append(call(turned(whole[0] * qn), given(whole[1], kn), whole[2]))
    if rotate:
        other.append(call(*parts, max(tiles, 1), **options(pos=pos + 1)))
    for out, *_ in other:
        differs = (out != want[0])[0].any(-1)
        assert bool(differs.all() if norm else differs.any())


# -- eviction ----------------------------------------------------------------------------------------------------------
def evict_case(dev, rows, nkv, hd, max_len, keep, recent, w, in_place, seed=0):
    g = gen(dev, seed)
    B = len(rows)
    data = torch.randint(0, 256, (B, nkv, max_len, hd * 5 // 4), dtype=torch.uint8, generator=g, device=dev)
    src, w0, old = data.clone(), w.clone(), torch.tensor(rows, dtype=torch.int64, device=dev)
    cache = Cache4(B, nkv, max_len, hd, data=data)
    new = torch.full((B,), 77, dtype=torch.int64, device=dev)
    if in_place:
        op, od, ow = Cache4EvictOp(cache, w, old, keep=keep, recent=recent, new_rows=new), data, w
        base_d, base_w = src.clone(), w0.clone()
    else:
        od = torch.full((B, nkv, keep + 3, hd * 5 // 4), 9, dtype=torch.uint8, device=dev)
        ow = torch.full((B, nkv, keep + 3), 9.0, device=dev)
        base_d, base_w = od.clone(), ow.clone()
        op = Cache4EvictOp(cache, w, old, keep=keep, recent=recent, out=Cache4(B, nkv, keep + 3, hd, data=od),
                           out_weights=ow, new_rows=new)
    op.launch()
    wl = w0.cpu().tolist()
    for b, n in enumerate(rows):
        n = min(n, max_len)
        assert int(new[b]) == min(n, keep)
        for h in range(nkv):
            want = ref.kept_rows(wl[b][h], n, keep, recent)
            assert op.kept[b, h].tolist() == want + [-1] * (keep - len(want))
            base_d[b, h, :len(want)] = src[b, h, want]
            base_w[b, h, :len(want)] = w0[b, h, want]
    assert torch.equal(od, base_d)
    assert torch.equal(ow.nan_to_num(-5), base_w.nan_to_num(-5))
    if not in_place:
        assert torch.equal(data, src) and torch.equal(w.nan_to_num(-5), w0.nan_to_num(-5))


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("max_len,keep,recent", [(1, 1, 0), (2, 1, 0), (2, 1, 1), (40, 7, 3), (40, 7, 7), (40, 7, 0), (40, 40, 5),
                                                 (1100, 1024, 64), (3000, 1000, 1), (1030, 1029, 1029), (2500, 2047, 500)])
def test_evict(max_len, keep, recent, hd, in_place, cuda_device):
    g = gen(cuda_device, max_len)
    rows = [max_len, max_len - 1, min(keep, max_len), 0, -1, max_len + 5, max(keep - 1, 0)]
    w = torch.rand(len(rows), 3, max_len, generator=g, device=cuda_device)
    evict_case(cuda_device, rows, 3, hd, max_len, keep, recent, w, in_place)


@pytest.mark.parametrize("in_place", [False, True])
def test_evict_odd_weights(in_place, cuda_device):
    """Ties, zeros of both signs, infinities, NaN, negative and subnormal weights."""
    dev = cuda_device
    g = gen(dev, 3)
    n = 700
    few = torch.tensor([0.0, -0.0, 1.0, float("inf"), float("nan"), -1.0, 1e-42, -float("inf")], device=dev)
    w = few[torch.randint(0, 8, (4, 2, n), generator=g, device=dev)]
    w[1] = 0.0
    w[2] = 3.5
    w[3, 0, ::2] = -0.0
    w[3, 0, 1::2] = 0.0
    for keep, recent in ((100, 0), (350, 100), (650, 649), (1, 0), (200, 199)):
        evict_case(dev, [n, n, n - 3, n], 2, 64, n, keep, recent, w.clone(), in_place)


def test_evict_long(cuda_device):
    g = gen(cuda_device, 7)
    w = torch.randn(2, 2, 70000, generator=g, device=cuda_device).mul(2).exp()
    w = w * (torch.rand(w.shape, generator=g, device=cuda_device) > 0.3)
    evict_case(cuda_device, [70000, 65537], 2, 64, 70000, 60000, 128, w, True)


# -- together, captured, and on other streams ---------------------------------------------------------------------------
def test_a_conversation(cuda_device):
    """A prompt into the cache, steps with their weights, eviction when the budget is passed, steps again, the next turn's
    prompt over the rows read back: every stage against 64 bits."""
    dev = cuda_device
    g = gen(dev, 21)
    nh, nkv, hd, max_len, keep, recent = 8, 2, 128, 128, 64, 8
    cache = Cache4(1, nkv, max_len, hd, dev)
    w = torch.zeros(1, nkv, max_len, device=dev)
    n = 70
    q, k, v = randn(g, n, nh, hd), randn(g, n, nkv, hd), randn(g, n, nkv, hd)
    out = torch.empty_like(q)
    PromptAttentionOp(q, k, v, out, scaling=0.09).launch()
    Cache4WriteOp(cache, k, v).launch()
    want, _, tol, _ = ref.attend(q, k, v, 0.09, True)
    check(out, want, tol)
    rows = torch.tensor([n], dtype=torch.int64, device=dev)
    qs, ks, vs = torch.empty(1, nh, hd, dtype=BF, device=dev), *(torch.empty(1, nkv, hd, dtype=BF, device=dev) for _ in "kv")
    o = torch.empty_like(qs)
    step = Cache4AttentionOp(qs, ks, vs, cache, rows, o, scaling=0.09, weights=w)
    evict = Cache4EvictOp(cache, w, rows, keep=keep, recent=recent)
    mirror, total = cache.data.clone(), [[0.0] * n for _ in range(nkv)]
    wtol = 0.0
    for i in range(40):
        for t in (qs, ks, vs):
            t.copy_(randn(g, *t.shape))
        step.launch()
        mirror[0, :, n] = ref.records(ks, vs)[0]
        for h in range(nkv):
            want, ww, tol, wt = ref.attend_cache(qs[0, 4 * h:4 * h + 4], mirror[0, h], n + 1, hd, 0.09)
            check(o[0, 4 * h:4 * h + 4], want, tol)
            total[h] = [a + b for a, b in zip(total[h] + [0.0], ww.tolist())]
            wtol = max(wtol, 41 * float(wt.max()) + 41 * 2.0 ** -20)
            got = w[0, h, :n + 1].tolist()
            assert max(abs(a - b) for a, b in zip(got, total[h])) <= wtol
        n += 1
        rows.fill_(n)
        if n == 80:
            kept = [ref.kept_rows(w[0, h, :n].tolist(), n, keep, recent) for h in range(nkv)]
            evict.launch()
            for h in range(nkv):
                assert evict.kept[0, h].tolist() == kept[h]
                mirror[0, h, :keep] = mirror[0, h, kept[h]].clone()
                total[h] = [total[h][j] for j in kept[h]]
            n = keep
            rows.fill_(n)
        assert torch.equal(cache.data, mirror)
    kp, vp = torch.empty(n, nkv, hd, dtype=BF, device=dev), torch.empty(n, nkv, hd, dtype=BF, device=dev)
    Cache4ReadOp(cache, kp, vp).launch()
    q2, k2, v2 = randn(g, 30, nh, hd), randn(g, 30, nkv, hd), randn(g, 30, nkv, hd)
    out = torch.empty_like(q2)
    ka, va = torch.cat((kp, k2)), torch.cat((vp, v2))
    PromptAttentionOp(q2, ka, va, out, scaling=0.09).launch()
    want, _, tol, _ = ref.attend(q2, ka, va, 0.09, True)
    check(out, want, tol)


def test_captured_graphs_replay(cuda_device):
    """All operators in one graph, replayed with new contents; a second graph of other ops between the replays."""
    dev = cuda_device
    g = gen(dev, 31)
    nh, nkv, hd, n, max_len = 8, 2, 64, 200, 300

    def build():
        t = dict(q=randn(g, n, nh, hd), k=randn(g, n, nkv, hd), v=randn(g, n, nkv, hd))
        t["out"], t["cache"] = torch.zeros_like(t["q"]), Cache4(1, nkv, max_len, hd, dev)
        t["rows"] = torch.tensor([n], dtype=torch.int64, device=dev)
        t["q1"], t["k1"], t["v1"] = randn(g, 1, nh, hd), randn(g, 1, nkv, hd), randn(g, 1, nkv, hd)
        t["o1"], t["w"] = torch.zeros_like(t["q1"]), torch.zeros(1, nkv, max_len, device=dev)
        t["out_c"], t["out_w"] = Cache4(1, nkv, 100, hd, dev), torch.zeros(1, nkv, 100, device=dev)
        t["live"] = torch.tensor([n + 1], dtype=torch.int64, device=dev)
        t["ops"] = [PromptAttentionOp(t["q"], t["k"], t["v"], t["out"], scaling=0.125),
                    Cache4WriteOp(t["cache"], t["k"], t["v"]),
                    Cache4AttentionOp(t["q1"], t["k1"], t["v1"], t["cache"], t["rows"], t["o1"], scaling=0.125,
                                      weights=t["w"]),
                    Cache4EvictOp(t["cache"], t["w"], t["live"], keep=100, recent=10, out=t["out_c"],
                                  out_weights=t["out_w"])]
        return t

    def go(t):
        t["w"].zero_()
        for op in t["ops"]:
            op.launch()

    sets = [build(), build()]
    graphs = []
    s = torch.cuda.Stream(dev)
    for t in sets:
        with torch.cuda.stream(s):
            go(t)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            go(t)
        graphs.append(graph)
    for turn in range(3):
        for t in sets:
            for name in ("q", "k", "v", "q1", "k1", "v1"):
                t[name].copy_(randn(g, *t[name].shape))
        for graph in graphs:
            graph.replay()
        for t in sets:
            want, _, tol, _ = ref.attend(t["q"], t["k"], t["v"], 0.125, True)
            check(t["out"], want, tol)
            rec = torch.cat((ref.records(t["k"], t["v"]), ref.records(t["k1"], t["v1"]))).transpose(0, 1)
            assert torch.equal(t["cache"].data[0, :, :n + 1], rec)
            for h in range(nkv):
                want, ww, tol, wtol = ref.attend_cache(t["q1"][0, 4 * h:4 * h + 4], rec[h], n + 1, hd, 0.125)
                check(t["o1"][0, 4 * h:4 * h + 4], want, tol)
                check(t["w"][0, h, :n + 1], ww, wtol)
                kept = ref.kept_rows(t["w"][0, h].tolist(), n + 1, 100, 10)
                assert t["ops"][3].kept[0, h].tolist() == kept
                assert torch.equal(t["out_c"].data[0, h], rec[h, kept])
    assert not take_timeout()


def test_prompt_workspace_on_the_stream_of_its_first_launch(cuda_device):
    """More pairs of tiles than SMs (they are given out by a counter in the workspace, which starts as whatever the memory
    held): an op built on one stream and launched on another, one whose first launch is captured, then both again."""
    dev = cuda_device
    g = gen(dev, 61)
    q, k, v = randn(g, 1500, 32, 64), randn(g, 1500, 8, 64), randn(g, 1500, 8, 64)
    want, _, tol, _ = ref.attend(q, k, v, 0.125, True)
    junk = [torch.full((n,), 255, dtype=torch.uint8, device=dev) for n in (8, 16, 512)]
    torch.cuda.synchronize()
    del junk
    out = torch.zeros_like(q)
    op = PromptAttentionOp(q, k, v, out, scaling=0.125)
    side = torch.cuda.Stream(dev)
    for _ in range(3):
        with torch.cuda.stream(side):
            op.launch()
    torch.cuda.synchronize()
    check(out, want, tol)
    junk = [torch.full((n,), 255, dtype=torch.uint8, device=dev) for n in (8, 16, 512)]
    torch.cuda.synchronize()
    del junk
    op = PromptAttentionOp(q, k, v, out, scaling=0.125)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        op.launch()
    for how in (op.launch, graph.replay, graph.replay, op.launch, graph.replay):
        out.zero_()
        how()
        check(out, want, tol)
    assert not take_timeout()


def test_ops_built_in_inference_mode_run_outside(cuda_device):
    """And the other way round; 512 units, so that the prompt's workspace holds tickets."""
    dev = cuda_device
    g = gen(dev, 47)
    q, k, v = randn(g, 2048, 8, 64), randn(g, 2048, 8, 64), randn(g, 2048, 8, 64)
    out, other = torch.empty_like(q), torch.empty_like(q)
    with torch.inference_mode():
        op = PromptAttentionOp(q, k, v, out, scaling=0.1)
    assert op._ws is not None
    op.launch()
    op = PromptAttentionOp(q, k, v, other, scaling=0.1)
    with torch.inference_mode():
        op.launch()
    op.launch()
    assert torch.equal(out, other) and not take_timeout()
    want, _, tol, _ = ref.attend(q[-200:], k, v, 0.1, True)
    check(out[-200:], want, tol)


def test_two_streams_at_once(cuda_device):
    """The same kinds of op with their own buffers on two streams at the same time."""
    dev = cuda_device
    g = gen(dev, 41)
    jobs = []
    for i in range(2):
        q, k, v = randn(g, 900, 8, 128), randn(g, 900, 2, 128), randn(g, 900, 2, 128)
        cache = filled(dev, g, 4, 2, 1000, 128)
        q1, rows = randn(g, 4, 8, 128), torch.tensor([900, 5, 1000, 64], dtype=torch.int64, device=dev)
        o, o1, w = torch.zeros_like(q), torch.zeros_like(q1), torch.zeros(4, 2, 1000, device=dev)
        jobs.append((q, k, v, cache, q1, rows, o, o1, w, PromptAttentionOp(q, k, v, o, scaling=0.1),
                     Cache4AttentionOp(q1, None, None, cache, rows, o1, scaling=0.1, weights=w), torch.cuda.Stream(dev)))
    torch.cuda.synchronize()
    for _ in range(5):
        for *_, w, prompt, step, stream in jobs:
            with torch.cuda.stream(stream):
                w.zero_()
                prompt.launch()
                step.launch()
    torch.cuda.synchronize()
    for q, k, v, cache, q1, rows, o, o1, w, *_ in jobs:
        want, _, tol, _ = ref.attend(q, k, v, 0.1, True)
        check(o, want, tol)
        for b in range(4):
            for h in range(2):
                n = int(rows[b])
                want, ww, tol, wtol = ref.attend_cache(q1[b, 4 * h:4 * h + 4], cache.data[b, h], n, 128, 0.1)
                check(o1[b, 4 * h:4 * h + 4], want, tol)
                check(w[b, h, :n], ww, wtol)


def test_results_do_not_change_between_runs(cuda_device):
    """No order of atomics or of blocks enters a result."""
    dev = cuda_device
    g = gen(dev, 51)
    q, k, v = randn(g, 40, 8, 128), randn(g, 9000, 2, 128), randn(g, 9000, 2, 128)
    cache = filled(dev, g, 2, 2, 6000, 128)
    q1, rows = randn(g, 2, 8, 128), torch.tensor([6000, 4321], dtype=torch.int64, device=dev)
    first = None
    for _ in range(5):
        o, o1, w = torch.zeros_like(q), torch.zeros_like(q1), torch.zeros(2, 2, 6000, device=dev)
        PromptAttentionOp(q, k, v, o, scaling=0.1).launch()
        Cache4AttentionOp(q1, None, None, cache, rows, o1, scaling=0.1, weights=w).launch()
        if first is None:
            first = (o, o1, w)
        assert all(torch.equal(a, b) for a, b in zip(first, (o, o1, w)))
