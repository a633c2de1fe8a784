"""GPU: Qwen3Decoder with the fused prompt attention, the 4-bit cache and eviction."""

import pytest
import torch

from rvq_b200 import synthetic
from rvq_b200.decoder import Qwen3Decoder, rmsnorm, rotate_half
from tests import _attention as ref

pytestmark = pytest.mark.gpu

MID = synthetic.BlockShape(hidden=512, intermediate=1536, n_heads=8, n_kv_heads=2, head_dim=64)
QW = synthetic.BlockShape()


def setup(shape, n_layers, vocab, seed, n, dev):
    art = synthetic.make_model_artifact(shape, n_layers, vocab, seed=seed)
    cfg = synthetic.qwen3_config(shape, n_layers, vocab)
    return art, cfg, torch.randint(0, vocab, (n,), generator=torch.Generator().manual_seed(seed)).to(dev)


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape,n_layers,n", [(MID, 3, 1), (MID, 3, 40), (MID, 3, 300), (QW, 2, 200)])
def test_fused_prompt_logits(shape, n_layers, n, causal, cuda_device):
    """Against the engine's ops.  Those round scores and probabilities to bf16 (2^-8 each, and a score of size s moves its
    probability by s 2^-8), the fused ones only probabilities: logits agree as the other step implementations do (2e-2)."""
    art, cfg, prompt = setup(shape, n_layers, 2048, 5, n, cuda_device)
    a, b = (Qwen3Decoder(cfg, art, cuda_device, mode="dense", max_len=320, causal=causal, prompt_attention=how)
            for how in ("engine", "fused"))
    assert rel(b.prefill(prompt), a.prefill(prompt)) < 2e-2
    # the caches of the first layer are the same: its keys and values come before any attention
    assert torch.equal(a.k_cache[0], b.k_cache[0]) and torch.equal(a.v_cache[0], b.v_cache[0])


class HeldDecoder(Qwen3Decoder):
    """The PyTorch step over the values that another decoder's 4-bit cache holds (its own keys would differ by a bf16
    rounding here and there, and then by a whole step of 4 bits)."""

    def _attention(self, l, q, k, v, pos):
        d, L = self.dims, self.layers[l]
        T = q.shape[0]
        q = rmsnorm(q.view(T, d.n_heads, d.head_dim), L["self_attn.q_norm.weight"], d.eps)
        k = rmsnorm(k.view(T, d.n_kv, d.head_dim), L["self_attn.k_norm.weight"], d.eps)
        v = v.view(T, d.n_kv, d.head_dim)
        at = torch.arange(T, device=q.device) if pos is None else pos
        c, s = self.cos[at][:, None], self.sin[at][:, None]
        q, k = q * c + rotate_half(q) * s, k * c + rotate_half(k) * s
        if l == 0:
            self.first = (k, v)
        keys, vals = k, v
        if pos is not None:
            n = int(pos) + 1
            keys, vals = (ref.values(*part).transpose(0, 1) for part in ref.unpack(self.source.data[l, :, :n], d.head_dim))
        out, *_ = ref.attend(q, keys, vals, self.scaling, pos is None and self.causal)
        return out.to(q.dtype).reshape(T, d.n_heads * d.head_dim)


@pytest.mark.parametrize("mode", ["dense", "fused", "slot"])
@pytest.mark.parametrize("shape,n_layers", [(MID, 3), (QW, 2)])
def test_int4_cache_logits(shape, n_layers, mode, cuda_device):
    """Teacher-forced steps over the 4-bit cache against PyTorch ops over the values it holds.

    The two round to bf16 at the same 14 places a layer (norms, projections, rotation, attention, products, residuals) and
    may do so apart; a rounding's relative rms is 2^-8 / sqrt(12) = 1.1e-3, so the logits differ by about
    sqrt(2 14 layers) 1.1e-3 = 1.0e-2 for 3 layers; twice that is allowed, and the 1e-2 of the table GEMV's fp16 tables (2^-11
    relative to the largest of 8 terms) in fused mode."""
    art, cfg, prompt = setup(shape, n_layers, 2048, 7, 50, cuda_device)
    dec = Qwen3Decoder(cfg, art, cuda_device, mode=mode, max_len=96, causal=True, prompt_attention="fused", kv_cache="int4")
    want = HeldDecoder(cfg, art, cuda_device, mode="dense", max_len=96, causal=True, step_impl="torch")
    want.source = dec.cache4
    ids = torch.randint(0, 2048, (20,), generator=torch.Generator().manual_seed(1)).to(cuda_device)
    dec.capture()
    tol = 3e-2 if mode == "fused" else 2e-2
    with torch.inference_mode():
        assert rel(dec.prefill(prompt), want._forward(prompt, None)) < tol
        # the first layer's rows come before any attention: the prompt's keys and values, byte for byte
        assert torch.equal(dec.cache4.data[0, :, :50], ref.records(*want.first).transpose(0, 1))
        for i, t in enumerate(ids):
            got = dec.step(t.view(1), 50 + i).clone()
            assert rel(got, want._forward(t.view(1), torch.tensor([50 + i], device=cuda_device))) < tol, i
            rec = ref.records(*want.first)[0]
            if mode != "fused":                             # the projections are the same: but for a rounding of the norm
                assert float((dec.cache4.data[0, :, 50 + i] != rec).float().mean()) < 0.05
    dec.check_waits()


def test_budget_beyond_the_text_changes_nothing(cuda_device):
    art, cfg, prompt = setup(MID, 3, 2048, 9, 30, cuda_device)
    kw = dict(mode="fused", max_len=128, causal=True, kv_cache="int4")
    a = Qwen3Decoder(cfg, art, cuda_device, **kw)
    b = Qwen3Decoder(cfg, art, cuda_device, kv_budget=100, kv_slack=4, **kw)
    (ia, la), (ib, lb) = a.generate(prompt, 40, return_logits=True), b.generate(prompt, 40, return_logits=True)
    assert torch.equal(ia, ib) and all(torch.equal(x, y) for x, y in zip(la, lb))
    assert b._dropped == 0


def test_generation_with_a_budget(cuda_device):
    """Rows stay under budget + slack while positions run on; every eviction keeps what the definition says, record by
    record; a second generation with the same graph gives the same."""
    art, cfg, prompt = setup(MID, 3, 2048, 11, 50, cuda_device)
    budget, recent, slack = 40, 10, 8
    dec = Qwen3Decoder(cfg, art, cuda_device, mode="fused", max_len=64, causal=True, prompt_attention="fused",
                       kv_cache="int4", kv_budget=budget, kv_recent=recent, kv_slack=slack, max_positions=400)
    seen = []
    plain = dec._evict

    def evict(live):
        data, w = dec.cache4.data.clone(), dec.kv_weights.clone()
        plain(live)
        for l in range(3):
            for h in range(2):
                rows = ref.kept_rows(w[l, h, :live].tolist(), live, budget, recent)
                assert torch.equal(dec.cache4.data[l, h, :budget], data[l, h, rows])
                assert torch.equal(dec.kv_weights[l, h, :budget], w[l, h, rows])
        seen.append(live)

    dec._evict = evict
    ids = dec.generate(prompt, 150)
    assert seen[0] == 50 + slack and all(n == budget + slack for n in seen[1:]) and len(seen) == 149 // slack
    assert dec._dropped == sum(seen) - budget * len(seen)
    again = dec.generate(prompt, 150)
    assert torch.equal(ids, again)
    # a step's weights sum to the query heads of a kv head, over all its rows
    row = 149 + 50 - 1 - dec._dropped + 1
    dec.prefill(prompt)
    dec.step(prompt[:1], 50)
    total = dec.kv_weights[:, :, :51].double().sum(-1)
    assert float((total - 4).abs().max()) < 4 * (60 * 2.0 ** -24 + 2.0 ** -16)
    assert row <= 64


def test_a_full_cache_is_evicted_before_the_slack(cuda_device):
    art, cfg, prompt = setup(MID, 2, 2048, 13, 60, cuda_device)
    dec = Qwen3Decoder(cfg, art, cuda_device, mode="dense", max_len=64, causal=True, kv_cache="int4", kv_budget=32,
                       kv_slack=1000, max_positions=256)
    ids = dec.generate(prompt, 100)
    assert ids.numel() == 100 and dec._dropped > 0


def test_steps_below_the_budget_are_no_slack(cuda_device):
    """A text that passes the budget on its way: the first eviction is due kv_slack steps after that, as every later one."""
    art, cfg, prompt = setup(MID, 2, 2048, 19, 30, cuda_device)
    dec = Qwen3Decoder(cfg, art, cuda_device, mode="dense", max_len=64, causal=True, kv_cache="int4", kv_budget=40, kv_slack=8,
                       max_positions=256)
    seen, plain = [], dec._evict
    dec._evict = lambda live: (seen.append(live), plain(live))
    dec.generate(prompt, 60)
    assert seen == [48] * ((30 + 59 - 40) // 8)


def test_going_back_after_an_eviction(cuda_device):
    """A step may be taken again at one of the recent positions, with the same logits; at earlier ones, whose rows are not there any
    more, it is refused and changes nothing."""
    art, cfg, prompt = setup(MID, 2, 2048, 23, 60, cuda_device)
    dec = Qwen3Decoder(cfg, art, cuda_device, mode="dense", max_len=96, causal=True, kv_cache="int4", kv_budget=40, kv_recent=10,
                       kv_slack=4, max_positions=256)
    dec.prefill(prompt)
    for i in range(4):
        dec.step(prompt[i:i + 1], 60 + i)
    assert dec._dropped == 24                               # rows 30 to 39 are positions 54 to 63
    data, weights = dec.cache4.data.clone(), dec.kv_weights.clone()
    for pos in (53, 30, 24):
        with pytest.raises(ValueError):
            dec.step(prompt[:1], pos)
    assert torch.equal(dec.cache4.data, data) and torch.equal(dec.kv_weights, weights)
    first = dec.step(prompt[9:10], 54).clone()
    after = dec.step(prompt[10:11], 55).clone()
    assert torch.equal(dec.step(prompt[9:10], 54), first) and torch.equal(dec.step(prompt[10:11], 55), after)
    dec.prefill(prompt)
    dec.step(prompt[:1], 10)                                # without an eviction any position will do


def test_evictions_inside_and_outside_of_inference_mode(cuda_device):
    """The first eviction within a caller's inference mode, a later one without."""
    art, cfg, prompt = setup(MID, 2, 2048, 13, 34, cuda_device)
    dec = Qwen3Decoder(cfg, art, cuda_device, mode="dense", max_len=64, causal=True, kv_cache="int4", kv_budget=32, kv_slack=2,
                       max_positions=256)
    with torch.inference_mode():
        ids = dec.generate(prompt, 12)
    assert dec._dropped > 0
    assert torch.equal(ids, dec.generate(prompt, 12))


class HeldAfterEviction(HeldDecoder):
    """The same for a cache whose rows were evicted: position ``pos`` is row ``pos - dropped``, its key rotated at ``pos``."""

    def _attention(self, l, q, k, v, pos):
        if pos is None:
            return super()._attention(l, q, k, v, pos)
        d, L = self.dims, self.layers[l]
        q = rmsnorm(q.view(1, d.n_heads, d.head_dim), L["self_attn.q_norm.weight"], d.eps)
        q = q * self.cos[pos][:, None] + rotate_half(q) * self.sin[pos][:, None]
        n = int(pos) + 1 - self.dropped
        keys, vals = (ref.values(*part).transpose(0, 1) for part in ref.unpack(self.source.data[l, :, :n], d.head_dim))
        return ref.attend(q, keys, vals, self.scaling, False)[0].to(q.dtype).reshape(1, d.n_heads * d.head_dim)


def test_a_prompt_that_fills_the_cache(cuda_device):
    """A prompt of max_len tokens with a budget: evicted before the first step, without weights: the first rows and the recent
    ones stay.  The step's logits are those over the kept rows (tolerance: test_int4_cache_logits, 2 layers)."""
    art, cfg, prompt = setup(MID, 2, 2048, 17, 64, cuda_device)
    kw = dict(mode="dense", max_len=64, causal=True, kv_cache="int4", kv_budget=32, kv_recent=10, max_positions=256)
    dec = Qwen3Decoder(cfg, art, cuda_device, **kw)
    want = HeldAfterEviction(cfg, art, cuda_device, mode="dense", max_len=256, causal=True, step_impl="torch")
    want.source, want.dropped = dec.cache4, 32
    dec.capture()
    dec.prefill(prompt)
    data = dec.cache4.data.clone()
    with pytest.raises(ValueError):
        dec.step(prompt[:1], 256)
    assert dec._dropped == 0 and torch.equal(dec.cache4.data, data)
    with torch.inference_mode():
        for i in range(3):
            got = dec.step(prompt[i:i + 1], 64 + i).clone()
            assert rel(got, want._forward(prompt[i:i + 1], torch.tensor([64 + i], device=cuda_device))) < 2e-2, i
    assert dec._dropped == 32
    assert torch.equal(dec.cache4.data[:, :, :32], data[:, :, list(range(22)) + list(range(54, 64))])
    ids = dec.generate(prompt, 100)
    assert ids.numel() == 100 and torch.equal(ids, dec.generate(prompt, 100))
    full = Qwen3Decoder(cfg, art, cuda_device, **{**kw, "max_positions": None})
    full.prefill(prompt)
    with pytest.raises(ValueError):                         # no position is left
        full.step(prompt[:1], 64)


def test_refusals(cuda_device):
    art, cfg, prompt = setup(MID, 2, 2048, 13, 60, cuda_device)
    make = lambda **kw: Qwen3Decoder(cfg, art, cuda_device, **kw)
    for kw in (dict(prompt_attention="other"), dict(kv_cache="int8"), dict(kv_budget=10), dict(kv_cache="int4", kv_budget=512),
               dict(kv_cache="int4", kv_budget=10, kv_recent=11), dict(kv_cache="int4", kv_recent=3),
               dict(kv_cache="int4", kv_budget=10, kv_slack=0), dict(max_positions=100), dict(kv_cache="int4", max_positions=1000)):
        with pytest.raises(ValueError):
            make(**kw)
    for kw in (dict(kv_cache="int4", step_impl="torch"), dict(kv_cache="int4", step_impl="persistent")):
        with pytest.raises(NotImplementedError):
            make(**kw)
    tiny = synthetic.qwen3_config(synthetic.BlockShape(hidden=64, intermediate=128, n_heads=4, n_kv_heads=2, head_dim=16), 2, 256)
    with pytest.raises(NotImplementedError):
        Qwen3Decoder(tiny, art, cuda_device, kv_cache="int4")
    dec = make(mode="dense", max_len=64, kv_cache="int4", kv_budget=32, max_positions=80)
    dec.prefill(prompt)
    with pytest.raises(ValueError):
        dec.step(prompt[:1], 64)                            # no row left: nothing was evicted yet
    with pytest.raises(ValueError):
        dec.step(prompt[:1], 80)
    with pytest.raises(ValueError):
        dec.step(prompt[:1], -1)
