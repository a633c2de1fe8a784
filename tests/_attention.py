"""Plain implementations in 64 bits of the attention operators, and bounds on their kernels' errors."""

import torch

GROUP = 32


def half_step(dtype):
    """Largest relative error of one rounding to ``dtype``."""
    return torch.finfo(dtype).eps / 2


# -- the 4-bit record, in 32 bits as the definition says (the host divides as IEEE does) ---------------------------------
def quantise(x):
    """[..., D] -> codes [..., G, 32] (float), zero and step [..., G] (fp32 values of bf16 numbers)."""
    g = x.float().cpu().unflatten(-1, (-1, GROUP))
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    zero = lo.bfloat16().float()
    step = ((hi - lo) / torch.full_like(lo, 15.0)).bfloat16().float()
    c = torch.round((g - zero) / step)
    c = torch.where((step > 0) & (c > 0), c.clamp(max=15), torch.zeros_like(c))
    return c, zero.squeeze(-1), step.squeeze(-1)


def values(c, zero, step):
    return (zero.unsqueeze(-1) + step.unsqueeze(-1) * c).flatten(-2)


def held(x):
    """The values that x is held as (fp32)."""
    return values(*quantise(x)).to(x.device)


def records(k, v):
    """[..., D] keys and values -> [..., 5 D / 4] record bytes, placed value by value."""
    d = k.shape[-1]
    out = torch.zeros(*k.shape[:-1], d * 5 // 4, dtype=torch.uint8)
    groups = d // GROUP
    for which, x in enumerate((k, v)):
        c, zero, step = quantise(x)
        c = c.flatten(-2).to(torch.uint8)
        for i in range(d):
            byte = which * (d // 2) + (i % 32 // 8 * groups + i // 32) * 4 + i % 8 // 2
            out[..., byte] |= c[..., i] << (4 * (i % 2))
        par = torch.stack((zero, step), -1).bfloat16().flatten(-2).contiguous().view(torch.uint8)
        at = d + which * (d // 8)
        out[..., at:at + d // 8] = par
    return out.to(k.device)


def unpack(rec, d):
    """[..., 5 D / 4] record bytes -> codes, zeros and steps of K and of V ([..., G, 32] and [..., G], fp32)."""
    groups, got = d // GROUP, []
    for which in (0, 1):
        c = torch.stack([rec[..., which * (d // 2) + (i % 32 // 8 * groups + i // 32) * 4 + i % 8 // 2] >> (4 * (i % 2)) & 15
                         for i in range(d)], -1).float()
        at = d + which * (d // 8)
        par = rec[..., at:at + d // 8].contiguous().view(torch.bfloat16).float().unflatten(-1, (groups, 2))
        got.append((c.unflatten(-1, (groups, GROUP)), par[..., 0], par[..., 1]))
    return got


# -- attention of one sequence -----------------------------------------------------------------------------------------
def attend(q, k, v, scaling, causal):
    """q [lq, nh, hd], k, v [lk, nkv, hd] -> out [lq, nh, hd], lse [nh, lq] in 64 bits, and the bound on a kernel's error.

    The kernel's scores are fp32 sums of hd exact products: off by at most d = (hd + 8) 2^-24 scaling sum|q||k| (8 for
    the scaling and the subtraction of the maximum); exp adds a relative 2^-21.  A probability is so off by a relative
    e = 2 d + 2^-21, and by u more where it is rounded to the operand type (u half a step); numerator and denominator
    both are, each over fp32 sums of lk terms (2^-24 sqrt(lk) in practice, lk 2^-24 at most).  One more rounding of
    the result: |error| <= u |out| + (u + 2 e + 2 lk 2^-24) sum p |v|.  2^-24 more absolutely, for results near zero
    (16-bit subnormals and products below fp32's precision).  fp16 probabilities below 2^-14 round to multiples of 2^-24, by
    at most 2^-25; they are held 2^7 times as large, and the largest of a row is at least 1, as is the sum that divides
    them: 2^-32 sum |v| more."""
    u = half_step(q.dtype)
    rep = q.shape[1] // k.shape[1]
    lq, lk = q.shape[0], k.shape[0]
    qd, kd, vd = q.double().transpose(0, 1), k.double().transpose(0, 1).repeat_interleave(rep, 0), \
        v.double().transpose(0, 1).repeat_interleave(rep, 0)
    hidden = torch.zeros(lq, lk, dtype=torch.bool, device=q.device)
    if causal:
        hidden = torch.arange(lk, device=q.device)[None] > torch.arange(lq, device=q.device)[:, None] + (lk - lq)
    # what is not seen counts as nothing, whatever it holds
    s = (qd @ kd.transpose(1, 2) * scaling).masked_fill(hidden, float("-inf"))
    size = (qd.abs() @ kd.abs().transpose(1, 2) * abs(scaling)).masked_fill(hidden, 0.0)
    if lk == 0:
        return (torch.zeros_like(q, dtype=torch.float64), torch.full((q.shape[1], lq), float("-inf"),
                dtype=torch.float64, device=q.device), torch.zeros_like(q, dtype=torch.float64),
                torch.zeros(q.shape[1], lq, dtype=torch.float64, device=q.device))
    lse = torch.logsumexp(s, -1)
    p = torch.where(torch.isneginf(lse)[..., None], torch.zeros_like(s), torch.exp(s - lse[..., None]))
    p = p.masked_fill(hidden, 0.0)
    if bool(torch.isfinite(vd).all()):
        out, mag = p @ vd, p @ vd.abs()
    else:                                   # a hidden NaN or infinity counts as nothing, a seen one counts
        weigh = lambda x: torch.where(hidden[None, :, :, None], torch.zeros_like(x[:, None]), p[..., None] * x[:, None]).sum(2)
        out, mag = weigh(vd), weigh(vd.abs())
    d = (q.shape[2] + 8) * 2.0 ** -24 * size.amax(-1)
    e = 2 * d + 2.0 ** -21
    tol = u * out.abs() + (u + 2 * e + 2 * lk * 2.0 ** -24)[..., None] * mag + 2.0 ** -24
    if q.dtype == torch.float16:
        tol = tol + 2.0 ** -32 * vd.nan_to_num(0, 0, 0).abs().sum(1, keepdim=True)
    lse_tol = e + lk * 2.0 ** -24 + 2.0 ** -22 * lse.abs()
    return out.transpose(0, 1), lse, tol.transpose(0, 1), lse_tol


def attend_cache(q, rec, n, d, scaling):
    """One kv head's query heads q [rep, D] over the first n of the records [max_len, 5 D / 4]: out [rep, D],
    weights [n] (summed over the heads) in 64 bits, and the bounds on a kernel's errors.

    A kernel may work on the codes: a product with a value z + s c is a sum of terms of at most |z| + 32 s (a code with
    an offset of up to 16 and its correction).  Scores: d = (D + 16) 2^-23 scaling sum |q| (|z| + 32 s), the weights' relative error e =
    2 d + 2^-21.  Weights are multiplied in parts whose sum is within 2^-16 of p s, sums are in fp32: |error of out| <=
    u |out| + (2^-16 + 2 e + 2 n 2^-24) sum p (|z| + 32 s), and 2^-24 near zero."""
    (kc, kz, ks), (vc, vz, vs) = ([t.double() for t in part] for part in unpack(rec[:n], d))
    k, v = values(kc, kz, ks), values(vc, vz, vs)
    wide = lambda z, s: (z.abs() + 32 * s.abs()).repeat_interleave(GROUP, -1)
    qd = q.double()
    s = qd @ k.T * scaling
    p = torch.softmax(s, -1)
    e = 2 * (d + 16) * 2.0 ** -23 * abs(scaling) * (qd.abs() @ wide(kz, ks).T).amax(-1) + 2.0 ** -21
    out = p @ v
    tol = half_step(q.dtype) * out.abs() + (2.0 ** -16 + 2 * e + 2 * n * 2.0 ** -24)[:, None] * (p @ wide(vz, vs)) + 2.0 ** -24
    w = p.sum(0)
    return out, w, tol, (p * (2 * e + 2 * n * 2.0 ** -24 + 2.0 ** -20)[:, None]).sum(0)


# -- eviction ----------------------------------------------------------------------------------------------------------
def kept_rows(w, n, keep, recent):
    """Rows of one (sequence, kv head) that stay, ascending: w a list of floats of the n live rows."""
    if n <= keep:
        return list(range(max(n, 0)))
    old = n - recent
    key = lambda i: (0 if w[i] != w[i] else 1, -w[i] if w[i] == w[i] else 0.0, i)
    return sorted(sorted(range(old), key=key)[:keep - recent]) + list(range(old, n))
