"""Measured cases of the attention operators: prompt attention, the 4-bit key/value cache (write, read, attention of one
new token) and eviction from it.

``run`` is either the plain form (elementary torch operations in 32 bits) or, with ``own`` set, the calls a user makes of
``rvq_b200.attention``.  ``exact`` is the operators' definition in 64 bits.

A cached token of one kv head is a record of bytes: K codes, V codes (two 4-bit codes a byte), K parameters, V
parameters (a bf16 zero and a bf16 step for each group of 32 values).  Within the codes of a row of D values, byte
16 w + 4 g + b (D = 128; 8 w + 4 g + b for D = 64) holds codes of group g, values 8 w + 2 b and 8 w + 2 b + 1 of it, the
first in the low half: code byte order [w in 0..3][g][b in 0..3].
"""

import math
import random

import numpy as np
import torch

own = False

GROUP = 32


# -- cases ------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # a short question to a small model: the launch is what it costs
        dict(name="prompt 24, 8/2 heads of 64", kind="prompt", seqs=1, longest=24, prefix=0, heads=8, kv=2, dim=64,
             causal=True, lse=False, dtype="bf16"),
        # an ordinary prompt at the 2560-wide block's heads
        dict(name="prompt 2048, 32/8 of 128", kind="prompt", seqs=1, longest=2048, prefix=0, heads=32, kv=8, dim=128,
             causal=True, lse=False, dtype="bf16"),
        # the longest prompt
        dict(name="prompt 16384, 32/8 of 128", kind="prompt", seqs=1, longest=16384, prefix=0, heads=32, kv=8, dim=128,
             causal=True, lse=False, dtype="bf16"),
        # several users' prompts in one call, lengths from one token on
        dict(name="prompt 12 packed to 1531", kind="prompt", seqs=12, longest=1531, prefix=0, heads=64, kv=8, dim=128,
             causal=True, lse=True, dtype="fp16"),
        # the next turn of a conversation: few new tokens over a long past
        dict(name="prompt 77 after 9000", kind="prompt", seqs=1, longest=77, prefix=9000, heads=32, kv=8, dim=128,
             causal=True, lse=False, dtype="bf16"),
        # a prompt put into the 4-bit cache and read back (as the next turn's attention does)
        dict(name="write and read 4096", kind="store", seqs=1, longest=4096, kv=8, dim=128, dtype="bf16"),
        dict(name="write and read 9 to 700 of 64", kind="store", seqs=9, longest=700, kv=2, dim=64, dtype="fp16"),
        # one token of one user, early in the answer
        dict(name="step 1 x 300", kind="step", seqs=1, longest=300, heads=32, kv=8, dim=128, weights=False, dtype="bf16"),
        # the same far into a long text, with the attention weights that eviction goes by
        dict(name="step 1 x 40000 weights", kind="step", seqs=1, longest=40000, heads=32, kv=8, dim=128, weights=True,
             dtype="bf16"),
        # many users at once
        dict(name="step 64 x 8191", kind="step", seqs=64, longest=8191, heads=64, kv=8, dim=128, weights=False,
             dtype="fp16"),
        # one layer's cache over its budget
        dict(name="evict 1 x 1100 to 1024", kind="evict", seqs=1, longest=1100, keep=1024, recent=64, kv=8, dim=128),
        # every layer of a 36-layer model at once
        dict(name="evict 36 x 8500 to 4096", kind="evict", seqs=36, longest=8500, keep=4096, recent=256, kv=8, dim=128),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["prompt", "prompt", "store", "step", "step", "evict"])
    kv = rng.choice([1, 2, 4, 8])
    dim = rng.choice([64, 128, 128])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "prompt":
        rep = rng.choice([1, 2, 3, 4, 5, 8])
        seqs = rng.choice([1, 1, 2, 5, 12])
        longest = _log(rng, 1, 8192 if seqs == 1 else 2000)
        prefix = rng.choice([0, 0, 0, _log(rng, 1, 8192)]) if longest <= 1024 else 0
        return dict(kind=kind, seqs=seqs, longest=longest, prefix=prefix, heads=rep * kv, kv=kv,
                    dim=rng.choice([dim, dim, dim, 80, 32]), causal=rng.random() < 0.75, lse=rng.random() < 0.5,
                    dtype=dtype)
    if kind == "store":
        return dict(kind=kind, seqs=rng.randint(1, 16), longest=_log(rng, 1, 6000), kv=kv, dim=dim, dtype=dtype)
    if kind == "step":
        seqs = _log(rng, 1, 64)
        return dict(kind=kind, seqs=seqs, longest=_log(rng, 1, 60000 if seqs == 1 else min(60000, 500000 // seqs)),
                    heads=rng.choice([1, 2, 3, 4, 6, 8, 12]) * kv, kv=kv, dim=dim, weights=rng.random() < 0.4, dtype=dtype)
    longest = _log(rng, 200, 9000)
    keep = rng.randint(100, longest)
    return dict(kind=kind, seqs=rng.randint(1, 36), longest=longest, keep=keep, recent=rng.randint(0, keep), kv=kv,
                dim=dim)


def _lengths(case, at_least=1):
    """The sequences' lengths: the longest, and others spread below it. They go by the case alone."""
    r = random.Random("%d %d" % (case["seqs"], case["longest"]))
    return [case["longest"]] + [r.randint(min(at_least, case["longest"]), case["longest"])
                                for _ in range(case["seqs"] - 1)]


def _evict_lengths(case):
    """Live rows: all over the budget but, where there are many, some under it."""
    lens = _lengths(case, case["keep"])
    return [min(n, case["keep"] - 1) if i % 9 == 7 else n for i, n in enumerate(lens)]


def _dtype(case):
    return torch.float16 if case.get("dtype") == "fp16" else torch.bfloat16


# -- inputs -----------------------------------------------------------------------------------------------------------
def _kv(gen, n, kv, dim, dtype):
    """Keys with a few strong channels, as rotated and normalised keys have; values without."""
    dev = gen.device
    k = torch.randn(n, kv, dim, generator=gen, device=dev)
    k = k * (1 + 3 * (torch.rand(kv, dim, generator=gen, device=dev) > 0.95)) \
        + 0.5 * torch.randn(kv, dim, generator=gen, device=dev)
    return k.to(dtype), torch.randn(n, kv, dim, generator=gen, device=dev).to(dtype)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(int(seed))
    kind, dt = case["kind"], _dtype(case)
    s = dict(case=case, kind=kind)
    if kind == "prompt":
        lq = _lengths(case)
        lk = [n + case["prefix"] for n in lq]
        s["lq"], s["lk"] = max(lq), max(lk)
        s["cu_q"] = torch.tensor(np.cumsum([0] + lq), dtype=torch.int32, device=dev)
        s["cu_k"] = torch.tensor(np.cumsum([0] + lk), dtype=torch.int32, device=dev)
        s["q"] = torch.randn(sum(lq), case["heads"], case["dim"], generator=gen, device=dev).to(dt)
        s["k"], s["v"] = _kv(gen, sum(lk), case["kv"], case["dim"], dt)
        s["scaling"] = case["dim"] ** -0.5
    elif kind == "store":
        lens = _lengths(case)
        s["max_len"] = case["longest"] + 8
        s["cu"] = torch.tensor(np.cumsum([0] + lens), dtype=torch.int32, device=dev)
        s["start"] = torch.tensor([i % 8 for i in range(len(lens))], dtype=torch.int64, device=dev)
        s["k"], s["v"] = _kv(gen, sum(lens), case["kv"], case["dim"], dt)
        s["data"] = torch.zeros(case["seqs"], case["kv"], s["max_len"], case["dim"] * 5 // 4, dtype=torch.uint8, device=dev)
    elif kind == "step":
        lens = _lengths(case)
        n, kv, dim = case["seqs"], case["kv"], case["dim"]
        s["max_len"] = case["longest"] + 1
        s["rows"] = torch.tensor(lens, dtype=torch.int64, device=dev)
        s["q"] = torch.randn(n, case["heads"], dim, generator=gen, device=dev).to(dt)
        s["k"], s["v"] = _kv(gen, n, kv, dim, dt)
        s["data"] = torch.zeros(n, kv, s["max_len"], dim * 5 // 4, dtype=torch.uint8, device=dev)
        for i in range(n):
            k, v = _kv(gen, s["max_len"], kv, dim, dt)
            s["data"][i] = _records(k, v).transpose(0, 1)
        s["weights"] = torch.rand(n, kv, s["max_len"], generator=gen, device=dev) if case["weights"] else None
        s["scaling"] = dim ** -0.5
    else:
        n, kv, dim = case["seqs"], case["kv"], case["dim"]
        s["max_len"] = case["longest"]
        s["rows"] = torch.tensor(_evict_lengths(case), dtype=torch.int64, device=dev)
        s["data"] = torch.randint(0, 256, (n, kv, s["max_len"], dim * 5 // 4), dtype=torch.uint8, generator=gen, device=dev)
        # a few rows hold most of the weight, some were never looked at
        w = torch.randn(n, kv, s["max_len"], generator=gen, device=dev).mul_(2).exp_()
        s["weights"] = w * (torch.rand(w.shape, generator=gen, device=dev) > 0.05)
    if own:
        s["ops"] = _own_ops(s)
    return s


def _own_ops(s):
    """The framework's operators, bound once to the buffers of a user's program."""
    from rvq_b200 import attention as A
    case, kind = s["case"], s["kind"]
    if kind == "prompt":
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(s["q"].shape[1], s["q"].shape[0], device=s["q"].device) if case["lse"] else None
        return [A.PromptAttentionOp(s["q"], s["k"], s["v"], s["out"], scaling=s["scaling"], causal=case["causal"],
                                    cu_q=s["cu_q"], cu_k=s["cu_k"], lse=s["lse"])]
    cache = A.Cache4(case["seqs"], case["kv"], s["max_len"], case["dim"], data=s["data"])
    if kind == "store":
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
        return [A.Cache4WriteOp(cache, s["k"], s["v"], cu=s["cu"], start=s["start"]),
                A.Cache4ReadOp(cache, s["k_out"], s["v_out"], cu=s["cu"], start=s["start"])]
    if kind == "step":
        s["out"], s["k_out"], s["v_out"] = torch.empty_like(s["q"]), torch.empty_like(s["k"]), torch.empty_like(s["v"])
        one = torch.arange(case["seqs"] + 1, dtype=torch.int32, device=s["q"].device)
        return [A.Cache4AttentionOp(s["q"], s["k"], s["v"], cache, s["rows"], s["out"], scaling=s["scaling"],
                                    weights=s["weights"]),
                A.Cache4ReadOp(cache, s["k_out"], s["v_out"], cu=one, start=s["rows"])]
    keep, shape = case["keep"], s["data"].shape
    s["data_out"] = torch.zeros(shape[0], shape[1], keep, shape[3], dtype=torch.uint8, device=s["data"].device)
    s["weights_out"] = torch.zeros(shape[0], shape[1], keep, device=s["data"].device)
    s["kept"] = torch.empty(shape[0], shape[1], keep, dtype=torch.int32, device=s["data"].device)
    s["new_rows"] = torch.empty_like(s["rows"])
    out = A.Cache4(case["seqs"], case["kv"], keep, case["dim"], data=s["data_out"])
    return [A.Cache4EvictOp(cache, s["weights"], s["rows"], keep=keep, recent=case["recent"], kept=s["kept"],
                            out=out, out_weights=s["weights_out"], new_rows=s["new_rows"])]


def run(state):
    if own:
        for op in state["ops"]:
            op.launch()
        return _own_outputs(state)
    return {"prompt": _plain_prompt, "store": _plain_store, "step": _plain_step, "evict": _plain_evict}[state["kind"]](state)


def _own_outputs(s):
    if s["kind"] == "prompt":
        return {"out": s["out"], "lse": s["lse"]}
    if s["kind"] == "store":
        return {"k": s["k_out"], "v": s["v_out"]}
    if s["kind"] == "step":
        return {"out": s["out"], "weights": s["weights"], "k": s["k_out"], "v": s["v_out"]}
    return {"kept": s["kept"], "rows": s["new_rows"], "weights": s["weights_out"], "records": s["data_out"]}


# -- the plain form ---------------------------------------------------------------------------------------------------
def _split(x, group=GROUP):
    return x.reshape(*x.shape[:-1], x.shape[-1] // group, group)


def _quantise(x):
    """[..., D] -> codes [..., G, 32] (float), zero and step [..., G] bf16."""
    g = _split(x.float())
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    zero, step = lo.bfloat16(), ((hi - lo) / torch.full_like(lo, 15)).bfloat16()      # a division, no product with 1 / 15
    c = torch.round((g - zero.float()) / step.float())
    c = torch.where(step > 0, c, torch.zeros_like(c)).clamp(0, 15)
    return c, zero.squeeze(-1), step.squeeze(-1)


def _values(c, zero, step):
    return (zero.float().unsqueeze(-1) + step.float().unsqueeze(-1) * c).flatten(-2)


def _bytes(c):
    """Codes [..., G, 32] -> [..., D / 2] bytes in record order."""
    c = c.to(torch.uint8).unflatten(-1, (4, 4, 2)).transpose(-3, -4)     # [..., w, g, b, 2] from [..., g, w, b, 2]
    return (c[..., 0] | (c[..., 1] << 4)).flatten(-3)


def _records(k, v):
    """[..., D] keys and values -> [..., 5 D / 4] bytes."""
    ck, zk, sk = _quantise(k)
    cv, zv, sv = _quantise(v)
    par = lambda z, s: torch.stack((z, s), -1).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat((_bytes(ck), _bytes(cv), par(zk, sk), par(zv, sv)), -1)


def _unpack(rec, dim):
    """[..., 5 D / 4] bytes -> keys and values [..., D] in 32 bits."""
    half, par = dim // 2, dim // 8

    def codes(b):
        b = b.unflatten(-1, (4, dim // GROUP, 4)).transpose(-2, -3)       # [..., g, w, b]
        return torch.stack((b & 15, b >> 4), -1).flatten(-3).float()

    def values(b, p):
        p = p.contiguous().view(torch.bfloat16).unflatten(-1, (dim // GROUP, 2))
        return _values(codes(b), p[..., 0], p[..., 1])

    k, v, pk, pv = rec.split((half, half, par, par), -1)
    return values(k, pk), values(v, pv)


def _padded(x, cu, longest, heads, dim):
    """Packed [T, H, D] -> [B, H, longest, D], zeros behind each sequence, and its lengths [B]."""
    start, n = cu[:-1].long(), (cu[1:] - cu[:-1]).long()
    at = torch.arange(longest, device=x.device)
    live = at < n[:, None]
    rows = torch.where(live, start[:, None] + at, torch.zeros_like(at))
    return torch.where(live[:, :, None, None], x[rows].float(), 0.0).transpose(1, 2), n, live


def _plain_prompt(s):
    case = s["case"]
    nh, nkv, dim = case["heads"], case["kv"], case["dim"]
    q, lq, live = _padded(s["q"], s["cu_q"], s["lq"], nh, dim)
    k, lk, _ = _padded(s["k"], s["cu_k"], s["lk"], nkv, dim)
    v, _, _ = _padded(s["v"], s["cu_k"], s["lk"], nkv, dim)
    b, rep = q.shape[0], nh // nkv
    i, j = torch.arange(s["lq"], device=q.device), torch.arange(s["lk"], device=q.device)
    limit = lk[:, None] - lq[:, None] + i + 1 if case["causal"] else lk[:, None].expand(b, s["lq"])
    hidden = j >= torch.minimum(limit, lk[:, None])[:, :, None]                        # [B, Lq, Lk]
    p = torch.matmul(q.reshape(b, nkv, rep * s["lq"], dim), k.transpose(-1, -2)).mul_(s["scaling"])
    p = p.view(b, nkv, rep, s["lq"], s["lk"]).masked_fill_(hidden[:, None, None], float("-inf"))
    top = p.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    p = p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p.view(b, nkv, rep * s["lq"], s["lk"]), v).view(b, nkv, rep, s["lq"], dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out)).view(b, nh, s["lq"], dim)
    lse = (top + torch.log(total)).view(b, nh, s["lq"])
    return {"out": out.transpose(1, 2)[live].to(s["q"].dtype),
            "lse": lse.transpose(0, 1)[:, live] if case["lse"] else None}


def _plain_store(s):
    t = s["k"].shape[0]
    at = torch.arange(t, device=s["k"].device)
    seq = torch.searchsorted(s["cu"][1:].long(), at, right=True)
    row = s["start"][seq] + at - s["cu"].long()[seq]
    s["data"][seq, :, row] = _records(s["k"], s["v"])
    k, v = _unpack(s["data"][seq, :, row], s["case"]["dim"])
    return {"k": k.to(s["k"].dtype), "v": v.to(s["v"].dtype)}


def _plain_step(s):
    case = s["case"]
    n, nh, nkv, dim = case["seqs"], case["heads"], case["kv"], case["dim"]
    seq, rows = torch.arange(n, device=s["q"].device), s["rows"]
    s["data"][seq, :, rows] = _records(s["k"], s["v"])
    k, v = _unpack(s["data"], dim)                                                    # [n, kv, max_len, D]
    j = torch.arange(s["max_len"], device=s["q"].device)
    p = torch.matmul(s["q"].float().view(n, nkv, nh // nkv, dim), k.transpose(-1, -2)).mul_(s["scaling"])
    p = p.masked_fill_((j > rows[:, None])[:, None, None], float("-inf"))
    p = (p - p.amax(-1, keepdim=True)).exp_()
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, v).view(n, nh, dim)
    if case["weights"]:
        w, new = p.sum(2), (j == rows[:, None])[:, None]
        s["weights"].copy_(torch.where(new, w, s["weights"] + w))
    new_k, new_v = _unpack(s["data"][seq, :, rows], dim)
    return {"out": out.to(s["q"].dtype), "weights": s["weights"], "k": new_k.to(s["k"].dtype), "v": new_v.to(s["v"].dtype)}


def _plain_evict(s):
    case = s["case"]
    keep, recent, rows, length = case["keep"], case["recent"], s["rows"], s["max_len"]
    j = torch.arange(length, device=rows.device)
    n = rows[:, None, None]
    # order: live rows before dead ones, recent ones first, then by weight; a stable sort leaves ties to the lowest row
    w = torch.where(j >= n - recent, float("inf"), s["weights"])
    w = torch.where(j >= n, float("-inf"), w)
    first = torch.sort(w, dim=-1, descending=True, stable=True).indices[..., :keep]
    count = rows.clamp(max=keep)
    slot = torch.arange(keep, device=rows.device)
    dead = (slot >= count[:, None, None]).expand(first.shape)
    first = torch.sort(torch.where(dead, length, first), dim=-1).values
    at = torch.where(dead, 0, first)
    records = torch.gather(s["data"], 2, at.unsqueeze(-1).expand(*at.shape, s["data"].shape[-1]))
    records = torch.where(dead.unsqueeze(-1), torch.zeros_like(records), records)
    weights = torch.where(dead, 0.0, torch.gather(s["weights"], 2, at))
    return {"kept": torch.where(dead, -1, first).int(), "rows": count, "weights": weights, "records": records}


# -- work -------------------------------------------------------------------------------------------------------------
def work(case):
    kind, kv, dim = case["kind"], case["kv"], case["dim"]
    if kind == "prompt":
        lq = _lengths(case)
        pairs = sum(n * (n + case["prefix"]) - (n * (n - 1) // 2 if case["causal"] else 0) for n in lq)
        tq, tk = sum(lq), sum(lq) + case["prefix"] * len(lq)
        return {"bytes": 2 * dim * (2 * tq * case["heads"] + 2 * tk * kv) + (4 * tq * case["heads"] if case["lse"] else 0),
                "flops": 4 * dim * case["heads"] * pairs}
    record = dim * 5 // 4
    if kind == "store":
        t = sum(_lengths(case))
        return {"bytes": t * kv * (8 * dim + 2 * record), "flops": t * kv * 2 * dim * 6}
    if kind == "step":
        n, t = case["seqs"], sum(_lengths(case))
        return {"bytes": t * kv * (record + (8 if case["weights"] else 0)) + n * 4 * dim * (case["heads"] + 2 * kv),
                "flops": 4 * dim * case["heads"] * (t + n)}
    lens = _evict_lengths(case)
    kept = sum(min(n, case["keep"]) for n in lens)
    return {"bytes": kv * (4 * sum(lens) + kept * (2 * record + 8)), "flops": kv * sum(lens)}


# -- the definition in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    def held(x):
        """What a [..., D] tensor's values are held as, computed in 64 bits."""
        parts = []
        for g in x.double().split(GROUP, -1):
            lo, hi = g.min(-1, keepdim=True).values, g.max(-1, keepdim=True).values
            zero, step = lo.to(torch.bfloat16).double(), ((hi - lo) / 15.0).to(torch.bfloat16).double()
            code = ((g - zero) / torch.where(step > 0, step, torch.ones_like(step))).round().clamp(0, 15)
            parts.append(zero + step * torch.where(step > 0, code, torch.zeros_like(code)))
        return torch.cat(parts, -1)

    def unpacked(rec, dim):
        """Bytes of [R, record] -> keys, values [R, D], by the record's description."""
        groups, half = dim // GROUP, dim // 2
        place = torch.tensor([(w * groups + g) * 4 + b for g in range(groups) for w in range(4) for b in range(4)],
                             device=rec.device)
        par = rec[:, 2 * half:].contiguous().view(torch.bfloat16).double().view(-1, 2, groups, 2)
        got = []
        for which in (0, 1):
            b = rec[:, which * half:(which + 1) * half][:, place].to(torch.int32)
            c = torch.stack((b % 16, b // 16), -1).double().view(-1, groups, GROUP)
            got.append((par[:, which, :, 0:1] + par[:, which, :, 1:2] * c).reshape(-1, dim))
        return got

    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "prompt":
        lq = _lengths(case)
        rep = case["heads"] // case["kv"]
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        lse = torch.zeros(case["heads"], s["q"].shape[0], dtype=torch.float64, device="cuda")
        q0 = k0 = 0
        for n in lq:
            m = n + case["prefix"]
            for h in range(case["heads"]):
                k, v = s["k"][k0:k0 + m, h // rep].double(), s["v"][k0:k0 + m, h // rep].double()
                for a in range(0, n, 4096):
                    e = min(n, a + 4096)
                    z = s["q"][q0 + a:q0 + e, h].double() @ k.T * s["scaling"]
                    if case["causal"]:
                        above = torch.arange(m, device="cuda")[None] > torch.arange(a, e, device="cuda")[:, None] + (m - n)
                        z[above] = float("-inf")
                    lse[h, q0 + a:q0 + e] = torch.logsumexp(z, 1)
                    out[q0 + a:q0 + e, h] = torch.softmax(z, 1) @ v
            q0, k0 = q0 + n, k0 + m
        return {"out": out, "lse": lse if case["lse"] else None}
    if kind == "store":
        return {"k": held(s["k"]), "v": held(s["v"])}
    if kind == "step":
        n, dim, rep = case["seqs"], case["dim"], case["heads"] // case["kv"]
        new_k, new_v = held(s["k"]), held(s["v"])
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        weights = s["weights"].double() if case["weights"] else None
        for b, m in enumerate(_lengths(case)):
            for g in range(case["kv"]):
                k, v = unpacked(s["data"][b, g, :m], dim)
                k, v = torch.cat((k, new_k[b, g:g + 1])), torch.cat((v, new_v[b, g:g + 1]))
                p = torch.softmax(s["q"][b, g * rep:(g + 1) * rep].double() @ k.T * s["scaling"], 1)
                out[b, g * rep:(g + 1) * rep] = p @ v
                if weights is not None:
                    weights[b, g, :m] += p.sum(0)[:m]
                    weights[b, g, m] = p.sum(0)[m]
        return {"out": out, "weights": weights, "k": new_k, "v": new_v}
    lens, w = _evict_lengths(case), s["weights"].double().cpu().numpy()
    weights = np.zeros((case["seqs"], case["kv"], case["keep"]))
    for b, m in enumerate(lens):
        old = max(0, m - case["recent"])
        for g in range(case["kv"]):
            rows = np.arange(m)
            if m > case["keep"]:
                best = np.lexsort((np.arange(old), -w[b, g, :old]))[:case["keep"] - case["recent"]]
                rows = np.concatenate((np.sort(best), np.arange(old, m)))
            weights[b, g, :len(rows)] = w[b, g, rows]
    return {"kept": None, "rows": None, "weights": torch.from_numpy(weights), "records": None}
