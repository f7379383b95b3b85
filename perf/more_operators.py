"""Operators of a training step on packed sequences, as a program that fine-tunes a language model calls them.

* ``attention`` / ``attention_grad``: attention of whole prompts that lie one behind the other in the rows of one tensor, grouped
  heads, and the gradients of queries, keys and values.
* ``norm_grad``: the backward half of layer norm and RMS norm, with the sums over all rows that the weights' gradients are.
* ``policy_loss``: the clipped policy loss with a KL term on log probabilities of tokens, and its gradient.

``own`` chooses between elementary torch operations in 32 bits and this package's kernels (``metalhlo_b200.cuda``).
"""
from __future__ import annotations

import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # the prompt of one GPT-2 sequence: latency
        dict(name="attention_1x201_q12_kv12_d64_f16", kind="attention", dt="f16", seqs=1, length=201, ragged=False, q_heads=12, kv_heads=12, head_dim=64,
             causal=True),
        # a batch of prompts between 512 and 2048 tokens, packed, grouped heads
        dict(name="attention_24x2048_q32_kv8_d128_bf16", kind="attention", dt="bf16", seqs=24, length=2048, ragged=True, q_heads=32, kv_heads=8,
             head_dim=128, causal=True),
        # one long document
        dict(name="attention_1x16384_q32_kv8_d128_bf16", kind="attention", dt="bf16", seqs=1, length=16384, ragged=False, q_heads=32, kv_heads=8,
             head_dim=128, causal=True),
        # short sequences in fp32, as in a check of gradients or a small model's training
        dict(name="attention_9x500_q12_kv12_d64_f32", kind="attention", dt="f32", seqs=9, length=500, ragged=True, q_heads=12, kv_heads=12, head_dim=64,
             causal=True),
        # the backward half of the benchmark's GPT-2 batch
        dict(name="attention_grad_32x1024_q12_kv12_d64_f16", kind="attention_grad", dt="f16", seqs=32, length=1024, ragged=False, q_heads=12, kv_heads=12,
             head_dim=64, causal=True),
        # long sequences of unequal length
        dict(name="attention_grad_3x8192_q32_kv8_d128_bf16", kind="attention_grad", dt="bf16", seqs=3, length=8192, ragged=True, q_heads=32, kv_heads=8,
             head_dim=128, causal=True),
        # few short sequences in fp32, seven query heads to a head of keys
        dict(name="attention_grad_5x333_q14_kv2_d64_f32", kind="attention_grad", dt="f32", seqs=5, length=333, ragged=True, q_heads=14, kv_heads=2,
             head_dim=64, causal=True),
        # the norms of a large batch, the gradient of the residual stream added on the way
        dict(name="layer_norm_grad_32768x4096_bf16", kind="norm_grad", dt="bf16", rows=32768, hidden=4096, rms=False, residual=True),
        # a width that is no multiple of anything
        dict(name="layer_norm_grad_1021x769_f16", kind="norm_grad", dt="f16", rows=1021, hidden=769, rms=False, residual=False),
        # a wide RMS norm in fp32
        dict(name="rms_norm_grad_4096x5120_f32", kind="norm_grad", dt="f32", rows=4096, hidden=5120, rms=True, residual=False),
        # a step on a few answers: latency
        dict(name="policy_loss_8x500", kind="policy_loss", seqs=8, length=500, ragged=True, ref=True, per_sequence=True),
        # all answers of a large batch at once
        dict(name="policy_loss_700x2048", kind="policy_loss", seqs=700, length=2048, ragged=True, ref=True, per_sequence=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attention", "attention", "attention_grad", "attention_grad", "norm_grad", "policy_loss"])
    if kind in ("attention", "attention_grad"):
        kv_heads, group = rng.choice([(12, 1), (8, 4), (1, 8), (4, 1), (2, 16), (4, 7), (16, 1), (5, 3)])
        c = dict(kind=kind, dt=rng.choice(["bf16", "bf16", "f16", "f32"]), q_heads=kv_heads * group, kv_heads=kv_heads,
                 head_dim=rng.choice([64, 64, 80, 96, 128, 128]), ragged=rng.random() < 0.6, causal=rng.random() < 0.8)
        grad, f32 = kind == "attention_grad", c["dt"] == "f32"
        c["length"] = _log_int(rng, 1, 1024 if f32 else 8192 if grad else 16384)
        # pairs of a query and a key times elements of a head: no more than the largest listed case, a 32nd of that in fp32
        most = (1.1e12 if grad else 5.4e11) / (32 if f32 else 1) / (c["q_heads"] * c["head_dim"])
        rows = 2.5e8 / ((c["q_heads"] + 2 * kv_heads) * c["head_dim"])
        c["seqs"] = _log_int(rng, 1, max(1, min(64, int(most / c["length"] ** 2 * (2 if c["causal"] else 1)), int(rows / c["length"]))))
        while c["length"] ** 2 * c["seqs"] > most * (2 if c["causal"] else 1):
            c["length"] = c["length"] * 3 // 4
        return c
    if kind == "norm_grad":
        dt = rng.choice(["bf16", "f16", "f32"])
        hidden = _log_int(rng, 64, 12288)
        hidden = rng.choice([hidden, hidden | 1, -(-hidden // 64) * 64, -(-hidden // 64) * 64])
        return dict(kind=kind, dt=dt, rows=_log_int(rng, 1, 32768 * 4096 * 2 // (hidden * SIZE[dt])), hidden=hidden, rms=rng.random() < 0.5,
                    residual=rng.random() < 0.5)
    length = _log_int(rng, 1, 16384)
    return dict(kind=kind, seqs=_log_int(rng, 1, max(1, min(4096, 700 * 2048 // length))), length=length, ragged=rng.random() < 0.7, ref=rng.random() < 0.6,
                per_sequence=rng.random() < 0.5)


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _lengths(c):
    """Tokens per sequence: equal ones, or spread from a quarter to all of the case's length. They belong to the case, so that
    results of every seed have one shape."""
    if not c["ragged"]:
        return [c["length"]] * c["seqs"]
    u = torch.rand(c["seqs"], generator=torch.Generator().manual_seed(c["length"] * 8209 + c["seqs"])).tolist()
    return [c["length"]] + [max(1, round(c["length"] * (0.25 + 0.75 * x))) for x in u[1:]]


def _starts(c):
    starts = [0]
    for n in _lengths(c):
        starts.append(starts[-1] + n)
    return starts


def _attention_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    starts, d, dt, hq, hkv = _starts(c), c["head_dim"], TORCH[c["dt"]], c["q_heads"], c["kv_heads"]
    # queries, keys and values side by side in the rows of one projection
    qkv = torch.randn(starts[-1], hq + 2 * hkv, d, generator=g, device="cuda")
    qkv[:, :hq] *= 1.5
    qkv = qkv.to(dt)
    s = dict(case=c, starts_host=starts, starts=torch.tensor(starts, dtype=torch.int32).cuda(), scale=1.0 / math.sqrt(d), q=qkv[:, :hq],
             k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:])
    if c["kind"] == "attention_grad":
        s["grad"] = (torch.randn(starts[-1], hq, d, generator=g, device="cuda") * 1e-2).to(dt)
        s["out"], s["lse"] = _attention_plain(s)  # what the forward half leaves
        d_qkv = torch.empty_like(qkv)  # the gradient of that projection's result
        s["grads"] = d_qkv[:, :hq], d_qkv[:, hq:hq + hkv], d_qkv[:, hq + hkv:]
    return s


def _norm_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt, shape = TORCH[c["dt"]], (c["rows"], c["hidden"])
    s = dict(case=c, eps=1e-5, x=(torch.randn(shape, generator=g, device="cuda") * 1.5 + 0.25).to(dt),
             grad=(torch.randn(shape, generator=g, device="cuda") * 1e-2).to(dt),
             gamma=(1 + 0.1 * torch.randn(c["hidden"], generator=g, device="cuda")).to(dt), residual=None)
    if c["residual"]:
        s["residual"] = (torch.randn(shape, generator=g, device="cuda") * 1e-2).to(dt)
    return s


def _policy_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    starts = _starts(c)
    n = starts[-1]
    rand = lambda: torch.rand(n, generator=g, device="cuda")  # noqa: E731
    new = torch.log(rand().clamp_min_(1e-6)) * 1.5  # log probabilities of sampled tokens: many near 0, some far below
    near = lambda width: (new + width * torch.randn(n, generator=g, device="cuda")).clamp_max_(0.0)  # noqa: E731
    # the first tokens of a sequence are its prompt, which takes no part
    position = torch.cat([torch.arange(m) / m for m in _lengths(c)]).cuda()
    seq = torch.repeat_interleave(torch.arange(c["seqs"]), torch.tensor(_lengths(c))).cuda()
    return dict(case=c, new=new, old=near(0.15), ref=near(0.3) if c["ref"] else None, mask=position >= 0.3 * rand()[:1],
                advantages=torch.randn(c["seqs"], generator=g, device="cuda")[seq], starts=torch.tensor(starts, dtype=torch.int32).cuda(), seq=seq,
                clip_low=0.2, clip_high=0.28, kl_weight=0.05 if c["ref"] else 0.0)


def prepare(case, seed):
    kind = case["kind"]
    if kind == "norm_grad":
        return _norm_inputs(case, seed)
    if kind == "policy_loss":
        return _policy_inputs(case, seed)
    s = _attention_inputs(case, seed)
    if own:  # how the sequences of a batch are cut into tiles: the same for all layers, forward and backward
        from metalhlo_b200 import cuda

        s["plan"] = cuda.packed_plan(s["starts"], s["q"].shape[0], case["q_heads"], case["kv_heads"], causal=case["causal"])
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)[state["case"]["kind"]](state)


def _attention_own(s):
    from metalhlo_b200 import cuda

    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=s["q"].device)
    return cuda.packed_attention(s["q"], s["k"], s["v"], s["plan"], s["scale"], lse=lse), lse


def _attention_grad_own(s):
    from metalhlo_b200 import cuda

    dq, dk, dv = s["grads"]
    return cuda.packed_attention_grad(s["q"], s["k"], s["v"], s["out"], s["lse"], s["grad"], s["plan"], s["scale"], dq=dq, dk=dk, dv=dv)


def _norm_grad_own(s):
    from metalhlo_b200 import cuda

    f = cuda.rms_norm_grad if s["case"]["rms"] else cuda.layer_norm_grad
    return f(s["x"], s["gamma"], s["grad"], eps=s["eps"], residual_grad=s["residual"])


def _policy_loss_own(s):
    from metalhlo_b200 import cuda

    r = cuda.policy_loss(s["new"], s["old"], s["advantages"], mask=s["mask"], ref_logprobs=s["ref"], starts=s["starts"] if s["case"]["per_sequence"] else None,
                         clip_low=s["clip_low"], clip_high=s["clip_high"], kl_weight=s["kl_weight"])
    return r.loss, r.grad, r.kl, r.clip_fraction


def _rows_of(x, s, i):
    """Rows of sequence i in 32 bits, heads first: [heads, tokens, head_dim]."""
    return x[s["starts_host"][i]:s["starts_host"][i + 1]].float().transpose(0, 1)


def _scores(s, i):
    """(q [kv_heads, group n, head_dim], scores [kv_heads, group n, n]) of sequence i."""
    c = s["case"]
    q, k = _rows_of(s["q"], s, i), _rows_of(s["k"], s, i)
    n = q.shape[1]
    q = q.reshape(c["kv_heads"], -1, c["head_dim"])
    z = torch.matmul(q, k.transpose(1, 2)).mul_(s["scale"])
    if c["causal"]:
        hidden = torch.ones(n, n, dtype=torch.bool, device=q.device).triu_(1)
        z.view(c["q_heads"], n, n).masked_fill_(hidden, -math.inf)
    return q, z


def _attention_plain(s):
    c = s["case"]
    o = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=s["q"].device)
    lse = torch.empty(s["q"].shape[:2], dtype=torch.float32, device=s["q"].device)
    for i in range(c["seqs"]):
        rows = slice(s["starts_host"][i], s["starts_host"][i + 1])
        _, z = _scores(s, i)
        m = z.amax(-1, keepdim=True)
        p = z.sub_(m).exp_()
        total = p.sum(-1, keepdim=True)
        out = torch.matmul(p, _rows_of(s["v"], s, i)) / total
        o[rows] = out.view(c["q_heads"], -1, c["head_dim"]).transpose(0, 1).to(o.dtype)
        lse[rows] = (m + torch.log(total)).view(c["q_heads"], -1).t()
    return o, lse


def _attention_grad_plain(s):
    c = s["case"]
    for i in range(c["seqs"]):
        rows = slice(s["starts_host"][i], s["starts_host"][i + 1])
        q, z = _scores(s, i)
        n, d = z.shape[-1], c["head_dim"]
        p = z.sub_(s["lse"][rows].t().reshape(c["kv_heads"], -1, 1)).exp_()
        do = _rows_of(s["grad"], s, i).reshape(c["kv_heads"], -1, d)
        dv = torch.matmul(p.transpose(1, 2), do)
        dp = torch.matmul(do, _rows_of(s["v"], s, i).transpose(1, 2))
        ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
        dq = torch.matmul(ds, _rows_of(s["k"], s, i)).view(c["q_heads"], n, d)
        dk = torch.matmul(ds.transpose(1, 2), q)
        for to, x in zip(s["grads"], (dq, dk, dv)):
            to[rows] = x.transpose(0, 1).to(to.dtype)
    return s["grads"]


def _norm_grad_plain(s):
    c = s["case"]
    x, dy, gamma = s["x"].float(), s["grad"].float(), s["gamma"].float()
    mean = 0.0 if c["rms"] else x.mean(1, keepdim=True)
    r = torch.rsqrt((x - mean).square().mean(1, keepdim=True) + s["eps"])
    y = (x - mean) * r
    t = dy * gamma
    dx = t - y * (t * y).mean(1, keepdim=True)
    if not c["rms"]:
        dx = dx - t.mean(1, keepdim=True)
    dx = dx * r
    if s["residual"] is not None:
        dx = dx + s["residual"].float()
    out = dx.to(s["x"].dtype), (dy * y).sum(0)
    return out if c["rms"] else out + (dy.sum(0),)


def _policy_loss_plain(s):
    c = s["case"]
    new, old, a = s["new"].double(), s["old"].double(), s["advantages"].double()  # in 64 bits: ratios next to the clip's borders, long sums
    mask = s["mask"].double()
    if c["per_sequence"]:
        counts = torch.zeros(c["seqs"], dtype=torch.float64, device=new.device).index_add_(0, s["seq"], mask)
        w = mask / (counts.clamp_min(1.0) * (counts > 0).sum())[s["seq"]]
    else:
        w = mask / mask.sum().clamp_min(1.0)
    ratio = torch.exp(new - old)
    clipped = ((a > 0) & (ratio > 1 + s["clip_high"])) | ((a < 0) & (ratio < 1 - s["clip_low"]))
    loss = -torch.minimum(ratio * a, ratio.clamp(1 - s["clip_low"], 1 + s["clip_high"]) * a)
    grad = torch.where(clipped, 0.0, -ratio * a)
    kl = None
    if s["ref"] is not None:
        x = s["ref"].double() - new
        k3 = torch.exp(x) - x - 1
        loss, grad, kl = loss + s["kl_weight"] * k3, grad + s["kl_weight"] * (1 - torch.exp(x)), (w * k3).sum().float()
    return (w * loss).sum().float(), (w * grad).float(), kl, (w * clipped).sum().float()


_run_own = {"attention": _attention_own, "attention_grad": _attention_grad_own, "norm_grad": _norm_grad_own, "policy_loss": _policy_loss_own}
_run_plain = {"attention": _attention_plain, "attention_grad": _attention_grad_plain, "norm_grad": _norm_grad_plain, "policy_loss": _policy_loss_plain}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] == "norm_grad":
        cells, es = c["rows"] * c["hidden"], SIZE[c["dt"]]
        return {"bytes": (4 if c["residual"] else 3) * cells * es + c["hidden"] * (es + (4 if c["rms"] else 8)), "flops": (12 if c["rms"] else 16) * cells}
    lengths = _lengths(c)
    tokens = sum(lengths)
    if c["kind"] == "policy_loss":
        return {"bytes": tokens * (4 * (5 if c["ref"] else 4) + 1) + 16, "flops": tokens * (40 if c["ref"] else 20)}
    d, es = c["head_dim"], SIZE[c["dt"]]
    pairs = sum(n * (n + 1) // 2 if c["causal"] else n * n for n in lengths)
    q, kv = tokens * c["q_heads"] * d * es, tokens * c["kv_heads"] * d * es
    lse = 4 * tokens * c["q_heads"]
    if c["kind"] == "attention":
        return {"bytes": 2 * q + 2 * kv + lse, "flops": 4 * pairs * c["q_heads"] * d}
    return {"bytes": 4 * q + 4 * kv + lse, "flops": 10 * pairs * c["q_heads"] * d}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    return _exact[case["kind"]](case, seed)


def _exact_blocks(c, s):
    """Blocks of query rows with all that they see, in 64 bits: (rows, key rows, q head, kv head, q, k, v, log weights)."""
    group = c["q_heads"] // c["kv_heads"]
    for first, end in zip(s["starts_host"], s["starts_host"][1:]):
        for h in range(c["q_heads"]):
            k, v = (s[x][first:end, h // group].double() for x in "kv")
            for a in range(first, end, 4096):
                b = min(end, a + 4096)
                seen = slice(0, b - first) if c["causal"] else slice(0, end - first)
                q = s["q"][a:b, h].double()
                z = torch.einsum("id,jd->ij", q, k[seen]) * s["scale"]
                if c["causal"]:
                    z = torch.where(torch.arange(a - first, b - first, device="cuda")[:, None] >= torch.arange(b - first, device="cuda")[None], z, -math.inf)
                yield slice(a, b), slice(first, first + z.shape[1]), h, h // group, q, k[seen], v[seen], z


def _exact_attention(c, seed):
    s = _attention_inputs(c, seed)
    o, lse = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda"), torch.empty(s["q"].shape[:2], dtype=torch.float64, device="cuda")
    for rows, _, h, _, _, _, v, z in _exact_blocks(c, s):
        lse[rows, h] = torch.logsumexp(z, 1)
        o[rows, h] = torch.softmax(z, 1) @ v
    return o, lse


def _exact_attention_grad(c, seed):
    s = _attention_inputs(c, seed)
    dq, dk, dv = (torch.zeros(s[x].shape, dtype=torch.float64, device="cuda") for x in "qkv")
    for rows, keys, h, kv, q, k, v, z in _exact_blocks(c, s):
        p, do = torch.softmax(z, 1), s["grad"][rows, h].double()
        dv[keys, kv] += torch.einsum("ij,id->jd", p, do)
        dp = torch.einsum("id,jd->ij", do, v)
        dz = p * (dp - torch.einsum("ij,ij->i", p, dp)[:, None]) * s["scale"]
        dq[rows, h] = torch.einsum("ij,jd->id", dz, k)
        dk[keys, kv] += torch.einsum("ij,id->jd", dz, q)
    return dq, dk, dv


def _exact_norm_grad(c, seed):
    s = _norm_inputs(c, seed)
    outs, dgamma, dbeta = [], 0.0, 0.0
    for a in range(0, c["rows"], 4096):
        rows = slice(a, min(c["rows"], a + 4096))
        x, g = s["x"][rows].double(), s["grad"][rows].double()
        centred = x if c["rms"] else x - x.mean(1, keepdim=True)
        norm = torch.sqrt(torch.mean(centred ** 2, 1, keepdim=True) + s["eps"])
        dgamma, dbeta = dgamma + torch.sum(g * centred / norm, 0), dbeta + torch.sum(g, 0)
        g = g * s["gamma"].double()
        # derivative of centred / norm, then of the mean that was taken off
        dx = g / norm - centred * torch.mean(g * centred, 1, keepdim=True) / norm ** 3
        if not c["rms"]:
            dx = dx - dx.mean(1, keepdim=True)
        outs.append(dx if s["residual"] is None else dx + s["residual"][rows].double())
    return (torch.cat(outs), dgamma) if c["rms"] else (torch.cat(outs), dgamma, dbeta)


def _exact_policy_loss(c, seed):
    s = _policy_inputs(c, seed)
    d = s["new"].double() - s["old"].double()
    a, kept = s["advantages"].double(), torch.nonzero(s["mask"])[:, 0]
    w = torch.zeros_like(d)
    if c["per_sequence"]:
        of = s["seq"][kept]
        sizes = torch.bincount(of, minlength=c["seqs"])
        w[kept] = 1.0 / sizes[of].double() / torch.count_nonzero(sizes)
    else:
        w[kept] = 1.0 / max(1, kept.numel())
    low, high = math.log1p(-s["clip_low"]), math.log1p(s["clip_high"])
    out_of = torch.where(a > 0, d > high, (a < 0) & (d < low))
    held = torch.where(out_of, torch.where(a > 0, torch.full_like(d, high), torch.full_like(d, low)), d)
    loss = -a * torch.exp(held)
    grad = torch.where(out_of, torch.zeros_like(d), loss)
    kl = None
    if s["ref"] is not None:
        x = s["ref"].double() - s["new"].double()
        k3 = torch.expm1(x) - x
        loss, grad, kl = loss + s["kl_weight"] * k3, grad - s["kl_weight"] * torch.expm1(x), torch.dot(w, k3)
    return torch.dot(w, loss), w * grad, kl, w[out_of].sum()


_exact = {"attention": _exact_attention, "attention_grad": _exact_attention_grad, "norm_grad": _exact_norm_grad, "policy_loss": _exact_policy_loss}
