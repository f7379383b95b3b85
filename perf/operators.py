"""Operators around a key/value cache and the logits of a language model, as a serving or training program calls them.

* ``append``: keys and values of new tokens are rotated by their positions and put into a paged cache of 8-bit codes with one
  scale per page and head; the queries of the same tokens are rotated beside them. What the call wrote is read back as the
  values that the codes stand for.
* ``attend``: attention of the newest tokens of each sequence over such a cache, for single tokens and for chunks.
* ``logprobs`` / ``logprobs_grad``: log probabilities of given tokens, entropy, the most likely alternatives, and the gradient.

``own`` chooses between elementary torch operations in 32 bits and this package's kernels (``metalhlo_b200.cuda``).
"""
from __future__ import annotations

import math

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
VOCAB = 50257  # the GPT-2 vocabulary of the benchmark


# ---- the cases -------------------------------------------------------------------------------------------------------

def listed():
    return [
        # one decoding step of 64 conversations: a token each, grouped heads, contexts of every fill of their last page
        dict(name="append_64x1_q32_kv8_d128_bf16", kind="append", dt="bf16", seqs=64, new=1, ragged=False, context=256, q_heads=32, kv_heads=8,
             head_dim=128, page=64, interleaved=False),
        # five prompts of unequal length, 8192 tokens in all at most
        dict(name="append_5x1638_q32_kv8_d128_bf16", kind="append", dt="bf16", seqs=5, new=1638, ragged=True, context=0, q_heads=32, kv_heads=8,
             head_dim=128, page=64, interleaved=False),
        # the rest of one GPT-2 prompt behind a short prefix that ends inside a page
        dict(name="append_1x987_q12_kv12_d64_f16", kind="append", dt="f16", seqs=1, new=987, ragged=False, context=37, q_heads=12, kv_heads=12,
             head_dim=64, page=16, interleaved=True),
        # the next token of one GPT-2 sequence: latency
        dict(name="attend_1x1_201_q12_kv12_d64_f16", kind="attend", dt="f16", seqs=1, new=1, ragged=False, context=200, q_heads=12, kv_heads=12,
             head_dim=64, page=16),
        # a decoding step of 32 conversations of very different length
        dict(name="attend_32x1_4096_q32_kv8_d128_bf16", kind="attend", dt="bf16", seqs=32, new=1, ragged=True, context=4095, q_heads=32, kv_heads=8,
             head_dim=128, page=64),
        # the largest decoding step: a gigabyte of codes
        dict(name="attend_64x1_8192_q32_kv8_d128_bf16", kind="attend", dt="bf16", seqs=64, new=1, ragged=False, context=8191, q_heads=32, kv_heads=8,
             head_dim=128, page=64),
        # drafted tokens checked five at a time, in fp32
        dict(name="attend_8x5_1000_q12_kv12_d64_f32", kind="attend", dt="f32", seqs=8, new=5, ragged=True, context=995, q_heads=12, kv_heads=12,
             head_dim=64, page=32),
        # a chunk of 512 prompt tokens each on top of long contexts
        dict(name="attend_4x512_8192_q32_kv8_d128_bf16", kind="attend", dt="bf16", seqs=4, new=512, ragged=True, context=7680, q_heads=32, kv_heads=8,
             head_dim=128, page=64),
        # the answers of a small decoding batch: chosen token, entropy and five alternatives
        dict(name="logprobs_8x50257_f16_top5", kind="logprobs", dt="f16", rows=8, vocab=VOCAB, top=5, scale=1.0),
        # scoring a batch of sequences (evaluation, policy gradients): no alternatives
        dict(name="logprobs_4096x50257_bf16", kind="logprobs", dt="bf16", rows=4096, vocab=VOCAB, top=0, scale=1.0),
        # scored prompts with twenty alternatives each, logits in fp32, at a temperature
        dict(name="logprobs_1021x32000_f32_top20", kind="logprobs", dt="f32", rows=1021, vocab=32000, top=20, scale=1.25),
        # the backward half of scoring: gradients of log probabilities and entropies to the logits
        dict(name="logprobs_grad_4096x50257_bf16", kind="logprobs_grad", dt="bf16", rows=4096, vocab=VOCAB, top=0, scale=1.0),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "logprobs", "logprobs_grad"])
    if kind in ("append", "attend"):
        kv_heads, group = rng.choice([(12, 1), (8, 4), (1, 8), (4, 1), (2, 16), (4, 7), (16, 1)])
        c = dict(kind=kind, dt=rng.choice(["bf16", "f16", "f32"]), kv_heads=kv_heads, q_heads=kv_heads * group,
                 head_dim=rng.choice([64, 64, 96, 128, 128, 256]), page=rng.choice([16, 32, 64, 128]), ragged=rng.random() < 0.6)
        width = kv_heads * c["head_dim"]
        if kind == "append":
            c["new"] = 1 if rng.random() < 0.4 else _log_int(rng, 2, 2048)
            c["seqs"] = _log_int(rng, 1, max(1, min(64, 8192 * 1024 // (c["new"] * max(width, c["q_heads"] * c["head_dim"] // 4)))))
            c["context"] = _log_int(rng, 1, 1024) if rng.random() < 0.8 else 0
            c["interleaved"] = rng.random() < 0.4
            return c
        c["new"] = 1 if rng.random() < 0.5 else rng.choice([2, 3, 4, 5, 8, _log_int(rng, 9, 512)])
        c["context"] = _log_int(rng, 1, 8192)
        most = 64 * 8192 * 1024 // ((c["context"] + c["new"]) * width)  # as many codes as the largest listed case
        pairs = 4 * 512 * 8192 * 32 * 128 // (2 * (c["context"] + c["new"]) * c["new"] * c["q_heads"] * c["head_dim"])
        c["seqs"] = _log_int(rng, 1, max(1, min(64, most, pairs)))
        return c
    dt = rng.choice(["bf16", "f16", "f32"])
    vocab = _log_int(rng, 100, 200000)
    rows = _log_int(rng, 1, max(1, min(8192, 4096 * VOCAB * 2 // (vocab * SIZE[dt]))))
    top = min(rng.choice([0, 1, 5, 20, 32]), vocab)
    return dict(kind=kind, dt=dt, rows=rows, vocab=vocab, top=top, scale=rng.choice([1.0, 1.0, 0.7, 1.25]))


# ---- inputs ----------------------------------------------------------------------------------------------------------

def _lengths(c):
    """(new, total) tokens per sequence: equal ones, or spread from about a quarter to all of the case's sizes. They belong to
    the case, so that results of every seed have one shape."""
    n = c["seqs"]
    if not c["ragged"]:
        if c["kind"] == "append" and c["new"] == 1:  # decoding: every fill of the last page
            return [1] * n, [max(0, c["context"] - (7 * i) % (c["page"] + 1)) + 1 for i in range(n)]
        return [c["new"]] * n, [c["new"] + c["context"]] * n
    u = torch.rand(2, n, generator=torch.Generator().manual_seed(c["new"] * 8209 + c["context"])).tolist()
    new = [max(1, round(c["new"] * (0.25 + 0.75 * u[0][i]))) for i in range(n)] if c["new"] > 8 else [c["new"]] * n
    new[0] = c["new"]
    context = [round(c["context"] * (0.25 + 0.75 * u[1][i])) for i in range(n)]
    context[0] = c["context"]
    return new, [a + b for a, b in zip(new, context)]


def _cache_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    new, total = _lengths(c)
    page, kv, d, dt = c["page"], c["kv_heads"], c["head_dim"], TORCH[c["dt"]]
    counts = [-(-t // page) for t in total]
    pages = sum(counts) + 1  # one spare page, as a pool has
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)  # pages of a sequence lie anywhere in the pool
    table = torch.zeros(len(total), max(counts), dtype=torch.int32)
    first = 0
    host_order = order.cpu()
    for i, n in enumerate(counts):
        table[i, :n] = host_order[first:first + n]
        first += n
    # codes of keys and values: roughly normal, the largest of a block at 127
    k, v = (torch.randint(-127, 128, (pages, kv, page, d), generator=g, device="cuda", dtype=torch.int8) for _ in range(2))
    k_scale, v_scale = ((0.5 + torch.rand(pages, kv, generator=g, device="cuda")) * 0.02 for _ in range(2))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    s = dict(case=c, new=new, total=total, starts_host=starts, k=k, v=v, k_scale=k_scale, v_scale=v_scale, table=table.cuda(),
             lengths=torch.tensor(total, dtype=torch.int32).cuda(),
             starts=None if all(n == 1 for n in new) else torch.tensor(starts, dtype=torch.int32).cuda())
    tokens = starts[-1]
    if c["kind"] == "attend":
        s["q"] = torch.randn(tokens, c["q_heads"], d, generator=g, device="cuda").to(dt)
        s["scale"] = 1.0 / math.sqrt(d)
        return s
    # q, k and v of the new tokens side by side in the rows of one projection
    qkv = torch.randn(tokens, c["q_heads"] + 2 * kv, d, generator=g, device="cuda").to(dt)
    s["q"], s["new_k"], s["new_v"] = qkv[:, :c["q_heads"]], qkv[:, c["q_heads"]:c["q_heads"] + kv], qkv[:, c["q_heads"] + kv:]
    angle = torch.arange(max(total), dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    s["rope"] = torch.cat([angle.cos(), angle.sin()], dim=1).float().cuda()  # [positions, cosines | sines]
    # the pages that the call writes, for reading them back
    touched = []
    for i, (n, t) in enumerate(zip(new, total)):
        touched += table[i, (t - n) // page:-(-t // page)].tolist()
    s["touched"] = torch.tensor(touched, dtype=torch.int32).cuda().view(-1, 1)
    valid = []
    for i, (n, t) in enumerate(zip(new, total)):
        valid += [min(page, t - page * j) for j in range((t - n) // page, -(-t // page))]
    s["valid"] = torch.tensor(valid, dtype=torch.int32).cuda()
    # where each token goes, for the plain form
    pos, seq, slot_of = [], [], []
    base = 0
    for i, (n, t) in enumerate(zip(new, total)):
        p = torch.arange(t - n, t)
        pos.append(p)
        seq.append(torch.full((n,), i))
        slot_of.append(base + p // page - (t - n) // page)
        base += -(-t // page) - (t - n) // page
    s["pos"], s["seq"], s["touched_of"] = (torch.cat(x).cuda() for x in (pos, seq, slot_of))
    s["first_slot"] = torch.tensor([x for n, t in zip(new, total) for x in [(t - n) % page] + [0] * (-(-t // page) - (t - n) // page - 1)],
                                   dtype=torch.int64).cuda()
    return s


def _logit_inputs(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = TORCH[c["dt"]]
    logits = torch.randn(c["rows"], c["vocab"], generator=g, device="cuda").mul_(2.5).to(dt)
    targets = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device="cuda")
    # the tokens of a sequence are mostly likely ones
    likely = torch.rand(c["rows"], generator=g, device="cuda") < 0.5
    targets = torch.where(likely, logits.argmax(dim=1), targets)
    s = dict(case=c, logits=logits, targets=targets)
    if c["kind"] == "logprobs_grad":
        r = c["rows"]
        s["grad"] = torch.randn(r, generator=g, device="cuda") / r
        s["grad_entropy"] = torch.randn(r, generator=g, device="cuda") * (0.01 / r)
        z = logits.double().mul_(c["scale"]) if logits.numel() <= 1 << 26 else None
        if z is not None:
            lse = z.logsumexp(1)
            ent = lse - (torch.exp(z - lse[:, None]) * z).sum(1)
        else:  # piece by piece
            parts = []
            for rows in logits.split(256):
                z = rows.double().mul_(c["scale"])
                l = z.logsumexp(1)
                parts.append((l, l - (torch.exp(z - l[:, None]) * z).sum(1)))
            lse, ent = (torch.cat(x) for x in zip(*parts))
        s["lse"], s["entropy"] = lse.float(), ent.float()  # what the forward half leaves
        if c["top"]:
            s["top_ids"] = _top(logits, c["top"])
            s["grad_top"] = torch.randn(r, c["top"], generator=g, device="cuda") * (0.1 / r)
    return s


def _top(logits, k):
    """Places of the k largest entries of each row, the lowest first among equals."""
    return torch.cat([torch.sort(rows, dim=1, descending=True, stable=True).indices[:, :k] for rows in logits.split(512)]).to(torch.int32)


def prepare(case, seed):
    s = _cache_inputs(case, seed) if case["kind"] in ("append", "attend") else _logit_inputs(case, seed)
    if own and case["kind"] in ("append", "attend"):
        from metalhlo_b200 import cuda

        s["cache"] = cuda.KvCache(s["k"], s["v"], s["k_scale"], s["v_scale"])
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------

def run(state):
    return (_run_own if own else _run_plain)[state["case"]["kind"]](state)


def _append_own(s):
    from metalhlo_b200 import cuda

    q = cuda.kv_cache_append(s["cache"], s["new_k"], s["new_v"], s["table"], s["lengths"], token_starts=s["starts"], rope=s["rope"],
                             interleaved=s["case"]["interleaved"], q=s["q"])
    k, v = cuda.kv_cache_read(s["cache"], s["touched"], s["valid"], s["case"]["page"], dtype=s["q"].dtype)
    return q, k, v


def _attend_own(s):
    from metalhlo_b200 import cuda

    return cuda.cached_attention(s["q"], s["cache"], s["table"], s["lengths"], s["scale"], token_starts=s["starts"])


def _logprobs_own(s):
    from metalhlo_b200 import cuda

    r = cuda.token_logprobs(s["logits"], s["targets"], top_k=s["case"]["top"], scale=s["case"]["scale"])
    out = (r.logprobs, r.entropy, r.lse)
    return out + (r.top_logprobs, r.top_ids) if s["case"]["top"] else out


def _logprobs_grad_own(s):
    from metalhlo_b200 import cuda

    return cuda.token_logprobs_grad(s["logits"], s["targets"], s["lse"], s["entropy"], s["grad"], grad_entropy=s["grad_entropy"],
                                    top_ids=s.get("top_ids"), grad_top=s.get("grad_top"), scale=s["case"]["scale"])


def _rotate(x, rope, interleaved):
    """x [tokens, heads, d], rope [tokens, d]: cosines, then sines."""
    d = x.shape[-1]
    c, s = rope[:, None, :d // 2], rope[:, None, d // 2:]
    a, b = (x[..., 0::2], x[..., 1::2]) if interleaved else (x[..., :d // 2], x[..., d // 2:])
    ra, rb = a * c - b * s, b * c + a * s
    return torch.stack([ra, rb], dim=-1).flatten(-2) if interleaved else torch.cat([ra, rb], dim=-1)


def _append_plain(s):
    c = s["case"]
    page, pos = c["page"], s["pos"]
    rope = s["rope"][pos]
    q = _rotate(s["q"].float(), rope, c["interleaved"])
    values = []
    for codes, scales, x in ((s["k"], s["k_scale"], _rotate(s["new_k"].float(), rope, c["interleaved"])), (s["v"], s["v_scale"], s["new_v"].float())):
        blocks = s["touched"][:, 0].long()
        of = s["touched_of"]
        largest = torch.zeros(blocks.numel(), x.shape[1], device=x.device)
        largest.scatter_reduce_(0, of[:, None].expand(-1, x.shape[1]), x.abs().amax(-1), "amax")
        before = torch.where(s["first_slot"][:, None] == 0, 0.0, scales[blocks])
        scale = torch.maximum(before, largest / 127.0)
        # earlier tokens of a block whose scale has grown
        earlier = torch.arange(page, device=x.device) < s["first_slot"][:, None]
        block_codes = codes[blocks]
        again = torch.round(block_codes.float() * (before / scale)[:, :, None, None]).to(torch.int8)
        codes[blocks] = torch.where(earlier[:, None, :, None] & (scale > before)[:, :, None, None], again, block_codes)
        scales[blocks] = scale
        codes[blocks[of], :, pos % page] = torch.round(x * torch.reciprocal(scale)[of][:, :, None]).to(torch.int8)
        read = codes[blocks].float() * scale[:, :, None, None]
        read = read * (torch.arange(page, device=x.device) < s["valid"][:, None])[:, None, :, None]
        values.append(read.transpose(1, 2).contiguous().to(s["q"].dtype))
    return q.to(s["q"].dtype), values[0], values[1]


def _attend_plain(s):
    c = s["case"]
    group, d = c["q_heads"] // c["kv_heads"], c["head_dim"]
    outs = []
    for i, (n, t) in enumerate(zip(s["new"], s["total"])):
        ids = s["table"][i, :-(-t // c["page"])].long()
        k, v = ((x[ids].float() * sc[ids][:, :, None, None]).transpose(0, 1).reshape(c["kv_heads"], -1, d)[:, :t]
                for x, sc in ((s["k"], s["k_scale"]), (s["v"], s["v_scale"])))
        q = s["q"][s["starts_host"][i]:s["starts_host"][i + 1]].float()
        q = q.view(n, c["kv_heads"], group, d).permute(1, 2, 0, 3).reshape(c["kv_heads"], group * n, d)
        z = torch.matmul(q, k.transpose(1, 2)) * s["scale"]
        hidden = torch.arange(t, device=q.device)[None, :] > torch.arange(t - n, t, device=q.device)[:, None]
        if n > 1:
            z = z.masked_fill(hidden.repeat(group, 1), -math.inf)
        p = torch.exp(z - z.amax(-1, keepdim=True))
        o = torch.matmul(p, v) / p.sum(-1, keepdim=True)
        outs.append(o.view(c["kv_heads"], group, n, d).permute(2, 0, 1, 3).reshape(n, c["q_heads"], d))
    return torch.cat(outs).to(s["q"].dtype)


def _logprobs_plain(s):
    c = s["case"]
    z = s["logits"].float() * c["scale"]
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(1, keepdim=True)
    lse = (m + torch.log(total))[:, 0]
    entropy = lse - (e * z).sum(1) / total[:, 0]
    out = (z.gather(1, s["targets"][:, None])[:, 0] - lse, entropy, lse)
    if not c["top"]:
        return out
    ids = _top(s["logits"], c["top"])
    return out + (z.gather(1, ids.long()) - lse[:, None], ids)


def _logprobs_grad_plain(s):
    c = s["case"]
    logp = s["logits"].float() * c["scale"] - s["lse"][:, None]
    p = torch.exp(logp)
    at = s["grad"]
    if c["top"]:
        at = at + s["grad_top"].sum(1)
    dz = -p * (at[:, None] + s["grad_entropy"][:, None] * (logp + s["entropy"][:, None]))
    dz.scatter_add_(1, s["targets"][:, None], s["grad"][:, None])
    if c["top"]:
        dz.scatter_add_(1, s["top_ids"].long(), s["grad_top"])
    return (dz * c["scale"]).to(s["logits"].dtype)


_run_own = {"append": _append_own, "attend": _attend_own, "logprobs": _logprobs_own, "logprobs_grad": _logprobs_grad_own}
_run_plain = {"append": _append_plain, "attend": _attend_plain, "logprobs": _logprobs_plain, "logprobs_grad": _logprobs_grad_plain}


# ---- what a pass cannot do without --------------------------------------------------------------------------------------

def work(case):
    c = case
    if c["kind"] in ("append", "attend"):
        new, total = _lengths(c)
        es, d = SIZE[c["dt"]], c["head_dim"]
        tokens = sum(new)
        if c["kind"] == "append":
            q, kv = c["q_heads"] * d, c["kv_heads"] * d
            written = sum(t - (t - n) // c["page"] * c["page"] for n, t in zip(new, total))  # tokens of the pages that are read back
            moved = tokens * ((2 * q + 2 * kv) * es + 2 * kv)
            return {"bytes": moved + written * 2 * kv * (1 + es), "flops": tokens * (3 * q + 3 * kv + 4 * kv)}
        keys = sum(total)
        pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, total))
        blocks = sum(-(-t // c["page"]) for t in total)
        return {"bytes": 2 * keys * c["kv_heads"] * d + 8 * blocks * c["kv_heads"] + 2 * tokens * c["q_heads"] * d * es,
                "flops": 4 * pairs * c["q_heads"] * d}
    cells = c["rows"] * c["vocab"]
    if c["kind"] == "logprobs":
        return {"bytes": cells * SIZE[c["dt"]] + c["rows"] * (20 + 8 * c["top"]), "flops": 6 * cells}
    return {"bytes": 2 * cells * SIZE[c["dt"]] + c["rows"] * (24 + 8 * c["top"]), "flops": 7 * cells}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------

def exact(case, seed):
    return _exact[case["kind"]](case, seed)


def _exact_append(c, seed):
    s = _cache_inputs(c, seed)
    d, page = c["head_dim"], c["page"]
    half = d // 2
    first = torch.arange(half, device="cuda") * 2 if c["interleaved"] else torch.arange(half, device="cuda")
    second = first + (1 if c["interleaved"] else half)

    def turned(x):  # complex multiplication by the table's unit vectors
        w = torch.complex(s["rope"][s["pos"], :half].double(), s["rope"][s["pos"], half:].double())[:, None, :]
        z = torch.complex(x[..., first].double(), x[..., second].double()) * w
        out = torch.empty(x.shape, dtype=torch.float64, device=x.device)
        out[..., first], out[..., second] = z.real, z.imag
        return out

    results = [turned(s["q"])]
    for codes, scales, x in ((s["k"], s["k_scale"], turned(s["new_k"])), (s["v"], s["v_scale"], s["new_v"].double())):
        blocks = []
        for i, (n, t) in enumerate(zip(s["new"], s["total"])):
            rows = x[s["starts_host"][i]:s["starts_host"][i + 1]]
            at = t - n
            while at < t:
                end = min(t, (at // page + 1) * page)
                piece = rows[at - (t - n):end - (t - n)].transpose(0, 1)  # heads, tokens, d
                p = int(s["table"][i, at // page])
                old = scales[p].double() if at % page else torch.zeros(c["kv_heads"], dtype=torch.float64, device="cuda")
                scale = torch.maximum(old, piece.abs().flatten(1).amax(1) / 127)
                block = torch.zeros(c["kv_heads"], page, d, dtype=torch.float64, device="cuda")
                kept = codes[p, :, :at % page].double()
                kept = torch.where((scale > old)[:, None, None], torch.round(kept * (old / scale)[:, None, None]), kept)
                block[:, :at % page] = kept
                block[:, at % page:at % page + end - at] = torch.round(piece / scale[:, None, None])
                blocks.append((block * scale[:, None, None]).transpose(0, 1))
                at = end
        results.append(torch.stack(blocks))
    return tuple(results)


def _exact_attend(c, seed):
    s = _cache_inputs(c, seed)
    group, out = c["q_heads"] // c["kv_heads"], torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, (n, t) in enumerate(zip(s["new"], s["total"])):
        ids = s["table"][i].long()[:(t + c["page"] - 1) // c["page"]]
        for h in range(c["kv_heads"]):
            k = (s["k"][ids, h].double() * s["k_scale"][ids, h].double()[:, None, None]).flatten(0, 1)[:t]
            v = (s["v"][ids, h].double() * s["v_scale"][ids, h].double()[:, None, None]).flatten(0, 1)[:t]
            for j in range(0, n, 64):
                rows = slice(s["starts_host"][i] + j, s["starts_host"][i] + min(n, j + 64))
                q = s["q"][rows, h * group:(h + 1) * group].double()
                z = torch.einsum("ngd,kd->ngk", q, k) * s["scale"]
                seen = torch.arange(t, device="cuda")[None] <= (t - n + j + torch.arange(q.shape[0], device="cuda"))[:, None]
                z = torch.where(seen[:, None, :], z, -math.inf)
                out[rows, h * group:(h + 1) * group] = torch.einsum("ngk,kd->ngd", torch.softmax(z, -1), v)
    return out


def _exact_logprobs(c, seed):
    s = _logit_inputs(c, seed)
    parts = []
    for x, t in zip(s["logits"].split(256), s["targets"].split(256)):
        logp = torch.log_softmax(x.double() * c["scale"], 1)
        lse = (x[:, 0].double() * c["scale"] - logp[:, 0])
        entropy = torch.special.entr(torch.exp(logp)).sum(1)
        part = (logp.gather(1, t[:, None])[:, 0], entropy, lse)
        if c["top"]:
            ids = torch.sort(x.double(), dim=1, descending=True, stable=True).indices[:, :c["top"]]
            part += (logp.gather(1, ids), ids.to(torch.int32))
        parts.append(part)
    return tuple(torch.cat(x) for x in zip(*parts))


def _exact_logprobs_grad(c, seed):
    s = _logit_inputs(c, seed)
    out = []
    for r in range(0, c["rows"], 256):
        rows = slice(r, min(c["rows"], r + 256))
        logp = s["logits"][rows].double() * c["scale"] - s["lse"][rows].double()[:, None]
        p, e = torch.exp(logp), s["grad_entropy"][rows].double()
        picked = torch.zeros_like(p)  # what each entry's own log probability weighs in the loss
        index = torch.arange(p.shape[0], device="cuda")
        picked[index, s["targets"][rows]] += s["grad"][rows].double()
        if c["top"]:
            for j in range(c["top"]):
                picked[index, s["top_ids"][rows, j].long()] += s["grad_top"][rows, j].double()
        dz = picked - p * picked.sum(1, keepdim=True) - e[:, None] * p * (logp + s["entropy"][rows].double()[:, None])
        out.append(dz * c["scale"])
    return torch.cat(out)


_exact = {"append": _exact_append, "attend": _exact_attend, "logprobs": _exact_logprobs, "logprobs_grad": _exact_logprobs_grad}
