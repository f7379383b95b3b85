"""Attention over packed sequences and its gradients in 64 bits, with the bounds on rounding that the tests of the kernels go by."""
import math

import torch


def inputs(lengths, q_heads, kv_heads, dim, dtype, seed=0, spare=0, size=1.0, grad_size=1.0, device="cuda"):
    """Views of one projection's rows [tokens + spare, q_heads + 2 kv_heads, dim]; rows of no sequence are NaN."""
    g = torch.Generator(device=device).manual_seed(seed)
    starts = [0]
    for n in lengths:
        starts.append(starts[-1] + n)
    rows = starts[-1] + spare
    qkv = torch.randn(rows, q_heads + 2 * kv_heads, dim, generator=g, device=device)
    qkv[:, :q_heads] *= size
    qkv[starts[-1]:] = math.nan
    grad = torch.randn(rows, q_heads, dim, generator=g, device=device) * grad_size
    grad[starts[-1]:] = math.nan
    qkv, grad = qkv.to(dtype), grad.to(dtype)
    return dict(starts=starts, starts_dev=torch.tensor(starts, dtype=torch.int32, device=device), rows=rows, q=qkv[:, :q_heads],
                k=qkv[:, q_heads:q_heads + kv_heads], v=qkv[:, q_heads + kv_heads:], grad=grad)


def reference(x, scale, causal, out=None):
    """(results, bounds) of the sequences' rows, dicts of o, lse, dq, dk, dv in 64 bits. A rounding is off by half a step, eps / 2 of the value: the
    results' own, that of each weight p and each ds (16-bit types), and that of o, which the backward half starts from. Beside those,
    of fp32 sums and exponentials: a score of size |z| is off by 2^-18 (1 + |z|) at most, and so, relatively, is its weight; fp16
    weights below 2^-14 of the largest are off by 2^-25 of it (the backward half scales them so that this does not count)."""
    dtype = x["q"].dtype
    half = torch.finfo(dtype).eps / 2
    low = 0.0 if dtype == torch.float32 else half  # of weights and ds
    q, k, v, grad = (x[n].double() for n in ("q", "k", "v", "grad"))
    group = q.shape[1] // k.shape[1]
    want = {n: torch.zeros(t.shape, dtype=torch.float64, device=q.device) for n, t in (("o", q), ("lse", q[..., 0]), ("dq", q), ("dk", k), ("dv", k))}
    off = {n: t.clone() for n, t in want.items()}
    for a, b in zip(x["starts"], x["starts"][1:]):
        if a == b:
            continue
        for h in range(q.shape[1]):
            qq, kk, vv, gg = q[a:b, h], k[a:b, h // group], v[a:b, h // group], grad[a:b, h]
            z = qq @ kk.T * scale
            if causal:
                z = z.masked_fill(torch.ones_like(z, dtype=torch.bool).triu(1), -math.inf)
            p = torch.softmax(z, 1)
            z_off = 2.0 ** -18 * (1 + (qq.abs() @ kk.abs().T * scale).amax())
            o = p @ vv
            want["o"][a:b, h], want["lse"][a:b, h] = o, torch.logsumexp(z, 1)
            pv = p @ vv.abs()
            off["o"][a:b, h] = half * o.abs() + (low + 2 * z_off) * pv + (2.0 ** -25 * vv.abs().sum(0) if dtype == torch.float16 else 0)
            off["lse"][a:b, h] = 2 * z_off
            dp = gg @ vv.T
            delta = (p * dp).sum(1, keepdim=True)
            ds = p * (dp - delta)
            gv, go = gg.abs() @ vv.abs().T, (gg.abs() * pv).sum(1, keepdim=True)
            ds_off = low * ds.abs() + p * (4 * z_off * (dp - delta).abs() + 2.0 ** -20 * (gv + go) + (half + low + 2 * z_off) * go)
            ds_off += (2.0 ** -24 * ds.abs().amax() if dtype == torch.float16 else 0)
            want["dq"][a:b, h] = ds @ kk * scale
            off["dq"][a:b, h] = half * want["dq"][a:b, h].abs() + ds_off @ kk.abs() * scale
            want["dk"][a:b, h // group] += ds.T @ qq * scale
            off["dk"][a:b, h // group] += ds_off.T @ qq.abs() * scale
            want["dv"][a:b, h // group] += p.T @ gg
            off["dv"][a:b, h // group] += (low + 4 * z_off) * (p.T @ gg.abs())
    for n in ("dk", "dv"):
        off[n] += half * want[n].abs()
    for n in off:
        off[n] += 1e-30 + (2.0 ** -25 if dtype == torch.float16 and n != "lse" else 0)  # fp16 has no steps below 2^-24
    return want, off


def check(got, want, off, names):
    for n in names:
        g = got[n].double()
        bad = ~((g - want[n]).abs() <= off[n])
        assert not bad.any(), (n, int(bad.sum()), bad.numel(), float((g - want[n]).abs().max()), float(((g - want[n]).abs() / off[n]).nan_to_num(1e9).max()),
                               bad.nonzero()[:3].tolist())
