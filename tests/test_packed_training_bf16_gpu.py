"""The gradients of a bf16 policy-gradient step that come back through attention and both norms, against 64 bits and beside what torch's own operators make of
the same step in bf16."""
import math

import pytest
import torch

from tests.test_packed_training_gpu import DIM, EPS, HIDDEN, KV_HEADS, Q_HEADS, batch, parameters, reference, step

pytestmark = pytest.mark.gpu


def torch_step(p, b):
    """The step in torch's operators on bf16 tensors, which round where the kernels round: after every operator. Loss in fp32."""
    p = {n: t.clone().requires_grad_() for n, t in p.items()}
    x = p["embed"][b["tokens"]]
    h = torch.nn.functional.layer_norm(x, (HIDDEN,), p["g1"], p["b1"], EPS)
    q, k, v = (h @ p["qkv"]).view(-1, Q_HEADS + 2 * KV_HEADS, DIM).split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
    o = []
    for s, e in zip(b["starts"], b["starts"][1:]):
        qq, kk, vv = q[s:e].transpose(0, 1), *(t[s:e].transpose(0, 1).repeat_interleave(Q_HEADS // KV_HEADS, 0) for t in (k, v))
        z = (qq.float() @ kk.float().transpose(1, 2) * DIM ** -0.5).masked_fill(torch.ones(e - s, e - s, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        o.append((torch.softmax(z, -1).to(qq.dtype) @ vv).transpose(0, 1))
    x2 = x + torch.cat(o).flatten(1) @ p["out"]
    y = (x2.float() * (x2.float().square().mean(1, keepdim=True) + EPS).rsqrt()).to(x2.dtype) * p["g2"]
    logp = torch.log_softmax((y @ p["head"]).float(), 1).gather(1, b["targets"][:, None])[:, 0]
    w = torch.zeros_like(logp)
    spans = [(s, e) for s, e in zip(b["starts"], b["starts"][1:]) if int(b["mask"][s:e].sum())]
    for s, e in spans:
        w[s:e][b["mask"][s:e]] = 1.0 / (int(b["mask"][s:e].sum()) * len(spans))
    ratio, a, t = torch.exp(logp - b["old"]), b["advantages"], b["ref"] - logp
    loss = (w * (-torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a) + 0.05 * (torch.exp(t) - t - 1))).sum()
    loss.backward()
    return {n: t.grad for n, t in p.items()}


def test_all_gradients():
    """The kernels round as often as torch's operators do, in part at other places: of errors of the same number of roundings neither is more than twice the other, against the
    norm of each gradient."""
    p, b = parameters(torch.bfloat16), batch()
    got, own, want = step(p, b)[2], torch_step(p, b), reference(p, b)[2]
    for n, w in want.items():
        off, of_torch = (float((t[n].double() - w).norm() / w.norm()) for t in (got, own))
        assert off <= 2 * of_torch, (n, off, of_torch)
