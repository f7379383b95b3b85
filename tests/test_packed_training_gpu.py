"""One policy-gradient step of a small language model on packed sequences, forward and backward through this package's operators, against autograd in
64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HIDDEN, Q_HEADS, KV_HEADS, DIM, VOCAB, EPS = 96, 6, 2, 16, 211, 1e-5
LENGTHS = [37, 1, 140, 0, 66]


def parameters(dtype):
    g = torch.Generator(device="cuda").manual_seed(0)
    make = lambda *shape, size=1.0: (torch.randn(*shape, generator=g, device="cuda") * size / math.sqrt(shape[0])).to(dtype)  # noqa: E731
    p = dict(embed=make(VOCAB, HIDDEN, size=8.0), qkv=make(HIDDEN, (Q_HEADS + 2 * KV_HEADS) * DIM), out=make(Q_HEADS * DIM, HIDDEN), head=make(HIDDEN, VOCAB, size=2.0))
    for n in ("g1", "g2"):
        p[n] = (1 + 0.2 * torch.randn(HIDDEN, generator=g, device="cuda")).to(dtype)
    p["b1"] = (0.2 * torch.randn(HIDDEN, generator=g, device="cuda")).to(dtype)
    return p


def batch():
    g = torch.Generator(device="cuda").manual_seed(1)
    n = sum(LENGTHS)
    starts = [0]
    for m in LENGTHS:
        starts.append(starts[-1] + m)
    return dict(tokens=torch.randint(0, VOCAB, (n,), generator=g, device="cuda"), targets=torch.randint(0, VOCAB, (n,), generator=g, device="cuda"),
                old=-3 - torch.rand(n, generator=g, device="cuda") * 4, ref=-3 - torch.rand(n, generator=g, device="cuda") * 4, starts=starts,
                advantages=torch.randn(n, generator=g, device="cuda"), mask=torch.rand(n, generator=g, device="cuda") < 0.7,
                starts_dev=torch.tensor(starts, dtype=torch.int32, device="cuda"))


def step(p, b):
    """Loss and gradients of all parameters."""
    from metalhlo_b200 import cuda

    n, scale = b["tokens"].numel(), DIM ** -0.5
    plan = cuda.packed_plan(b["starts_dev"], n, Q_HEADS, KV_HEADS)
    x = p["embed"][b["tokens"]]
    h = cuda.layer_norm(x, p["g1"], p["b1"], EPS)
    qkv = cuda.gemm(h, p["qkv"]).view(n, Q_HEADS + 2 * KV_HEADS, DIM)
    q, k, v = qkv[:, :Q_HEADS], qkv[:, Q_HEADS:Q_HEADS + KV_HEADS], qkv[:, Q_HEADS + KV_HEADS:]
    lse = torch.empty(n, Q_HEADS, device="cuda")
    o = cuda.packed_attention(q, k, v, plan, scale, lse=lse)
    x2, y = cuda.add_rms_norm(cuda.gemm(o.view(n, -1), p["out"]), x, p["g2"], EPS)
    logits = cuda.gemm(y, p["head"])
    r = cuda.token_logprobs(logits, b["targets"], entropy=False)
    loss = cuda.policy_loss(r.logprobs, b["old"], b["advantages"], mask=b["mask"], ref_logprobs=b["ref"], starts=b["starts_dev"], kl_weight=0.05)
    # and back
    d = {}
    d_logits = cuda.token_logprobs_grad(logits, b["targets"], r.lse, grad_logprobs=loss.grad)
    d["head"] = cuda.gemm(y, d_logits, trans_a=True)
    d_y = cuda.gemm(d_logits, p["head"], trans_b=True)
    d_x2, d["g2"] = cuda.rms_norm_grad(x2, p["g2"], d_y, EPS)
    d["out"] = cuda.gemm(o.view(n, -1), d_x2, trans_a=True)
    d_o = cuda.gemm(d_x2, p["out"], trans_b=True).view(n, Q_HEADS, DIM)
    d_qkv = torch.empty_like(qkv)
    cuda.packed_attention_grad(q, k, v, o, lse, d_o, plan, scale, d_qkv[:, :Q_HEADS], d_qkv[:, Q_HEADS:Q_HEADS + KV_HEADS], d_qkv[:, Q_HEADS + KV_HEADS:])
    d_qkv = d_qkv.view(n, -1)
    d["qkv"] = cuda.gemm(h, d_qkv, trans_a=True)
    d_h = cuda.gemm(d_qkv, p["qkv"], trans_b=True)
    d_x, d["g1"], d["b1"] = cuda.layer_norm_grad(x, p["g1"], d_h, EPS, residual_grad=d_x2)
    d["embed"] = torch.zeros(VOCAB, HIDDEN, device="cuda").index_add_(0, b["tokens"], d_x.float())
    assert cuda.device_error() == 0
    return loss.loss, loss.kl, d


def reference(p, b):
    p = {n: t.double().requires_grad_() for n, t in p.items()}
    x = p["embed"][b["tokens"]]
    h = torch.nn.functional.layer_norm(x, (HIDDEN,), p["g1"], p["b1"], EPS)
    q, k, v = (h @ p["qkv"]).view(-1, Q_HEADS + 2 * KV_HEADS, DIM).split([Q_HEADS, KV_HEADS, KV_HEADS], 1)
    o = []
    for s, e in zip(b["starts"], b["starts"][1:]):
        qq, kk, vv = q[s:e].transpose(0, 1), *(t[s:e].transpose(0, 1).repeat_interleave(Q_HEADS // KV_HEADS, 0) for t in (k, v))
        z = (qq @ kk.transpose(1, 2) * DIM ** -0.5).masked_fill(torch.ones(e - s, e - s, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        o.append((torch.softmax(z, -1) @ vv).transpose(0, 1))
    x2 = x + torch.cat(o).flatten(1) @ p["out"]
    y = x2 * (x2.square().mean(1, keepdim=True) + EPS).rsqrt() * p["g2"]
    logp = torch.log_softmax(y @ p["head"], 1).gather(1, b["targets"][:, None])[:, 0]
    w = torch.zeros_like(logp)
    spans = [(s, e) for s, e in zip(b["starts"], b["starts"][1:]) if int(b["mask"][s:e].sum())]
    for s, e in spans:
        w[s:e][b["mask"][s:e]] = 1.0 / (int(b["mask"][s:e].sum()) * len(spans))
    ratio, a = torch.exp(logp - b["old"].double()), b["advantages"].double()
    t = b["ref"].double() - logp
    k3 = torch.exp(t) - t - 1
    loss = (w * (-torch.minimum(ratio * a, ratio.clamp(0.8, 1.2) * a) + 0.05 * k3)).sum()
    loss.backward()
    return loss.detach(), (w * k3).sum().detach(), {n: t.grad for n, t in p.items()}


@pytest.mark.parametrize("dtype,off", [(torch.float32, 2.0 ** -14), (torch.bfloat16, 2.0 ** -4)])
def test_a_step(dtype, off):
    """Against the norm of each gradient. fp32: some hundred roundings of 2^-24 one behind the other, and sums of two hundred terms of both signs that
    are up to eight times their result: 2^-14. bf16: a dozen roundings of 2^-8 on the way there and back, of either sign: four times one, and four times that for three
    normalising steps and the cancellation in softmax's gradient: 2^-4. A ratio that rounding takes over a border of the clip changes one token's gradient; with this seed none is that near in fp32."""
    p, b = parameters(dtype), batch()
    loss, kl, d = step(p, b)
    want_loss, want_kl, want = reference(p, b)
    assert abs(float(loss) - float(want_loss)) <= off * (abs(float(want_loss)) + abs(float(want_kl))) and abs(float(kl) / float(want_kl) - 1) <= off
    for n, g in d.items():
        assert torch.isfinite(g).all()
        if dtype == torch.float32 or n in ("head", "g2", "out"):
            assert float((g.double() - want[n]).norm()) <= off * float(want[n].norm()), n


def test_gradients_lower_the_loss():
    """A small step against the gradient lowers the loss by what the gradient says, to a tenth: the second order of a step of this size is less."""
    p, b = parameters(torch.float32), batch()
    loss, _, d = step(p, b)
    norm2 = sum(float(g.double().square().sum()) for g in d.values())
    rate = 1e-3 / math.sqrt(norm2)
    moved = {n: (t.double() - rate * d[n].double()).float() for n, t in p.items()}
    fall = float(reference(p, b)[0] - reference(moved, b)[0])
    assert abs(fall / (rate * norm2) - 1) < 0.1
