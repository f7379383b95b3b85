"""Attention over packed sequences, the gradients of the norms and the policy loss as programs call them: on other streams, two at once, captured and
replayed, with plans kept over layers, and with very many sequences."""
import math

import pytest
import torch

from tests.packed_reference import check, inputs, reference

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def both(x, plan, scale, stream=None):
    from metalhlo_b200 import cuda

    lse = torch.empty(x["q"].shape[:2], device="cuda")
    o = cuda.packed_attention(x["q"], x["k"], x["v"], plan, scale, lse=lse, stream=stream)
    return (o, lse, *cuda.packed_attention_grad(x["q"], x["k"], x["v"], o, lse, x["grad"], plan, scale, stream=stream))


def plan_of(x, causal=True):
    from metalhlo_b200 import cuda

    return cuda.packed_plan(x["starts_dev"], x["rows"], x["q"].shape[1], x["k"].shape[1], causal)


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F32, 64)])
def test_rows_in_front_of_the_first_sequence(dtype, dim):
    from metalhlo_b200 import cuda

    x = inputs([50, 200, 131], 4, 2, dim, dtype)
    starts = [50, 250, 381]
    y = dict(x, starts=starts, starts_dev=torch.tensor(starts, dtype=torch.int32, device="cuda"))
    for n in ("q", "k", "v", "grad"):
        y[n] = y[n].clone()
        y[n][:50] = math.nan
    plan = plan_of(y)
    outs = [torch.full(x[n].shape, 7.0, dtype=dtype, device="cuda") for n in ("q", "q", "k", "v")]
    lse = torch.full(x["q"].shape[:2], 7.0, device="cuda")
    cuda.packed_attention(y["q"], y["k"], y["v"], plan, 0.1, out=outs[0], lse=lse)
    cuda.packed_attention_grad(y["q"], y["k"], y["v"], outs[0], lse, y["grad"], plan, 0.1, *outs[1:])
    assert cuda.device_error() == 0
    assert all((t[:50] == 7.0).all() for t in (*outs, lse))
    want, off = reference({**{n: t[50:] if torch.is_tensor(t) else t for n, t in x.items()}, "starts": [0, 200, 331]}, 0.1, True)
    check(dict(zip(("o", "dq", "dk", "dv", "lse"), (t[50:] for t in (*outs, lse)))), want, off, ("o", "lse", "dq", "dk", "dv"))


@pytest.mark.parametrize("dtype,dim,heads", [(BF16, 128, (4, 1)), (F16, 64, (3, 3)), (BF16, 80, (14, 2)), (F32, 32, (2, 2))])
def test_a_sequence_does_not_depend_on_the_others(dtype, dim, heads):
    """The bits of a sequence's results among a thousand others, many of them empty, are those that it has alone."""
    lengths = [(37 * i * i + 11 * i) % 90 if i % 3 else 0 for i in range(1500)] + [700] + [5] * 200
    x = inputs(lengths, *heads, dim, dtype)
    scale = dim ** -0.5
    together = both(x, plan_of(x), scale)
    for b in (1, 4, 500, 1499, 1500, 1501, 1700):
        rows = slice(x["starts"][b], x["starts"][b + 1])
        n = rows.stop - rows.start
        y = dict(starts=[0, n], starts_dev=torch.tensor([0, n], dtype=torch.int32, device="cuda"), rows=n, **{k: x[k][rows] for k in ("q", "k", "v", "grad")})
        alone = both(y, plan_of(y), scale)
        for name, a, t in zip(("o", "lse", "dq", "dk", "dv"), alone, together):
            if name in ("o", "lse", "dq"):
                assert torch.equal(a, t[rows]), (b, name)
        # alone, few tiles of keys are cut into shares, which are added in another order; fp16 scales its products by the largest gradient of the call
        want, off = reference(y, scale, True)
        check(dict(zip(("dk", "dv"), (t[rows] for t in together[3:]))), want, off, ("dk", "dv"))


def test_very_many_sequences():
    from metalhlo_b200 import cuda

    x = inputs([3] * 30000 + [1] * 7000 + [0] * 5000 + [2] * 100, 2, 1, 64, BF16)
    o, lse, dq, dk, dv = both(x, plan_of(x), 0.125)
    assert cuda.device_error() == 0
    # sequences of three, all at once
    q, k, v, g = (x[n][:90000].double().view(30000, 3, -1, 64) for n in ("q", "k", "v", "grad"))
    z = torch.einsum("bihd,bjkd->bhij", q, k) * 0.125
    z = z.masked_fill(torch.ones(3, 3, dtype=torch.bool, device="cuda").triu(1), -math.inf)
    p = torch.softmax(z, -1)
    want = torch.einsum("bhij,bjkd->bihd", p, v).reshape(90000, 2, 64)
    # half a step of the result, and half a step of each weight: torch.finfo(bfloat16).eps / 2 = 2^-8
    assert ((o[:90000].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * torch.einsum("bhij,bjkd->bihd", p, v.abs()).reshape(90000, 2, 64)).all()
    want = torch.einsum("bhij,bihd->bjd", p, g).reshape(90000, 1, 64)
    assert ((dv[:90000].double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -14) * torch.einsum("bhij,bihd->bjd", p, g.abs()).reshape(90000, 1, 64)).all()
    assert torch.equal(o[90000:97000], x["v"][90000:97000].expand(-1, 2, -1))  # sequences of one


@pytest.mark.parametrize("dtype,dim", [(BF16, 128), (F16, 64), (F32, 64)])
def test_another_stream_and_two_at_once(dtype, dim):
    x, y = inputs([300, 77, 513], 4, 2, dim, dtype, seed=1), inputs([40, 640], 4, 2, dim, dtype, seed=2)
    px, py = plan_of(x), plan_of(y)
    want = both(x, px, 0.1), both(y, py, 0.1)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(4):  # raw handles: the view makes the stream current for what it allocates
        got.append([both(t, p, 0.1, stream=s.cuda_stream) for t, p, s in zip((x, y), (px, py), streams)])
    # one plan on two streams at once
    got += [[both(x, px, 0.1, stream=streams[0].cuda_stream), None], [both(x, px, 0.1, stream=streams[1].cuda_stream), None]]
    torch.cuda.synchronize()
    for pair in got:
        for a, w in zip(pair, want):
            assert a is None or all(torch.equal(s, t) for s, t in zip(a, w))


@pytest.mark.parametrize("dtype,dim", [(BF16, 120), (F16, 56), (F32, 40)])
def test_captured_and_replayed(dtype, dim):
    """Two graphs of the same calls (the first calls of their kind in this process may be among them), replayed with other contents."""
    from metalhlo_b200 import cuda

    x = inputs([130, 61], 4, 2, dim, dtype, seed=3)
    a, b = {n: x[n].clone() for n in ("q", "k", "v", "grad")}, {n: x[n].clone() for n in ("q", "k", "v", "grad")}
    plan = plan_of(x)
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    for t in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(both(t, plan, 0.1))
        graphs.append(g)
    y = inputs([130, 61], 4, 2, dim, dtype, seed=4)
    for n in b:
        b[n].copy_(y[n])
    for g in (graphs[0], graphs[1], graphs[0]):
        g.replay()
    torch.cuda.synchronize()
    assert cuda.device_error() == 0
    for t, got in zip((x, y), outs):
        assert all(torch.equal(s, w) for s, w in zip(got, both(t, plan, 0.1)))
    # the plan captured too: other starts, the same shapes
    starts = x["starts_dev"].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        made = cuda.packed_plan(starts, x["rows"], 4, 2)
        out = both(a, made, 0.1)
    starts.copy_(torch.tensor([0, 17, 191]))
    g.replay()
    torch.cuda.synchronize()
    z = dict(x, starts=[0, 17, 191], starts_dev=torch.tensor([0, 17, 191], dtype=torch.int32, device="cuda"))
    assert all(torch.equal(s, w) for s, w in zip(out, both(z, plan_of(z), 0.1)))


@pytest.mark.parametrize("hidden", [128, 1000, 4096, 20000])
def test_norms_captured_and_on_two_streams(hidden):
    from metalhlo_b200 import cuda

    g = torch.Generator(device="cuda").manual_seed(0)
    make = lambda: [torch.randn(200, hidden, generator=g, device="cuda").to(BF16) for _ in range(3)]  # noqa: E731
    gamma = torch.randn(hidden, generator=g, device="cuda").to(BF16)
    one, two = make(), make()
    want = [cuda.layer_norm_grad(x, gamma, dy, residual_grad=r) for x, dy, r in (one, two)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[cuda.layer_norm_grad(t[0], gamma, t[1], residual_grad=t[2], stream=s.cuda_stream) for t, s in zip((one, two), streams)] for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for u, w in zip(pair, want) for a, b in zip(u, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        out = cuda.layer_norm_grad(one[0], gamma, one[1], residual_grad=one[2])
    for t, s in zip(one, two):
        t.copy_(s)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[1]))


@pytest.mark.parametrize("tokens,cut", [(2000, True), (60000, True), (60000, False)])
def test_policy_loss_captured_and_on_two_streams(tokens, cut):
    from metalhlo_b200 import cuda
    from tests.test_policy_loss_gpu import inputs as policy_inputs

    x, y = policy_inputs(tokens, 1), policy_inputs(tokens, 2)
    starts = torch.tensor([0, tokens // 3, tokens], dtype=torch.int32, device="cuda") if cut else None

    def run(t, stream=None):
        return cuda.policy_loss(t["logprobs"], t["old_logprobs"], t["advantages"], mask=t["mask"], ref_logprobs=t["ref_logprobs"], starts=starts, kl_weight=0.1, stream=stream)

    want = run(x), run(y)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[run(t, s.cuda_stream) for t, s in zip((x, y), streams)] for _ in range(5)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for pair in got for u, w in zip(pair, want) for a, b in zip(u, w))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=streams[0]):
        out = run(x)
    for n in x:
        x[n].copy_(y[n])
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want[1]))
