"""The operators of a decoding loop together, as a program uses them: layer products, the cache, attention over it, logits, log
probabilities, and the likeliest id as the next token. A step's launches follow each other without the host in between, so each has to
wait for what it reads."""
import os
import subprocess
import sys

import pytest
import torch

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADS, KV_HEADS, DIM, LAYERS, VOCAB, PAGE, STEPS = 8, 2, 64, 3, 1000, 32, 40
PROMPTS = [40, 1, 17, 70, 3]


class Decoder:
    def __init__(self):
        from metalhlo_b200 import cuda

        self.cuda = cuda
        g = torch.Generator().manual_seed(5)
        hidden = HEADS * DIM

        def weights(rows, cols):
            return (torch.randn(rows, cols, generator=g) * rows ** -0.5).bfloat16().cuda()

        self.embedding = torch.randn(VOCAB, hidden, generator=g).bfloat16().cuda()
        self.qkv = [weights(hidden, hidden + 2 * KV_HEADS * DIM) for _ in range(LAYERS)]
        self.out = [weights(hidden, hidden) for _ in range(LAYERS)]
        self.head = weights(hidden, VOCAB)
        self.prompt = torch.randint(0, VOCAB, (sum(PROMPTS),), generator=g).cuda()
        pages = [-(-(n + STEPS) // PAGE) for n in PROMPTS]
        self.table = torch.full((len(PROMPTS), max(pages)), -1, dtype=torch.int32)
        order = torch.randperm(sum(pages), generator=g).tolist()
        for b, n in enumerate(pages):
            self.table[b, :n] = torch.tensor([order.pop() for _ in range(n)])
        self.table = self.table.cuda()
        self.pages = sum(pages)
        self.rope = cuda.rope_table(max(PROMPTS) + STEPS, DIM)

    def fresh(self):
        return [self.cuda.KvCache.empty(self.pages, KV_HEADS, DIM, PAGE) for _ in range(LAYERS)]

    def hidden(self, caches, ids, lengths, starts=None):
        cuda = self.cuda
        x = self.embedding[ids]
        for cache, w, wo in zip(caches, self.qkv, self.out):
            rows = cuda.gemm(x, w).unflatten(1, (-1, DIM))
            q = cuda.kv_cache_append(cache, rows[:, HEADS:HEADS + KV_HEADS], rows[:, HEADS + KV_HEADS:], self.table, lengths, token_starts=starts,
                                     rope=self.rope, q=rows[:, :HEADS])
            o = cuda.cached_attention(q, cache, self.table, lengths, DIM ** -0.5, token_starts=starts)
            x = cuda.gemm(o.flatten(1), wo, residual=x)
        return x

    def score(self, x):
        logits = self.cuda.gemm(x, self.head)
        return logits, self.cuda.token_logprobs(logits, top_k=5)

    def begin(self, caches):
        lengths = torch.tensor(PROMPTS, dtype=torch.int32, device="cuda")
        starts = torch.tensor([0] + torch.tensor(PROMPTS).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
        x = self.hidden(caches, self.prompt, lengths, starts)
        return lengths, self.score(x[starts[1:].long() - 1])[1]

    def run(self, captured=False):
        caches = self.fresh()
        lengths, r = self.begin(caches)
        ids = r.top_ids[:, 0].long()
        tokens, tops = [ids.clone()], [r.top_logprobs]

        def step():
            lengths.add_(1)
            logits, r = self.score(self.hidden(caches, ids, lengths))
            ids.copy_(r.top_ids[:, 0])
            return logits, r.top_logprobs

        if captured:
            keep = lengths.clone(), ids.clone()
            state = [[t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale)] for c in caches]
            step()  # as programs warm up
            for c, s in zip(caches, state):
                for t, old in zip((c.k, c.v, c.k_scale, c.v_scale), s):
                    t.copy_(old)
            lengths.copy_(keep[0])
            ids.copy_(keep[1])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                result = step()
        for _ in range(STEPS):
            if captured:
                graph.replay()
            else:
                result = step()
            tokens.append(ids.clone())
            tops.append(result[1].clone())
        torch.cuda.synchronize()
        assert self.cuda.device_error() == 0
        return torch.stack(tokens), torch.stack(tops), result[0], caches


def test_a_decoding_loop_and_its_replay_give_the_same_tokens():
    d = Decoder()
    tokens, tops, logits, caches = d.run()
    again, again_tops, _, again_caches = d.run(captured=True)
    assert torch.equal(tokens, again) and torch.equal(tops, again_tops)
    for a, b in zip(caches, again_caches):
        assert torch.equal(a.k, b.k) and torch.equal(a.v, b.v) and torch.equal(a.k_scale, b.k_scale) and torch.equal(a.v_scale, b.v_scale)
    # the bounds of a log probability: its exponentials', their sum's, and its own roundings
    z, u = logits.double(), 2.0 ** -24
    top = float(z.abs().max())
    bound = 2.0 ** -22 + 8 * u * top + (VOCAB / 128 + 32) * u + 2 * u * (top + 7) + 4 * u * top + u * (2 * top + 7)
    ids = torch.sort(logits.float(), dim=-1, descending=True, stable=True).indices[:, :5]
    assert torch.equal(tokens[-1], ids[:, 0])
    assert bool(((tops[-1] - z.log_softmax(-1).gather(1, ids)).abs() <= bound).all())


def test_launches_that_overlap_wait_for_what_they_read():
    """METALHLO_PDL turns the overlap of launches on or off for all kernels of a process: the same bits come out."""
    program = """
import hashlib, sys, torch
sys.path.insert(0, "tests")
from test_lm_decoding_gpu import Decoder
d = Decoder()
out = [d.run(c) for c in (False, True)]
print(hashlib.sha256(b"".join(t.cpu().numpy().tobytes() for tokens, tops, _, caches in out for t in (tokens, tops, caches[-1].k, caches[-1].v_scale))).hexdigest())
"""
    hashes = []
    for mode in ("0", "1", None):
        env = {k: v for k, v in os.environ.items() if k != "METALHLO_PDL"}
        if mode is not None:
            env["METALHLO_PDL"] = mode
        r = subprocess.run([sys.executable, "-c", program], cwd=ROOT, env=env, capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]
        hashes.append(r.stdout.split()[-1])
    assert len(set(hashes)) == 1, hashes
