"""The paged operators and the sampler as they are used together: whole serving steps against a dense 64-bit
restatement, steps captured into CUDA graphs, other streams, caches beyond 2^31 elements, and sampled batched decode."""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

from test_paged import DT, attention_reference, cuda
from test_sample import reference as sample_reference

pytestmark = pytest.mark.gpu


class Model:
    """Two attention layers with a projection between them and logits: q, k, v and logits are products with fixed
    matrices of the layer's input, the layer's output is its input plus the attention's output times another."""

    def __init__(self, dtype, H=8, KV=2, hd=64, vocab=300, layers=2, seed=0, context=512):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g, device="cuda") / math.sqrt(s[0])  # noqa: E731
        self.dtype, self.H, self.KV, self.hd, self.vocab = dtype, H, KV, hd, vocab
        D = 96
        self.embed = torch.randn(vocab, D, generator=g, device="cuda")
        self.qkv = [rnd(D, (H + 2 * KV) * hd) for _ in range(layers)]
        self.o = [rnd(H * hd, D) for _ in range(layers)]
        self.out = rnd(D, vocab) * 3
        self.qn = [1 + 0.1 * torch.randn(hd, generator=g, device="cuda") for _ in range(layers)]
        self.kn = [1 + 0.1 * torch.randn(hd, generator=g, device="cuda") for _ in range(layers)]
        inv = 1e6 ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        ang = torch.arange(context, dtype=torch.float64, device="cuda")[:, None] * inv
        self.cos, self.sin = ang.cos().float(), ang.sin().float()

    def caches(self, n_pages, page):
        return [tuple(torch.full((n_pages, page, self.KV, self.hd), math.nan, dtype=DT[self.dtype], device="cuda")
                      for _ in "kv") for _ in self.qkv]

    def step(self, paged, tokens, plan, caches, table, ws):
        """One serving step over the paged operators; logits of every token of the (padded) batch."""
        x = self.embed[tokens]
        H, KV, hd = self.H, self.KV, self.hd
        for l, (kc, vc) in enumerate(caches):
            q, k, v = (x @ self.qkv[l]).view(-1, H + 2 * KV, hd).split([H, KV, KV], 1)
            q = paged.append(k, v, kc, vc, plan.positions, plan.slots, self.cos, self.sin, q=q, q_norm=self.qn[l],
                             k_norm=self.kn[l])
            a = paged.attention(q, kc, vc, table, plan.lens, plan.cu_new, ws)
            x = x + a.float().flatten(1) @ self.o[l]
        return x @ self.out

    def dense(self, tokens):
        """Logits of every token of one whole sequence, 64 bits but for the roundings to the cache's type."""
        d = lambda t: t.double()  # noqa: E731
        x = d(self.embed)[tokens]
        H, KV, hd, n = self.H, self.KV, self.hd, len(tokens)
        rd = lambda t: t.to(DT[self.dtype]).double()  # noqa: E731
        cos, sin = d(self.cos)[:n, None], d(self.sin)[:n, None]

        def turn(y, w):
            y = y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * d(w)
            a, b = y.chunk(2, -1)
            return rd(torch.cat([a * cos - b * sin, b * cos + a * sin], -1))

        for l in range(len(self.qkv)):
            q, k, v = (x @ d(self.qkv[l])).view(n, H + 2 * KV, hd).split([H, KV, KV], 1)
            q, k, v = turn(q, self.qn[l]), turn(k, self.kn[l]), rd(v)
            s = torch.einsum("ihd,jhd->hij", q, k.repeat_interleave(H // KV, 1)) / math.sqrt(hd)
            s = s.masked_fill(torch.ones(n, n, device="cuda").triu(1).bool(), -math.inf)
            a = rd(torch.einsum("hij,jhd->ihd", s.softmax(-1), v.repeat_interleave(H // KV, 1)))
            x = x + a.flatten(1) @ d(self.o[l])
        return x @ d(self.out)


def _server(n_req, max_pages, n_pages):
    table = torch.full((n_req, max_pages), -1, dtype=torch.int32, device="cuda")
    ring = torch.arange(n_pages, dtype=torch.int32, device="cuda").flip(0).contiguous()
    state = torch.tensor([0, n_pages], dtype=torch.int64, device="cuda")
    return table, ring, state, torch.zeros(n_req, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_requests_that_come_and_go(pkg, dtype):
    """Prompts' chunks beside decodes over several steps, requests finishing and their pages serving others: logits of
    every token against the dense restatement (f32: the operators' and cuBLAS' f32 roundings through two layers, 1e-4
    of the largest logit; 16 bits: a cached value or output on the other side of a rounding, one of eps in each of two
    layers' four roundings), and the sampled tokens against the definition on the same logits."""
    from minicpmo_b200 import paged

    m = Model(dtype)
    page, n_req, n_pages, cap = 16, 4, 16, 96
    caches = m.caches(n_pages, page)
    table, ring, state, lens = _server(n_req, 8, n_pages)
    ws = paged.workspace()
    rng = np.random.default_rng(5)
    seqs = [[] for _ in range(n_req)]
    # what each request adds in each step; -1: finished (and the slot free for another)
    steps = [[40, 0, 7, 1], [1, 33, 1, 0], [1, 1, 1, 50], [-1, 1, 30, 1], [20, -1, 1, 1], [1, 70, 1, -1], [1, 1, -1, 9]]
    eps = torch.finfo(DT[dtype]).eps
    for new in steps:
        toks = [rng.integers(0, m.vocab, max(a, 0)).tolist() for a in new]
        flat = sum(toks, [])
        batch = torch.tensor(flat + [0] * (cap - len(flat)), device="cuda")
        p = paged.plan(lens, cuda(new, torch.int32), table, ring, state, page, cap)
        lens, state = p.lens, p.ring_state
        assert p.status[0] == 0
        logits = m.step(paged, batch, p, caches, table, ws)
        at = 0
        for r, a in enumerate(new):
            if a < 0:
                seqs[r] = []
                continue
            seqs[r] += toks[r]
            if a:
                want = m.dense(torch.tensor(seqs[r], device="cuda"))[-a:]
                got = logits[at:at + a].double()
                tol = (1e-4 if dtype == "f32" else 8 * eps) * float(want.abs().max())
                assert float((got - want).abs().max()) <= tol
            at += a
        assert lens.tolist() == [len(s) for s in seqs]
        # draw from the last rows
        rows = logits[:n_req].contiguous()
        u = rng.random(n_req).astype(np.float32)
        top_p = np.float32(0.9)
        r = paged.sample(rows, cuda(u), top_p=torch.full((n_req,), float(top_p), device="cuda"))
        for b in range(n_req):
            t, _, k, _ = sample_reference(rows[b].double().cpu().numpy(), u[b], 1.0, 0, top_p, 0.0)
            assert (int(r.token[b]), int(r.kept[b])) == (t, k)
    held = sum(-(-len(s) // page) for s in seqs)
    assert int(state[1] - state[0]) == n_pages - held


def test_a_captured_step_replays_on_new_lengths(pkg):
    """One decode step (plan in place, append, attention, sample) captured once and replayed: positions, pages and
    lengths move on the device alone; the same tokens come from eager steps."""
    from minicpmo_b200 import paged

    m = Model("bf16", context=128)
    page, n_req, n_pages = 8, 3, 24
    prompt = [20, 5, 13]
    results = []
    for captured in (False, True):
        caches = m.caches(n_pages, page)
        table, ring, state, lens = _server(n_req, 8, n_pages)
        ws = paged.workspace()
        batch = torch.arange(sum(prompt), device="cuda") % m.vocab
        p = paged.plan(lens, cuda(prompt, torch.int32), table, ring, state, page, sum(prompt))
        lens.copy_(p.lens)
        state.copy_(p.ring_state)
        logits = m.step(paged, batch, p, caches, table, ws)
        token = logits[p.cu_new[1:].long() - 1].argmax(-1)
        uniforms = torch.rand(12, n_req, generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
        ones = torch.ones(n_req, dtype=torch.int32, device="cuda")
        i32 = lambda n: torch.zeros(n, dtype=torch.int32, device="cuda")  # noqa: E731
        out = paged.PagedPlan(lens, state, i32(n_req + 1), i32(n_req), i32(n_req).long(), i32(2))
        u = torch.zeros(n_req, device="cuda")
        temp = torch.full((n_req,), 0.8, device="cuda")
        drawn = paged.Sampled(i32(n_req), torch.zeros(n_req, device="cuda"), i32(n_req))

        def step():
            paged.plan(lens, ones, table, ring, state, page, n_req, out=out)
            rows = m.step(paged, token, out, caches, table, ws)
            paged.sample(rows, u, temperature=temp, out=drawn)
            token.copy_(drawn.token)

        got = []
        if captured:
            keep = [t.clone() for t in (lens, state, table, ring, token)] + [c.clone() for kv in caches for c in kv]
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()  # libraries set themselves up outside the capture
            torch.cuda.current_stream().wait_stream(s)
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
            for t, k in zip([lens, state, table, ring, token] + [c for kv in caches for c in kv], keep):
                t.copy_(k)
        for i in range(12):
            u.copy_(uniforms[i])
            graph.replay() if captured else step()
            got.append((drawn.token.tolist(), lens.tolist(), out.status.tolist()))
        results.append(got)
    assert results[0] == results[1]
    assert results[0][-1][1] == [n + 12 for n in prompt] and results[0][-1][2][0] == 0


def test_other_streams(pkg):
    """Work enqueued behind a long kernel on a side stream waits for it there, and only there."""
    from minicpmo_b200 import paged

    m = Model("f16")
    caches = m.caches(8, 16)
    table, ring, state, lens = _server(2, 4, 8)
    new = cuda([30, 4], torch.int32)
    batch = torch.arange(34, device="cuda")
    ws = paged.workspace()
    p = paged.plan(lens, new, table, ring, state, 16, 34)
    want = m.step(paged, batch, p, caches, table, ws)
    caches2 = m.caches(8, 16)
    table2, ring2, state2, lens2 = _server(2, 4, 8)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        x = torch.randn(4096, 4096, device="cuda")
        for _ in range(20):
            x = x @ x * 1e-2
        lens2.add_((x[0, 0] * 0).nan_to_num(0).int())  # behind the products
        p2 = paged.plan(lens2, new, table2, ring2, state2, 16, 34)
        got = m.step(paged, batch, p2, caches2, table2, ws)
    s.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("chunk", [1, 200])
def test_caches_beyond_31_bits(pkg, dtype, chunk):
    """Pages whose first element lies behind 2^31 elements (and 2^32 bytes) of the cache."""
    from minicpmo_b200 import paged

    page, KV, hd, H, n = 16, 2, 128, 4, 300
    n_pages = (2 ** 31 + 2 ** 28) // (page * KV * hd)
    kc, vc = (torch.empty(n_pages, page, KV, hd, dtype=DT[dtype], device="cuda") for _ in "kv")
    held = -(-n // page)
    table = torch.arange(n_pages - held, n_pages, dtype=torch.int32, device="cuda").flip(0)[None].contiguous()
    g = torch.Generator(device="cuda").manual_seed(1)
    k, v, q = (torch.randn(n, h, hd, generator=g, device="cuda").to(DT[dtype]) for h in (KV, KV, H))
    pos = torch.arange(n, device="cuda")
    slots = table[0].long()[pos // page] * page + pos % page
    one, zero = torch.ones(n, hd // 2, device="cuda"), torch.zeros(n, hd // 2, device="cuda")
    paged.append(k, v, kc, vc, pos.int(), slots, one, zero)  # no norm, no rotation: the rows as they are
    assert torch.equal(kc.view(-1, KV, hd)[slots], k) and torch.equal(vc.view(-1, KV, hd)[slots], v)
    q = q[-chunk:]
    out = paged.attention(q, kc, vc, table, cuda([n], torch.int32), cuda([0, chunk], torch.int32), paged.workspace())
    want, _, mag = attention_reference(q, kc, vc, table, [n], [0, chunk], hd ** -0.5)
    # f32: the score's error moves a weight by less than 2^-16 here; 16 bits: weights and result rounded once each
    tol = (2.0 ** -16 if dtype == "f32" else torch.finfo(DT[dtype]).eps) * mag + 1e-30
    assert ((out.double() - want).abs() <= tol).all()


def test_wrong_device_and_host_memory_are_refused(pkg):
    """The C entry points check that the buffers are the current device's memory."""
    lib = pkg.lib()
    host = torch.zeros(4096, dtype=torch.int32)
    err = C.create_string_buffer(512)
    p = host.data_ptr()
    p -= p % 256
    assert lib.minicpmo_gpu_sample(p, 0, 2, 10, 10, None, None, None, None, p, p, None, None, None, err, 512) == 0
    assert b"not memory of the current device" in err.value
    assert lib.minicpmo_gpu_paged_plan(p, p + 64, 4, p, 8, 8, p, 32, p, 16, 64, p, p, p + 128, p, p, p, None, err, 512) == 0
    assert b"not memory of the current device" in err.value


@pytest.mark.parametrize("B", [2, 5])
def test_sampled_batched_decode(pkg, B):
    """sample_batch draws from the logits of the last batched step as the definition does, and generate_batch_sampled
    feeds what it draws; temperature 0 is the greedy decode."""
    from minicpmo_b200 import gguf
    from minicpmo_b200.gpu import GpuError
    from minicpmo_b200.qwen3 import Qwen3Runtime

    shape = gguf.Qwen3Shape(layers=2, hidden=512, heads=8, kv_heads=2, head_dim=128, ffn=1536, vocab=2048, context=48)
    tensors = gguf.synth_model(shape, gguf.ALL_Q8_0, seed_base=6)
    P, n = 8, 10
    prompts = np.stack([gguf.prompt_ids(P, shape.vocab, seed=30 + b) for b in range(B)])
    rng = np.random.default_rng(B)
    u = rng.random((n, B)).astype(np.float32)
    par = dict(temperature=0.9, top_k=[0, 30, 5, 200, 1][:B], top_p=0.95, min_p=0.01)
    rt = Qwen3Runtime.open(tensors, shape=shape, context=shape.context, kv_f16=True, max_batch=B)
    with pytest.raises(GpuError, match="no step has computed logits"):
        rt.sample_batch(u[0])
    rt.append_prompt_batch(prompts)
    drawn = rt.generate_batch_sampled(n, u, **par)
    rt.close()
    rt = Qwen3Runtime.open(tensors, shape=shape, context=shape.context, kv_f16=True, max_batch=B)
    nxt, _ = rt.append_prompt_batch(prompts[:, :-1])
    _, _, lg = rt.forward_batch(prompts[:, -1], np.full(B, P - 1, np.uint32), want_logits=True)
    for i in range(n):
        tok, prob, kept = rt.sample_batch(u[i], **par)
        for b in range(B):
            t, p, k, _ = sample_reference(lg[b].astype(np.float64), u[i, b], np.float32(0.9), par["top_k"][b],
                                          np.float32(0.95), np.float32(0.01))
            assert (tok[b], kept[b]) == (t, k) and abs(prob[b] - p) <= 2.0 ** -23 * p
        assert np.array_equal(tok, drawn[:, i])
        greedy, _, lg = rt.forward_batch(tok, np.full(B, P + i, np.uint32), want_logits=True)
        assert np.array_equal(rt.sample_batch(u[i], temperature=0.0)[0], greedy)
    with pytest.raises(GpuError, match="n_seq"):
        rt.sample_batch(u[0][:1])
    rt.close()
