"""Cases and plain forms of the paged serving operators: page planning, the K/V append, attention of new tokens over a
paged cache, and sampling.

One serving step of this framework's paged path runs them in this order: ``plan`` gives every request's new tokens their
pages, positions and cache slots, ``append`` writes their K and V rows there (after QK-norm and RoPE), ``attention``
attends them over the pages, and ``sample`` draws the next tokens from the logits.  Each case below is one call of one
of them.  With ``own`` false, ``run`` computes the operator with elementary torch operations; with ``own`` true it makes
the framework's call.
"""
from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
EPS = 1e-6
ROPE_BASE = 1e6
WORKSPACE_BYTES = 64 << 20  # MINICPMO_PAGED_WORKSPACE_BYTES
TOP_P_OFF = float(np.float32(0.999999))  # top_p from here on keeps everything
GREEDY_BELOW = float(np.float32(1e-6))  # temperatures up to here take the largest logit


def _paged():
    """The framework's paged operators (its package directory is not an identifier, so it is loaded by path)."""
    if "minicpmo_b200" not in sys.modules:
        import importlib.util

        pkg_dir = Path(__file__).resolve().parents[1] / "minicpm-o-uya_b200"
        spec = importlib.util.spec_from_file_location("minicpmo_b200", pkg_dir / "__init__.py",
                                                      submodule_search_locations=[str(pkg_dir)])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["minicpmo_b200"] = mod
        spec.loader.exec_module(mod)
    from minicpmo_b200 import paged

    return paged


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a full batch: every request adds a token
        {"name": "plan decode 32", "op": "plan", "requests": 32, "chunk": 1, "finished": 0.0, "page": 16,
         "context": 4096, "shape": 1},
        # a large scheduler step: prompts' chunks beside decodes, some requests finished
        {"name": "plan mixed 512", "op": "plan", "requests": 512, "chunk": 256, "finished": 0.05, "page": 64,
         "context": 16384, "shape": 2},
        # the K/V rows of a 32-sequence decode step of the 8B shape, f32 activations into an f16 cache
        {"name": "append decode 32", "op": "append", "tokens": 32, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "input": "f32", "cache": "f16", "norm": True, "page": 16, "padding": 0},
        # a prompt pass of the 8B shape, f32 activations into a bf16 cache, the batch padded to its capacity
        {"name": "append prompt 8192", "op": "append", "tokens": 8192, "heads": 32, "kv_heads": 8, "head_dim": 128,
         "input": "f32", "cache": "bf16", "norm": True, "page": 64, "padding": 37},
        # one sequence decoding behind a 512-token prompt: latency
        {"name": "attention decode 1", "op": "attention", "requests": 1, "chunk": 1, "context": 565, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dtype": "f16", "page": 16, "lse": False, "shape": 3},
        # 32 sequences of ragged lengths decoding, up to the runtime's context
        {"name": "attention decode 32", "op": "attention", "requests": 32, "chunk": 1, "context": 4096, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dtype": "f16", "page": 16, "lse": False, "shape": 4},
        # a few short odd chunks over the f32 cache that is this framework's default
        {"name": "attention f32 5", "op": "attention", "requests": 5, "chunk": 33, "context": 1000, "heads": 16,
         "kv_heads": 8, "head_dim": 128, "dtype": "f32", "page": 32, "lse": True, "shape": 5},
        # a 512-token prompt from an empty cache
        {"name": "attention prompt 512", "op": "attention", "requests": 1, "chunk": 512, "context": 512, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "page": 64, "lse": False, "shape": 6},
        # four long prompts' chunks over what they have cached
        {"name": "attention chunk 4x2048", "op": "attention", "requests": 4, "chunk": 2048, "context": 16384,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "dtype": "bf16", "page": 128, "lse": True, "shape": 7},
        # one sequence's next token over the full vocabulary: latency
        {"name": "sample 1", "op": "sample", "rows": 1, "vocab": 151936, "dtype": "f32", "filters": True},
        # a batch's next tokens, every row with its own settings
        {"name": "sample 32", "op": "sample", "rows": 32, "vocab": 151936, "dtype": "f32", "filters": True},
        # many rows of 16-bit logits, temperature alone: the whole distribution is drawn from
        {"name": "sample 128 bf16", "op": "sample", "rows": 128, "vocab": 151936, "dtype": "bf16", "filters": False},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attention", "attention", "sample"])
    shape = rng.randrange(1 << 20)
    heads, kv = rng.choice([(32, 8), (16, 8), (64, 8), (8, 8), (14, 2), (28, 4), (20, 4)])
    page = rng.choice([16, 32, 64, 128])
    if op == "plan":
        requests = _log(rng, 1, 512)
        chunk = _log(rng, 1, 256)
        return {"op": op, "requests": requests, "chunk": chunk, "finished": rng.choice([0.0, 0.05, 0.3]),
                "page": page, "context": max(2 * chunk, _log(rng, 64, 16384)), "shape": shape}
    if op == "append":
        return {"op": op, "tokens": _log(rng, 1, 4096), "heads": heads, "kv_heads": kv,
                "head_dim": rng.choice([64, 128]), "input": rng.choice(["f32", "f16", "bf16"]),
                "cache": rng.choice(["f32", "f16", "bf16"]), "norm": rng.random() < 0.7, "page": page,
                "padding": rng.randrange(40)}
    if op == "sample":
        return {"op": op, "rows": _log(rng, 1, 100), "vocab": _log(rng, 200, 151936),
                "dtype": rng.choice(["f32", "f16", "bf16"]), "filters": rng.random() < 0.7}
    dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"])
    hd = rng.choice([64, 128, 128, 256])
    if rng.random() < 0.5:  # decode, or a few speculated tokens each
        requests, chunk = _log(rng, 1, 96), rng.choice([1, 1, 1, 3, 8])
        context = max(chunk, _log(rng, 40, 16384))
    else:  # prompts' chunks
        requests, chunk = _log(rng, 1, 8), _log(rng, 16, 2048)
        context = max(chunk, _log(rng, 64, 16384))
    most = 2 ** 31 if dtype != "f32" and hd != 256 else 2 ** 28  # scores: the largest listed case has 2^32
    while requests * chunk * context * heads > most or requests * context * kv * hd > 2 ** 28:
        if requests > 1:
            requests = (requests + 1) // 2
        else:
            context = max(chunk, context // 2)
            chunk = max(1, chunk // 2)
    return {"op": op, "requests": requests, "chunk": chunk, "context": context, "heads": heads, "kv_heads": kv,
            "head_dim": hd, "dtype": dtype, "page": page, "lse": rng.random() < 0.5, "shape": shape}


def _plan_lengths(case):
    """Cached lengths and new tokens of every request (-1: finished) of a scheduler step."""
    r = np.random.RandomState(case["shape"])
    R, chunk, context = case["requests"], case["chunk"], case["context"]
    if chunk == 1:
        new = np.ones(R, np.int64)
    else:  # decodes and prompts' chunks, and requests that wait this step
        new = np.where(r.rand(R) < 0.5, 1, r.randint(0, chunk + 1, R))
        new[r.randint(R)] = chunk
    lens = r.randint(0, context - chunk + 1, R)
    new[r.rand(R) < case["finished"]] = -1
    if not (new > 0).any():
        new[0] = 1
    return lens.astype(np.int64), new


def _attention_lengths(case):
    """Total lengths and new tokens of every request: lengths from a quarter of the context up, chunks from a third up."""
    r = np.random.RandomState(case["shape"])
    R, chunk, context = case["requests"], case["chunk"], case["context"]
    new = r.randint(max(1, chunk // 3), chunk + 1, R)
    new[r.randint(R)] = chunk
    if R <= 4 and chunk >= 256:
        new[:] = chunk
    lens = r.randint(max(1, context // 4), context + 1, R)
    lens[r.randint(R)] = context
    return np.maximum(lens, new).astype(np.int64), new.astype(np.int64)


def work(case):
    op = case["op"]
    if op == "plan":
        lens, new = _plan_lengths(case)
        add, page = np.maximum(new, 0), case["page"]
        held, want = -(-lens // page), -(-(lens + add) // page)
        moved = int((want - held).sum() + held[new < 0].sum())
        tokens = _capacity(int(add.sum()))
        return {"bytes": 4.0 * (4 * len(lens) + 2 * moved) + 12.0 * tokens, "flops": 0.0}
    if op == "append":
        T = case["tokens"]
        values = T * (case["heads"] + 2 * case["kv_heads"]) * case["head_dim"]
        turned = T * (case["heads"] + case["kv_heads"]) * case["head_dim"]
        return {"bytes": float(values * (SIZES[case["input"]] + SIZES[case["cache"]]) + T * (12 + 4 * case["head_dim"])),
                "flops": 7.0 * turned}
    if op == "sample":
        return {"bytes": float(case["rows"] * case["vocab"] * SIZES[case["dtype"]]), "flops": 0.0}
    lens, new = _attention_lengths(case)
    pairs = float(sum(n * (l - n) + n * (n + 1) / 2 for l, n in zip(lens.tolist(), new.tolist())))
    hd, size = case["head_dim"], SIZES[case["dtype"]]
    return {"bytes": float(size * hd * (2 * case["heads"] * int(new.sum()) + 2 * case["kv_heads"] * int(lens.sum()))),
            "flops": 4.0 * hd * case["heads"] * pairs}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _capacity(tokens):
    """A batch's token capacity: programs pad it, so that captured graphs fit several steps."""
    return -(-tokens // 64) * 64


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _pages(held, n_pages, max_pages, perm):
    """Block table rows whose first held[r] entries are pages of `perm`, in order; the rest is stale (-1)."""
    held = torch.from_numpy(held).cuda()
    first = torch.cumsum(held, 0) - held
    col = torch.arange(max_pages, device="cuda")
    at = (first[:, None] + col).clamp(max=n_pages - 1)
    return torch.where(col < held[:, None], perm[at], -1).to(torch.int32)


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = {"case": dict(case)}
    if op == "plan":
        lens, new = _plan_lengths(case)
        page, R = case["page"], len(lens)
        max_pages = -(-case["context"] // page)
        held, want = -(-lens // page), -(-(lens + np.maximum(new, 0)) // page)
        n_pages = int(want.sum()) + 64
        perm = torch.randperm(n_pages, generator=g, device="cuda")
        s["block_table"] = _pages(held, n_pages, max_pages, perm)
        # the ring of free pages: `tail - head` ids from `head` on, somewhere inside it
        head = 5 * n_pages + seed % n_pages
        ring = torch.full((n_pages,), -1, dtype=torch.int32, device="cuda")
        free = perm[int(held.sum()):]
        ring[(head + torch.arange(free.numel(), device="cuda")) % n_pages] = free.to(torch.int32)
        s["free_ring"] = ring
        s["ring_state"] = torch.tensor([head, head + free.numel()], dtype=torch.int64, device="cuda")
        s["lens"] = torch.from_numpy(lens).to("cuda", torch.int32)
        s["new_lens"] = torch.from_numpy(new).to("cuda", torch.int32)
        s["tokens"] = _capacity(int(np.maximum(new, 0).sum()))
        s["page"] = page
        return s
    if op == "append":
        T, H, KV, hd, page = case["tokens"], case["heads"], case["kv_heads"], case["head_dim"], case["page"]
        dt, ct = DTYPES[case["input"]], DTYPES[case["cache"]]
        # q, k and v rows as one projection writes them
        s["qkv"] = torch.randn(T + case["padding"], (H + 2 * KV) * hd, generator=g, device="cuda").to(dt)
        n_pages = -(-2 * T // page)
        s["k_cache"] = torch.randn(n_pages, page, KV, hd, generator=g, device="cuda").to(ct)
        s["v_cache"] = torch.randn(n_pages, page, KV, hd, generator=g, device="cuda").to(ct)
        slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:T]
        s["slots"] = torch.cat([slots, slots.new_full((case["padding"],), -1)])
        context = 4096
        s["positions"] = torch.randint(0, context, (T + case["padding"],), generator=g, device="cuda", dtype=torch.int32)
        inv = ROPE_BASE ** (-torch.arange(0, hd, 2, dtype=torch.float64, device="cuda") / hd)
        angle = torch.arange(context, dtype=torch.float64, device="cuda")[:, None] * inv
        s["rope_cos"], s["rope_sin"] = angle.cos().float(), angle.sin().float()
        s["q_norm"] = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if case["norm"] else None
        s["k_norm"] = 1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if case["norm"] else None
        s["q_out"] = torch.zeros(T + case["padding"], H, hd, dtype=ct, device="cuda")
        return s
    if op == "sample":
        B, V = case["rows"], case["vocab"]
        # a flat bulk, a few likely tokens, and tokens that a grammar forbids
        x = 2.0 * torch.randn(B, V, generator=g, device="cuda")
        likely = torch.randint(0, V, (B, 24), generator=g, device="cuda")
        x.scatter_(1, likely, 4 + 7 * torch.rand(B, 24, generator=g, device="cuda"))
        x.masked_fill_(torch.rand(B, V, generator=g, device="cuda") < 0.02, -math.inf)
        s["logits"] = x.to(DTYPES[case["dtype"]])
        pick = lambda values: torch.tensor(values, device="cuda")[  # noqa: E731
            torch.randint(0, len(values), (B,), generator=g, device="cuda")]
        s["uniform"] = torch.rand(B, generator=g, device="cuda")
        if case["filters"]:
            s["temperature"] = pick([0.6, 0.7, 0.9, 1.0, 1.3])
            if B > 1:
                s["temperature"][seed % B] = 0.0  # a greedy row
            s["top_k"] = pick([0, 20, 50, 400]).to(torch.int32)
            s["top_p"] = pick([0.8, 0.9, 0.95, 1.0])
            s["min_p"] = pick([0.0, 0.0, 0.02, 0.1])
        else:
            s["temperature"] = 0.7 + 0.6 * torch.rand(B, generator=g, device="cuda")
            s["top_k"] = s["top_p"] = s["min_p"] = None
        return s
    lens, new = _attention_lengths(case)
    H, KV, hd, page, dt = case["heads"], case["kv_heads"], case["head_dim"], case["page"], DTYPES[case["dtype"]]
    held = -(-lens // page)
    n_pages = int(held.sum()) + 3
    max_pages = -(-case["context"] // page) + 1
    perm = torch.randperm(n_pages, generator=g, device="cuda")
    s["block_table"] = _pages(held, n_pages, max_pages, perm)
    T = int(new.sum())
    s["q"] = (1.5 * torch.randn(T, H, hd, generator=g, device="cuda")).to(dt)
    s["k_cache"] = torch.randn(n_pages, page, KV, hd, generator=g, device="cuda").to(dt)
    s["v_cache"] = torch.randn(n_pages, page, KV, hd, generator=g, device="cuda").to(dt)
    s["lens"] = torch.from_numpy(lens).to("cuda", torch.int32)
    s["cu_new"] = torch.from_numpy(np.concatenate([[0], np.cumsum(new)])).to("cuda", torch.int32)
    s["scale"] = hd ** -0.5
    s["most"] = (int(new.max()), int(lens.max()))
    s["out"] = torch.zeros_like(s["q"])
    s["lse"] = torch.zeros(T, H, device="cuda") if case["lse"] else None
    s["workspace"] = torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def run(s):
    op = s["case"]["op"]
    if own:
        return {"plan": _own_plan, "append": _own_append, "attention": _own_attention, "sample": _own_sample}[op](s)
    return {"plan": _plan, "append": _append, "attention": _attention, "sample": _sample}[op](s)


def _own_plan(s):
    p = _paged().plan(s["lens"], s["new_lens"], s["block_table"], s["free_ring"], s["ring_state"], s["page"],
                      s["tokens"])
    return {"block_table": s["block_table"], "free_ring": s["free_ring"], "lens": p.lens, "ring_state": p.ring_state,
            "cu_new": p.cu_new, "positions": p.positions, "slots": p.slots, "status": p.status}


def _own_append(s):
    c = s["case"]
    H, KV, hd = c["heads"], c["kv_heads"], c["head_dim"]
    q, k, v = s["qkv"].view(-1, H + 2 * KV, hd).split([H, KV, KV], 1)
    _paged().append(k, v, s["k_cache"], s["v_cache"], s["positions"], s["slots"], s["rope_cos"], s["rope_sin"], q=q,
                    q_norm=s["q_norm"], k_norm=s["k_norm"], eps=EPS, q_out=s["q_out"])
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _own_attention(s):
    _paged().attention(s["q"], s["k_cache"], s["v_cache"], s["block_table"], s["lens"], s["cu_new"], s["workspace"],
                       scale=s["scale"], out=s["out"], lse=s["lse"])
    return {"out": s["out"], "lse": s["lse"]}


def _own_sample(s):
    r = _paged().sample(s["logits"], s["uniform"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                        min_p=s["min_p"])
    return {"token": r.token, "prob": r.prob, "kept": r.kept}


def _plan(s):
    """Pages by prefix sums over the requests: new ones leave the ring at its head, finished requests' join its tail."""
    lens, new, table, ring, page = s["lens"].long(), s["new_lens"].long(), s["block_table"], s["free_ring"], s["page"]
    head, tail = s["ring_state"][0], s["ring_state"][1]
    add, done = new.clamp(min=0), new < 0
    held = (lens + page - 1) // page
    need = (lens + add + page - 1) // page - held
    back = torch.where(done, held, 0)
    need_before, back_before = torch.cumsum(need, 0) - need, torch.cumsum(back, 0) - back
    col = torch.arange(table.shape[1], device=table.device)
    at = (head + need_before[:, None] + col - held[:, None]) % ring.numel()
    taken = (col >= held[:, None]) & (col < (held + need)[:, None])
    table.copy_(torch.where(taken, ring[at], table))
    # the ring's entry j takes the released page number (j - tail) mod its size, where there is one
    nth = (torch.arange(ring.numel(), device=ring.device) - tail) % ring.numel()
    total = back.sum()
    row = torch.searchsorted(torch.cumsum(back, 0), nth, right=True).clamp(max=lens.numel() - 1)
    page_of = table[row, (nth - back_before[row]).clamp(0, table.shape[1] - 1)]
    ring.copy_(torch.where(nth < total, page_of, ring))
    state = torch.stack([head + need.sum(), tail + total])
    cu = torch.cat([lens.new_zeros(1), torch.cumsum(add, 0)])
    t = torch.arange(s["tokens"], device=table.device)
    of = torch.searchsorted(cu[1:], t, right=True).clamp(max=lens.numel() - 1)
    live = t < cu[-1]
    pos = torch.where(live, lens[of] + t - cu[of], 0)
    slot = table[of, (pos // page).clamp(max=table.shape[1] - 1)].long() * page + pos % page
    status = torch.stack([state.new_zeros(()), state[1] - state[0]]).to(torch.int32)
    return {"block_table": table, "free_ring": ring, "lens": torch.where(done, 0, lens + add).to(torch.int32),
            "ring_state": state, "cu_new": cu.to(torch.int32), "positions": pos.to(torch.int32),
            "slots": torch.where(live, slot, -1), "status": status}


def _turned(x, weight, cos, sin):
    """RMSNorm by head (with a weight), then the rotation of the pairs (d, d + head_dim / 2)."""
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * weight
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _append(s):
    c = s["case"]
    H, KV, hd = c["heads"], c["kv_heads"], c["head_dim"]
    live = s["slots"] >= 0
    q, k, v = s["qkv"][live].float().view(-1, H + 2 * KV, hd).split([H, KV, KV], 1)
    pos, at = s["positions"][live].long(), s["slots"][live]
    cos, sin = s["rope_cos"][pos][:, None], s["rope_sin"][pos][:, None]
    s["q_out"][live] = _turned(q, s["q_norm"], cos, sin).to(s["q_out"].dtype)
    s["k_cache"].view(-1, KV, hd)[at] = _turned(k, s["k_norm"], cos, sin).to(s["k_cache"].dtype)
    s["v_cache"].view(-1, KV, hd)[at] = v.to(s["v_cache"].dtype)
    return {"q": s["q_out"], "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention(s):
    """Every request padded to the longest: gathered K and V, masked scores, softmax, product."""
    q, kc, vc, lens, cu = s["q"], s["k_cache"], s["v_cache"], s["lens"].long(), s["cu_new"].long()
    T, H, hd = q.shape
    page, KV, R = kc.shape[1], kc.shape[2], lens.numel()
    most_new, most_len = s["most"]
    key = torch.arange(most_len, device=q.device)
    there = key < lens[:, None]
    page_of = torch.where(there, s["block_table"][:, key // page].long(), 0)
    k = kc[page_of, key % page].float()  # [R, len, KV, hd]
    v = torch.where(there[..., None, None], vc[page_of, key % page].float(), 0)
    j = torch.arange(most_new, device=q.device)
    new = cu[1:] - cu[:-1]
    padded = q[(cu[:-1, None] + j).clamp(max=T - 1)].float().view(R, most_new, KV, H // KV, hd)
    score = torch.einsum("rjkgd,rlkd->rkgjl", padded, k).mul_(s["scale"])
    seen = key <= (lens - new)[:, None, None] + j[:, None]  # [R, new, len]
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0, top)
    weight = score.sub_(top).exp_()
    total = weight.sum(-1, keepdim=True)
    out = torch.einsum("rkgjl,rlkd->rjkgd", weight, v) / total.clamp(min=1e-38).permute(0, 3, 1, 2, 4)
    t = torch.arange(T, device=q.device)
    of = torch.searchsorted(cu[1:], t, right=True)
    s["out"].copy_(out.reshape(R, most_new, H, hd)[of, t - cu[of]].to(q.dtype))
    if s["lse"] is not None:
        lse = (top + total.log()).squeeze(-1).permute(0, 3, 1, 2).reshape(R, most_new, H)
        s["lse"].copy_(lse[of, t - cu[of]])
    return {"out": s["out"], "lse": s["lse"]}


def _sample(s):
    """Tokens in order of their logits (equal ones by index); the kept ones are a prefix, and so is what the draw passes."""
    x = s["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    B, V = x.shape
    value, index = torch.sort(x, dim=1, descending=True, stable=True)
    temp = s["temperature"].double()[:, None] if s["temperature"] is not None else 1.0
    away = torch.where(value == value[:, :1], 0.0, (value.double() - value[:, :1].double()) / temp)
    weight = torch.where(value == -math.inf, 0.0, away.exp())
    mass = torch.cumsum(weight, 1)
    kept = (value != -math.inf).sum(1)
    if s["top_k"] is not None:
        kept = torch.where(s["top_k"] > 0, torch.minimum(kept, s["top_k"].long()), kept)
    if s["top_p"] is not None:
        top_p = s["top_p"].double()
        before = (mass < top_p[:, None] * mass[:, -1:]).sum(1)
        kept = torch.where(s["top_p"] >= TOP_P_OFF, kept, torch.minimum(kept, before + 1))
    if s["min_p"] is not None:
        likely = (weight >= s["min_p"].double()[:, None]).sum(1)
        kept = torch.where(s["min_p"] > 0, torch.minimum(kept, likely), kept)
    kept = kept.clamp(min=1)
    if s["temperature"] is not None:
        kept = torch.where(s["temperature"] > GREEDY_BELOW, kept, 1)
    norm = mass.gather(1, kept[:, None] - 1)
    passed = (mass < s["uniform"].double()[:, None] * norm).sum(1)
    at = torch.minimum(passed, kept - 1)[:, None]
    prob = (weight.gather(1, at) / norm).float()
    return {"token": index.gather(1, at)[:, 0].to(torch.int32), "prob": prob[:, 0], "kept": kept.to(torch.int32)}


# ---------------------------------------------------------------------------------------------------------------------
# from the definition, in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"plan": _exact_plan, "append": _exact_append, "attention": _exact_attention, "sample": _exact_sample}[
        case["op"]](s)


def _exact_plan(s):
    """Request by request, as a scheduler on the host would."""
    lens, new = s["lens"].tolist(), s["new_lens"].tolist()
    table, ring, page = s["block_table"].cpu().numpy(), s["free_ring"].cpu().numpy(), s["page"]
    head, tail = s["ring_state"].tolist()
    cu, positions, slots, total = [0], [], [], []
    for r, (n, a) in enumerate(zip(lens, new)):
        held = -(-n // page)
        if a < 0:
            for j in range(held):
                ring[tail % len(ring)] = table[r, j]
                tail += 1
        for j in range(held, -(-(n + max(a, 0)) // page)):
            table[r, j] = ring[head % len(ring)]
            head += 1
        for p in range(n, n + max(a, 0)):
            positions.append(p)
            slots.append(int(table[r, p // page]) * page + p % page)
        total.append(0 if a < 0 else n + a)
        cu.append(len(positions))
    pad = s["tokens"] - len(positions)
    return {"block_table": table, "free_ring": ring, "lens": np.array(total, np.int32),
            "ring_state": np.array([head, tail]), "cu_new": np.array(cu, np.int32),
            "positions": np.array(positions + [0] * pad, np.int32), "slots": np.array(slots + [-1] * pad, np.int64),
            "status": np.array([0, tail - head], np.int32)}


def _exact_append(s):
    c = s["case"]
    H, KV, hd = c["heads"], c["kv_heads"], c["head_dim"]
    T = c["tokens"]
    x = s["qkv"][:T].double().view(T, H + 2 * KV, hd)
    half = hd // 2
    cos, sin = (s[n].double()[s["positions"][:T].long()] for n in ("rope_cos", "rope_sin"))

    def head_rows(rows, weight):
        if weight is not None:
            rows = rows / ((rows ** 2).sum(-1, keepdim=True) / hd + EPS).sqrt() * weight.double()
        out = torch.empty_like(rows)
        out[..., :half] = rows[..., :half] * cos[:, None] - rows[..., half:] * sin[:, None]
        out[..., half:] = rows[..., half:] * cos[:, None] + rows[..., :half] * sin[:, None]
        return out

    q_out, kc, vc = s["q_out"].double(), s["k_cache"].double(), s["v_cache"].double()
    q_out[:T] = head_rows(x[:, :H], s["q_norm"])
    at = s["slots"][:T]
    page = kc.shape[1]
    kc[at // page, at % page] = head_rows(x[:, H:H + KV], s["k_norm"])
    vc[at // page, at % page] = x[:, H + KV:]
    return {"q": q_out, "k_cache": kc, "v_cache": vc}


def _exact_attention(s):
    """Request by request and head by head."""
    q, cu, lens = s["q"], s["cu_new"].tolist(), s["lens"].tolist()
    T, H, hd = q.shape
    page, KV = s["k_cache"].shape[1], s["k_cache"].shape[2]
    out = torch.zeros(T, H, hd, dtype=torch.float64, device="cuda")
    lse = torch.zeros(T, H, dtype=torch.float64, device="cuda")
    for r, n in enumerate(lens):
        pages = s["block_table"][r, : -(-n // page)].long()
        k = s["k_cache"][pages].reshape(-1, KV, hd)[:n].double()
        v = s["v_cache"][pages].reshape(-1, KV, hd)[:n].double()
        rows = slice(cu[r], cu[r + 1])
        last = torch.arange(n - (cu[r + 1] - cu[r]), n, device="cuda")
        hidden = torch.arange(n, device="cuda") > last[:, None]
        for h in range(H):
            score = q[rows, h].double() @ k[:, h * KV // H].T * s["scale"]
            score[hidden] = -math.inf
            lse[rows, h] = torch.logsumexp(score, 1)
            out[rows, h] = torch.exp(score - lse[rows, h, None]) @ v[:, h * KV // H]
    return {"out": out, "lse": lse if s["lse"] is not None else None}


def _exact_sample(s):
    """Row by row on the host: order the tokens, cut, draw."""
    logits = s["logits"].double().cpu().numpy()
    B, V = logits.shape
    get = lambda name, off: s[name].cpu().numpy() if s[name] is not None else np.full(B, off)  # noqa: E731
    temp, top_k, top_p, min_p = (get(n, o) for n, o in (("temperature", 1.0), ("top_k", 0), ("top_p", 1.0), ("min_p", 0.0)))
    uniform = s["uniform"].cpu().numpy()
    token, prob, count = np.zeros(B, np.int32), np.zeros(B), np.zeros(B, np.int32)
    for b in range(B):
        x = logits[b]
        if temp[b] <= GREEDY_BELOW:
            token[b], prob[b], count[b] = int(np.argmax(x)), 1.0, 1
            continue
        order = np.lexsort((np.arange(V), -x))
        order = order[np.isfinite(x[order])]
        w = np.exp((x[order] - x[order[0]]) / float(temp[b]))
        sums = np.cumsum(w)
        n = len(order)
        if top_k[b] > 0:
            n = min(n, int(top_k[b]))
        if top_p[b] < TOP_P_OFF:
            n = min(n, int(np.searchsorted(sums, float(top_p[b]) * sums[-1], side="left")) + 1)
        if min_p[b] > 0:
            n = max(1, min(n, int((w >= float(min_p[b])).sum())))
        i = min(n - 1, int(np.searchsorted(sums, float(uniform[b]) * sums[n - 1], side="left")))
        token[b], prob[b], count[b] = order[i], w[i] / sums[n - 1], n
    return {"token": token, "prob": prob, "kept": count}
