"""Paged serving operators: refusals on the CPU, every operator against plain implementations on the GPU.

Tolerances: a result computed in f32 and rounded once to type t is off by at most eps(t) / 2 of its value, plus the
f32 arithmetic's own error, which the test of each operator states.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ------------------------------------------------------------------ refusals (CPU: nothing is launched)
def _refused(fn, *args):
    err = C.create_string_buffer(512)
    assert fn(*args, None, err, 512) == 0
    assert err.value.startswith(b"error: paged")
    return err.value.decode()


def _cache_struct(**kw):
    from minicpmo_b200.gpu import PagedCache

    c = dict(k=4096, v=8192, dtype=1, page_size=16, kv_heads=2, head_dim=64, n_pages=8, page_stride=2048, token_stride=128,
             head_stride=64)
    c.update(kw)
    return PagedCache(**c)


def test_plan_refusals(pkg):
    fn = pkg.lib().minicpmo_gpu_paged_plan
    p = 4096  # a pointer that no check may follow
    good = [p, p + 64, 4, p, 8, 8, p, 32, p, 16, 64, p, p, p + 128, p, p, p]

    def bad(**kw):
        a = list(good)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return _refused(fn, *a)

    assert "null" in bad(_0=None) and "null" in bad(_14=None)
    assert "requests" in bad(_2=0) and "requests" in bad(_2=8193)
    assert "page_size" in bad(_9=24) and "page_size" in bad(_9=4) and "page_size" in bad(_9=512)
    assert "table rows" in bad(_4=0) and "table rows" in bad(_5=7)
    assert "ring" in bad(_7=0)
    assert "capacity" in bad(_10=1 << 31)
    assert "only lens_out" in bad(_13=p) and "only lens_out" in bad(_11=p + 64)


@pytest.mark.parametrize("kw, word", [
    (dict(k=None), "null"), (dict(dtype=6), "dtype"), (dict(page_size=48), "page_size"), (dict(head_dim=96), "head_dim"),
    (dict(kv_heads=0), "kv heads"), (dict(n_pages=0), "pages"), (dict(token_stride=64), "overlap"),
    (dict(page_stride=1024), "overlap"), (dict(head_stride=32), "overlap"), (dict(k=4100), "16 bytes"),
    (dict(token_stride=132), "16 bytes"), (dict(page_stride=1 << 41), "range"),
])
def test_cache_refusals(pkg, kw, word):
    lib, p = pkg.lib(), 4096
    c = C.byref(_cache_struct(**kw))
    if kw == dict(token_stride=132):
        c = C.byref(_cache_struct(token_stride=132, page_stride=132 * 16))
    assert word in _refused(lib.minicpmo_gpu_paged_append, c, None, p, p, 0, 4, 0, 0, 128, 128, None, None, 1e-6, p, p, 64, p,
                            p, None, 0, None)
    assert word in _refused(lib.minicpmo_gpu_paged_attention, c, p, 4, 4, 256, p, 8, 8, p, p, 2, 0.125, p, 256, None, p)


def test_append_refusals(pkg):
    fn, p = pkg.lib().minicpmo_gpu_paged_append, 4096
    good = [C.byref(_cache_struct()), p, p, p, 0, 4, 4, 512, 512, 512, None, None, 1e-6, p, p, 64, p, p, p, 256, None]

    def bad(**kw):
        a = list(good)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return _refused(fn, *a)

    assert "input dtype" in bad(_4=8)
    assert "null" in bad(_2=None) and "null" in bad(_18=None) and "null" in bad(_17=None)
    assert "table rows" in bad(_15=0) and "tokens" in bad(_5=1 << 25)
    assert "overlap" in bad(_8=64) and "overlap" in bad(_7=255) and "overlap" in bad(_19=128)
    assert "16 bytes" in bad(_2=4100) and "16 bytes" in bad(_9=513)
    assert "too many rows" in bad(_5=1 << 24, _6=8192, _7=8192 * 64, _19=8192 * 64)


def test_attention_refusals(pkg):
    fn, p = pkg.lib().minicpmo_gpu_paged_attention, 4096
    good = [C.byref(_cache_struct()), p, 4, 4, 256, p, 8, 8, p, p, 2, 0.125, p, 256, None, p]

    def bad(**kw):
        a = list(good)
        for i, v in kw.items():
            a[int(i[1:])] = v
        return _refused(fn, *a)

    assert "null" in bad(_1=None) and "null" in bad(_15=None) and "null" in bad(_9=None)
    assert "requests" in bad(_10=0) and "requests" in bad(_10=8193)
    assert "q heads" in bad(_3=3) and "q heads" in bad(_3=1) and "q heads" in bad(_3=34)
    assert "table rows" in bad(_6=0) and "table rows" in bad(_7=7) and "table rows" in bad(_6=1 << 31, _7=1 << 31)
    assert "overlap" in bad(_4=255) and "overlap" in bad(_13=128)
    assert "multiples" in bad(_15=4096 + 16) and "multiples" in bad(_1=4104) and "multiples" in bad(_4=260)
    assert "finite" in bad(_11=math.inf) and "finite" in bad(_11=math.nan)


def test_tensor_checks_raise(pkg):
    """The Python entry points refuse tensors of the wrong kind before the library is called."""
    from minicpmo_b200 import paged
    from minicpmo_b200.gpu import GpuError

    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(GpuError, match="CUDA"):
        paged.plan(i, i, i.view(2, 2), i, torch.zeros(2, dtype=torch.int64), 16, 8)
    k = torch.zeros(2, 16, 2, 64)
    with pytest.raises(GpuError, match="CUDA"):
        paged.append(k[0], k[0], k, k, i, i.long(), i, i)
    with pytest.raises(GpuError, match="alike"):
        paged.attention(k[0], k, k.half(), i.view(2, 2), i, i, i)


# ------------------------------------------------------------------ helpers
def _table(rng, held, max_pages, n_pages):
    """A block table whose rows hold distinct pages, and the pages left; stale entries are far out of range."""
    perm = rng.permutation(n_pages).astype(np.int32)
    table = np.full((len(held), max_pages), -7777, np.int32)
    at = 0
    for r, n in enumerate(held):
        table[r, :n] = perm[at:at + n]
        at += n
    return table, perm[at:]


def cuda(x, dtype=None):
    return torch.as_tensor(x, dtype=dtype).cuda()


# ------------------------------------------------------------------ plan
def plan_reference(lens, new, table, ring, state, page, capacity):
    """Request by request on the host."""
    lens, new, table, ring = list(lens), list(new), table.copy(), ring.copy()
    head, tail = state
    n, cap, width = len(lens), len(ring), table.shape[1]
    ceil = lambda a: -(-a // page)  # noqa: E731
    flags = 0
    if any(l < 0 or a < -1 for l, a in zip(lens, new)):
        flags |= 8
    ok = [(l, a) for l, a in zip(lens, new) if l >= 0 and a >= -1]
    if any(ceil(l + max(a, 0)) > width for l, a in ok):
        flags |= 2
    back = sum(ceil(l) for l, a in ok if a < 0)
    if head < 0 or tail < head or tail - head > cap or tail - head + back > cap:
        flags |= 16
    if sum(ceil(l + max(a, 0)) - ceil(l) for l, a in ok) > tail - head:
        flags |= 1
    if sum(max(a, 0) for _, a in ok) > capacity:
        flags |= 4
    if flags:
        return dict(lens=lens, state=[head, tail], cu=[0] * (n + 1), pos=[0] * capacity, slots=[-1] * capacity,
                    status=[flags, max(0, tail - head)], table=table, ring=ring)
    cu, pos, slots, out = [0], [], [], []
    for r in range(n):
        l, a = lens[r], max(new[r], 0)
        if new[r] < 0:
            for j in range(ceil(l)):
                ring[tail % cap] = table[r, j]
                tail += 1
        for j in range(ceil(l), ceil(l + a)):
            table[r, j] = ring[head % cap]
            head += 1
        for p in range(l, l + a):
            pos.append(p)
            slots.append(int(table[r, p // page]) * page + p % page)
        cu.append(len(pos))
        out.append(0 if new[r] < 0 else l + a)
    rest = capacity - len(pos)
    return dict(lens=out, state=[head, tail], cu=cu, pos=pos + [0] * rest, slots=slots + [-1] * rest,
                status=[0, tail - head], table=table, ring=ring)


def _plan_case(seed, n, page, max_len, chunk, done, spare, ring_extra=0):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, max_len + 1, n)
    new = np.where(rng.random(n) < 0.5, 1, rng.integers(0, chunk + 1, n))
    new[rng.random(n) < done] = -1
    held = -(-lens // page)
    want = -(-(lens + np.maximum(new, 0)) // page)
    n_pages = int(want.sum()) + spare
    table, free = _table(rng, held, -(-(max_len + chunk) // page), n_pages)
    cap = n_pages + ring_extra
    head = int(rng.integers(0, 10 * cap))
    ring = np.full(cap, -5, np.int32)
    ring[(head + np.arange(len(free))) % cap] = free
    return lens, new, table, ring, [head, head + len(free)]


def _run_plan(paged, lens, new, table, ring, state, page, capacity, in_place=False):
    d = dict(lens=cuda(lens, torch.int32), new=cuda(new, torch.int32), table=cuda(table), ring=cuda(ring),
             state=cuda(state, torch.int64))
    out = None
    if in_place:
        z = lambda k, t: torch.full((k,), 99, dtype=t, device="cuda")  # noqa: E731
        out = paged.PagedPlan(d["lens"], d["state"], z(len(lens) + 1, torch.int32), z(capacity, torch.int32),
                              z(capacity, torch.int64), z(2, torch.int32))
    p = paged.plan(d["lens"], d["new"], d["table"], d["ring"], d["state"], page, capacity, out=out)
    got = dict(lens=p.lens, state=p.ring_state, cu=p.cu_new, pos=p.positions, slots=p.slots, status=p.status,
               table=d["table"], ring=d["ring"])
    return {k: v.cpu().numpy() for k, v in got.items()}


def _same(got, want):
    for k, v in want.items():
        assert np.array_equal(got[k], np.asarray(v)), k


@pytest.mark.gpu
@pytest.mark.parametrize("seed, n, page, max_len, chunk, done, spare", [
    (1, 1, 16, 0, 1, 0, 0), (2, 1, 8, 100, 70, 0, 3), (3, 32, 16, 500, 1, 0, 5), (4, 33, 64, 900, 200, 0.2, 1),
    (5, 257, 16, 300, 40, 0.1, 0), (6, 1025, 32, 100, 9, 0.5, 7), (7, 8192, 16, 60, 3, 0.1, 2), (8, 5, 256, 3000, 5000, 0, 0),
    (9, 40, 128, 700, 0, 1.0, 0), (10, 3, 16, 16, 16, 0, 0),
])
@pytest.mark.parametrize("in_place", [False, True])
def test_plan_matches_the_host(pkg, seed, n, page, max_len, chunk, done, spare, in_place):
    from minicpmo_b200 import paged

    case = _plan_case(seed, n, page, max_len, chunk, done, spare, ring_extra=seed % 3)
    total = int(np.maximum(case[1], 0).sum())
    for capacity in {total, total + 37}:
        _same(_run_plan(paged, *case, page, capacity, in_place), plan_reference(*case, page, capacity))


@pytest.mark.gpu
def test_plan_refuses_whole_steps(pkg):
    from minicpmo_b200 import paged

    lens, new, table, ring, (head, tail) = _plan_case(11, 6, 16, 200, 50, 0, 0)
    total = int(new.sum())
    width = table.shape[1]
    longest = np.array(new)
    longest[0] = width * 16 + 1 - lens[0]
    cases = [
        (lens, new, table, ring, [head, tail - 1], total, 1),
        (lens, longest, table, ring, [head, head + len(ring)], 10 ** 6, 2),
        (lens, new, table, ring, [head, tail], total - 1, 4),
        (np.where(np.arange(6) == 3, -1, lens), new, table, ring, [head, tail], total, 8),
        (lens, np.where(np.arange(6) == 2, -2, new), table, ring, [head, tail], total, 8),
        (lens, new, table, ring, [head, head - 1], total, 16),
        (lens, new, table, ring, [head, head + len(ring) + 1], total, 16),
        (lens, new, table, ring, [-1, tail], total, 16),
    ]
    for l, a, t, r, state, capacity, flag in cases:
        want = plan_reference(l, a, t, r, state, 16, capacity)
        assert want["status"][0] & flag
        _same(_run_plan(paged, l, a, t, r, state, 16, capacity), want)


# ------------------------------------------------------------------ append
@pytest.mark.gpu
@pytest.mark.parametrize("heads, kv, hd", [(8, 2, 128), (3, 1, 64), (5, 5, 256), (0, 3, 128)])
@pytest.mark.parametrize("src, dst", [("f32", "f16"), ("f32", "f32"), ("bf16", "bf16"), ("f16", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("tokens, norm, heads_out", [(1, True, False), (67, True, True), (130, False, False)])
def test_append(pkg, heads, kv, hd, src, dst, tokens, norm, heads_out):
    """Against 64 bits: three f32 roundings each in the norm's factor and the rotation, a sum of hd squares (relative
    error below hd * 2^-24 / 2 after the root), one rounding to the cache's type."""
    from minicpmo_b200 import paged

    g = torch.Generator(device="cuda").manual_seed(hd + tokens)
    page, context = 16, 77
    n_pages = -(-tokens // page) + 3
    packed = torch.randn(tokens, (heads + 2 * kv) * hd, generator=g, device="cuda").to(DT[src])
    q, k, v = packed.view(tokens, -1, hd).split([heads, kv, kv], 1)
    if heads_out:  # pages of [kv, page, hd]
        kc, vc = (torch.randn(n_pages, kv, page, hd, generator=g, device="cuda").to(DT[dst]).transpose(1, 2) for _ in "kv")
    else:  # all layers' rows in one page, this layer the second
        kc, vc = (torch.randn(n_pages, 2, page, kv, hd, generator=g, device="cuda").to(DT[dst])[:, 1] for _ in "kv")
    before = kc.clone(), vc.clone()
    slots = torch.randperm(n_pages * page, generator=g, device="cuda")[:tokens]
    slots[::5] = -1
    positions = torch.randint(0, context, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    if tokens > 10:
        positions[-1], slots[-2] = context, n_pages * page  # out of range: left out, and reported
    cos, sin = (torch.randn(context, hd // 2, generator=g, device="cuda") for _ in "cs")
    qn, kn = ((1 + torch.randn(hd, generator=g, device="cuda"), 1 + torch.randn(hd, generator=g, device="cuda")) if norm
              else (None, None))
    q_out = torch.full((tokens, heads, hd), 7.0, device="cuda").to(DT[dst]) if heads else None
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    got = paged.append(k, v, kc, vc, positions, slots, cos, sin, q=q if heads else None, q_norm=qn, k_norm=kn, eps=1e-6,
                       q_out=q_out, status=status)
    assert int(status) == ((3 if (tokens - 1) % 5 and (tokens - 2) % 5 else int(status)) if tokens > 10 else 0)

    live = (slots >= 0) & (slots < n_pages * page) & (positions < context)
    p, at = positions[live].long(), slots[live]

    def turned(x, w):
        x = x[live].double()
        if w is not None:
            x = x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        a, b = x.chunk(2, -1)
        c, s = cos[p].double()[:, None], sin[p].double()[:, None]
        # error of the rotation: of both products, not of their sum
        size = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()], -1)
        return torch.cat([a * c - b * s, b * c + a * s], -1), size

    def close(x, want, size):
        tol = torch.finfo(DT[dst]).eps / 2 * want.abs() + (hd / 2 + 8) * 2.0 ** -24 * size + torch.finfo(DT[dst]).tiny
        assert ((x.double() - want).abs() <= tol).all()

    wk, wv = before[0].clone(), before[1].clone()
    wv[at // page, at % page] = v[live].to(DT[dst])
    assert torch.equal(vc, wv)
    want, size = turned(k, kn)
    close(kc[at // page, at % page], want, size)
    kc2 = kc.clone()
    kc2[at // page, at % page] = wk[at // page, at % page]
    assert torch.equal(kc2, wk)  # nothing else was written
    if heads:
        assert got is q_out
        want, size = turned(q, qn)
        close(q_out[live], want, size)
        assert (q_out[~live] == 7.0).all()


# ------------------------------------------------------------------ attention
def attention_reference(q, kc, vc, table, lens, cu, scale):
    """64 bits, request by request; also sum_i w_i |V_i|, the scale of the weights' rounding errors."""
    T, H, hd = q.shape
    page, kv = kc.shape[1], kc.shape[2]
    out, mag = (torch.zeros(T, H, hd, dtype=torch.float64, device=q.device) for _ in "om")
    lse = torch.full((T, H), -math.inf, dtype=torch.float64, device=q.device)
    for r, n in enumerate(lens):
        rows = slice(cu[r], cu[r + 1])
        m = cu[r + 1] - cu[r]
        if m == 0 or n == 0:
            continue
        ids = table[r, : -(-n // page)].long()
        k = kc[ids].flatten(0, 1)[:n].double()
        v = vc[ids].flatten(0, 1)[:n].double()
        seen = torch.arange(n, device=q.device) <= torch.arange(n - m, n, device=q.device)[:, None]
        for h in range(H):
            s = (q[rows, h].double() @ k[:, h * kv // H].T * scale).masked_fill(~seen, -math.inf)
            l = torch.logsumexp(s, 1)
            w = torch.where(l[:, None] == -math.inf, 0.0, torch.exp(s - l[:, None]))
            lse[rows, h] = l
            hv = v[:, h * kv // H]
            # a row sees none of the values behind it, whatever they are
            if torch.isfinite(hv).all():
                out[rows, h], mag[rows, h] = w @ hv, w @ hv.abs()
            else:
                for i in range(m):
                    e = max(0, n - m + i + 1)
                    out[cu[r] + i, h], mag[cu[r] + i, h] = w[i, :e] @ hv[:e], w[i, :e] @ hv[:e].abs()
    return out, lse, mag


def _attention_case(seed, dtype, hd, heads, kv, page, reqs, heads_out=False, spoil=True):
    """reqs: (length, new tokens) of each; rows behind the lengths, free pages and stale table entries hold NaN and worse."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    lens, new = [a for a, _ in reqs], [b for _, b in reqs]
    held = [-(-a // page) for a in lens]
    n_pages = sum(held) + 2
    max_pages = max(held) + 2
    table, _ = _table(rng, held, max_pages, n_pages)
    shape = (n_pages, kv, page, hd) if heads_out else (n_pages, page, kv, hd)
    kc, vc = (torch.randn(shape, generator=g, device="cuda").to(DT[dtype]) for _ in "kv")
    if heads_out:
        kc, vc = kc.transpose(1, 2), vc.transpose(1, 2)
    if spoil:
        used = torch.zeros(n_pages, page, dtype=torch.bool)
        for r, a in enumerate(lens):
            for p in range(a):
                used[table[r, p // page], p % page] = True
        kc[~used.cuda()] = math.nan
        vc[~used.cuda()] = math.inf
    cu = np.concatenate([[0], np.cumsum(new)])
    T = int(cu[-1]) + 5  # a padded batch
    packed = torch.randn(T, heads + 3, hd, generator=g, device="cuda").to(DT[dtype])
    return dict(q=packed[:, :heads] * 1.5, kc=kc, vc=vc, table=cuda(table), lens=lens, cu=cu.tolist(), T=T)


def _run_attention(paged, c, ws, scale=None):
    q = c["q"]
    out = torch.full(q.shape, 3.0, dtype=q.dtype, device="cuda")
    lse = torch.full(q.shape[:2], 3.0, device="cuda")
    paged.attention(q, c["kc"], c["vc"], c["table"], cuda(c["lens"], torch.int32), cuda(c["cu"], torch.int32), ws,
                    scale=scale, out=out, lse=lse)
    return out, lse


def _check_attention(c, out, lse, scale=None):
    """f32: scores off by (hd + 2) 2^-24 of sum |q k| scale, which moves every weight by that; sums of n terms by n 2^-24,
    the bound taken at half the terms (they are added in tiles).  f16, bf16: products are exact in f32, weights and the
    result are rounded once each (f16 weights below 2^-14 of the largest by at most 2^-25 of it)."""
    q, dt = c["q"], c["q"].dtype
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    live = c["cu"][-1]
    want, wlse, mag = attention_reference(q[:live], c["kc"], c["vc"], c["table"], c["lens"], c["cu"], scale)
    assert (out[live:] == 3.0).all() and (lse[live:] == 3.0).all()
    n, hd = max(c["lens"] + [1]), q.shape[-1]
    kmax = 1.0
    for r, a in enumerate(c["lens"]):
        if a and c["cu"][r + 1] > c["cu"][r]:
            ids = c["table"][r, : -(-a // c["kc"].shape[1])].long()
            k = c["kc"][ids].flatten(0, 1)[:a].double()
            kmax = max(kmax, float(k[torch.isfinite(k)].abs().max()))
    score = (hd + 2) * 2.0 ** -24 * float(q[:live].double().abs().sum(-1).max()) * kmax * abs(scale) * 0.5 + 2.0 ** -21
    tol_lse = score + n * 2.0 ** -25 + 2.0 ** -23 * wlse.abs().clamp(max=1e30)
    nothing = wlse == -math.inf
    assert torch.equal(lse[:live] == -math.inf, nothing)
    assert ((lse[:live].double() - wlse).abs() <= tol_lse)[~nothing].all()
    half = torch.finfo(dt).eps / 2
    weights = 0.0 if dt == torch.float32 else half
    tiny = 2.0 ** -24 * n if dt == torch.float16 else 0.0
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(out[:live]), fine)
    assert torch.equal(torch.isnan(out[:live]), torch.isnan(want))
    inf = torch.isinf(want)
    assert torch.equal(out[:live][inf].double(), want[inf])
    tol = half * want.abs() + (weights + 2 * score + n * 2.0 ** -24) * mag + tiny + torch.finfo(dt).tiny
    assert ((out[:live].double() - want).abs() <= tol)[fine].all()


F32_CASES = [
    (128, 4, 2, 16, [(1, 1)]), (64, 8, 8, 32, [(65, 1), (33, 33), (0, 0), (7, 3)]), (128, 14, 2, 16, [(130, 1), (257, 40)]),
    (256, 4, 1, 64, [(300, 2), (5, 5), (129, 129)]), (64, 16, 1, 8, [(31, 31), (32, 32), (33, 1)]),
    (128, 8, 2, 128, [(1000, 1)] * 5 + [(2, 1)] * 40), (64, 3, 1, 16, [(0, 2), (3, 5), (40, 7)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(len(F32_CASES)))
@pytest.mark.parametrize("heads_out", [False, True])
def test_attention_f32(pkg, case, heads_out):
    from minicpmo_b200 import paged

    hd, heads, kv, page, reqs = F32_CASES[case]
    c = _attention_case(100 + case, "f32", hd, heads, kv, page, reqs, heads_out)
    ws = paged.workspace()
    first = _run_attention(paged, c, ws)
    _check_attention(c, *first)
    again = _run_attention(paged, c, ws)  # the workspace is ready again, and the result does not move
    assert all(torch.equal(a, b) for a, b in zip(first, again))


CASES_16 = F32_CASES + [
    (128, 32, 8, 16, [(565, 1)]), (128, 8, 2, 8, [(77, 1), (1, 1), (64, 64), (65, 65), (63, 2)]),
    (128, 16, 1, 256, [(4096, 1), (17, 2)]), (64, 12, 4, 16, [(129, 129), (700, 5), (128, 128), (4, 4)]),
    (256, 16, 2, 32, [(513, 3), (64, 1)]), (128, 28, 4, 64, [(900, 300), (257, 257), (2, 2)]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("case", range(len(CASES_16)))
@pytest.mark.parametrize("heads_out", [False, True])
def test_attention_16_bits(pkg, dtype, case, heads_out):
    from minicpmo_b200 import paged

    hd, heads, kv, page, reqs = CASES_16[case]
    c = _attention_case(200 + case, dtype, hd, heads, kv, page, reqs, heads_out)
    ws = paged.workspace()
    first = _run_attention(paged, c, ws)
    _check_attention(c, *first)
    again = _run_attention(paged, c, ws)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd, heads, kv, reqs", [(128, 4, 2, [(40, 12), (300, 5)]), (64, 8, 8, [(600, 500)]),
                                                 (128, 8, 1, [(300, 290), (170, 170)]), (256, 2, 2, [(90, 33)])])
def test_values_behind_a_token_do_not_reach_it(pkg, dtype, hd, heads, kv, reqs):
    """Infinities and NaN in the K and V rows of the newest tokens: tokens before them keep finite results, tokens from
    them on get what the definition gives."""
    from minicpmo_b200 import paged

    c = _attention_case(7, dtype, hd, heads, kv, 16, reqs)
    for r, (n, m) in enumerate(reqs):
        row = lambda p: (int(c["table"][r, p // 16]), p % 16)  # noqa: E731
        c["vc"][row(n - 1)][0, 3] = math.inf
        c["vc"][row(n - 2)][kv - 1, 5] = math.nan
        c["vc"][row(n - m + 1)][0, 0] = -math.inf
        c["kc"][row(n - 1)][kv - 1, 2] = math.nan
    ws = paged.workspace()
    out, lse = _run_attention(paged, c, ws)
    for r, (n, m) in enumerate(reqs):  # only the last token of each request meets the NaN key
        assert torch.isnan(lse[c["cu"][r + 1] - 1, heads - 1]) and torch.isfinite(lse[c["cu"][r]:c["cu"][r + 1] - 1]).all()
        assert torch.isfinite(out[c["cu"][r]]).all()
    live = c["cu"][-1]
    want, _, _ = attention_reference(c["q"][:live], c["kc"], c["vc"], c["table"], c["lens"], c["cu"], hd ** -0.5)
    assert torch.equal(torch.isnan(out[:live]), torch.isnan(want))
    inf = torch.isinf(want)
    assert inf.any() and torch.equal(out[:live][inf].double(), want[inf])
    assert torch.isfinite(out[:live][torch.isfinite(want)]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_of_bad_tables(pkg, dtype):
    """Table entries outside the cache read as rows of zeros; prefix sums and lengths out of range are clamped."""
    from minicpmo_b200 import paged

    c = _attention_case(9, dtype, 128, 4, 2, 16, [(100, 1), (50, 20)])
    c["table"][0, 2], c["table"][1, 1] = -3, c["kc"].shape[0]
    out, lse = _run_attention(paged, c, paged.workspace())
    zero = dict(c)
    pages = c["kc"].shape[0]
    zero["kc"], zero["vc"] = (torch.cat([x, torch.zeros_like(x[:1])]) for x in (c["kc"], c["vc"]))
    zero["table"] = torch.where((c["table"] == -3) | (c["table"] == pages), pages, c["table"])
    _check_attention(zero, out, lse)
    c["cu"] = [-5, 21, c["T"] + 100]
    c["lens"] = [10 ** 9, 60]
    out, _ = _run_attention(paged, c, paged.workspace())
    assert out.shape[0] == c["T"]


@pytest.mark.gpu
def test_negative_scale_and_one_workspace_for_many_shapes(pkg):
    from minicpmo_b200 import paged

    ws = paged.workspace()
    for seed, (dtype, hd, heads, kv, page, reqs) in enumerate([
            ("bf16", 128, 32, 8, 16, [(3000, 1)] * 3), ("f32", 64, 4, 4, 16, [(500, 2)]), ("f16", 64, 8, 2, 32, [(90, 90)] * 9),
            ("bf16", 128, 32, 8, 64, [(1500, 700), (700, 700)]), ("f16", 256, 4, 1, 16, [(5000, 1)])]):
        c = _attention_case(seed, dtype, hd, heads, kv, page, reqs)
        for scale in (-0.05, 0.0, 0.11):
            _check_attention(c, *_run_attention(paged, c, ws, scale), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("hd, heads, kv, page, reqs", [
    (128, 8, 2, 8, [(0, 70), (3, 90), (200, 150), (0, 0), (64, 64)]),  # tokens before the cache's beginning see nothing
    (128, 16, 1, 256, [(900, 130), (257, 257)]), (64, 3, 3, 32, [(129, 128), (500, 129), (128, 1)]),
    (128, 7, 1, 16, [(333, 300), (20, 19)]), (64, 16, 1, 64, [(65, 65)] * 7), (128, 10, 2, 128, [(1000, 513), (4, 4), (700, 1)]),
    (128, 32, 8, 64, [(2500, 600), (1, 1), (3000, 40), (90, 90)]),
])
def test_attention_of_long_chunks(pkg, dtype, hd, heads, kv, page, reqs):
    """Many rows per request: the 256-row blocks, both tiles of them or one, every group size and page size."""
    from minicpmo_b200 import paged

    c = _attention_case(31, dtype, hd, heads, kv, page, reqs, heads_out=page == 16)
    ws = paged.workspace()
    first = _run_attention(paged, c, ws)
    _check_attention(c, *first)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, _run_attention(paged, c, ws)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n_req, chunk", [(1000, 1), (8192, 1), (700, 9)])
def test_attention_of_many_requests(pkg, dtype, n_req, chunk):
    from minicpmo_b200 import paged

    rng = np.random.default_rng(n_req)
    reqs = [(int(n), int(min(n, rng.integers(0, chunk + 1)))) for n in rng.integers(0, 40, n_req)]
    c = _attention_case(5, dtype, 64, 8 if chunk > 1 else 2, 1, 16, reqs, spoil=False)
    _check_attention(c, *_run_attention(paged, c, paged.workspace()))


@pytest.mark.gpu
def test_workspaces_apart_on_two_streams(pkg):
    """Two calls that overlap, each with its own workspace, give what they give alone."""
    from minicpmo_b200 import paged

    a = _attention_case(1, "bf16", 128, 32, 8, 16, [(4000, 1)] * 8)
    b = _attention_case(2, "bf16", 128, 32, 8, 64, [(1200, 600)] * 2)
    wa, wb = paged.workspace(), paged.workspace()
    alone = [_run_attention(paged, a, wa), _run_attention(paged, b, wb)]
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(20):
        with torch.cuda.stream(sa):
            ra = _run_attention(paged, a, wa)
        with torch.cuda.stream(sb):
            rb = _run_attention(paged, b, wb)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for r, s in zip((ra, rb), alone) for x, y in zip(r, s))
