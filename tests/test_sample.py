"""The sampler: refusals on the CPU; tokens, kept counts and probabilities against a 64-bit implementation on the GPU.

The kernel's sums of weights are off by at most vocab * 2^-(shift + 1) of the largest weight (shift = min(50, 62 -
ceil(log2(vocab)))), which is below 2^-24 of it at the sizes here, and usually far less (roundings cancel).  A border
that close to a target decides nothing that the test could: the reference says which targets are nearer than that, and
those rows (none with the seeds used) would be refused by the test itself.  Probabilities are rounded to f32 once.
"""
from __future__ import annotations

import ctypes as C
import math

import numpy as np
import pytest
import torch

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
TOP_P_OFF, GREEDY_BELOW = float(np.float32(0.999999)), float(np.float32(1e-6))


def test_refusals(pkg):
    fn, p = pkg.lib().minicpmo_gpu_sample, 4096
    good = [p, 0, 2, 100, 100, None, None, None, None, p, p, None, None]

    def bad(**kw):
        a = list(good)
        for i, v in kw.items():
            a[int(i[1:])] = v
        err = C.create_string_buffer(512)
        assert fn(*a, None, err, 512) == 0
        assert err.value.startswith(b"error: sample")
        return err.value.decode()

    assert "dtype" in bad(_1=8)
    assert "null" in bad(_0=None) and "null" in bad(_9=None) and "null" in bad(_10=None)
    assert "rows of" in bad(_3=0) and "rows of" in bad(_3=(1 << 19) + 1, _4=1 << 20) and "rows of" in bad(_2=1 << 21)
    assert "apart" in bad(_4=99)
    assert "misaligned" in bad(_0=4098)


def test_tensor_checks_raise(pkg):
    from minicpmo_b200 import paged
    from minicpmo_b200.gpu import GpuError

    with pytest.raises(GpuError, match="CUDA"):
        paged.sample(torch.zeros(2, 8), torch.zeros(2))


def reference(x, u, temp, top_k, top_p, min_p):
    """One row in 64 bits: token, probability, kept, and the distance of the nearest border from its target, in weights."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    n = int((x > -np.inf).sum())
    if n == 0:
        return 0, 0.0, 0, math.inf
    if not temp > GREEDY_BELOW or top_k == 1:
        return int(np.argmax(x)), 1.0, 1, math.inf
    order = np.lexsort((np.arange(len(x)), -x))[:n]
    v = x[order]
    with np.errstate(invalid="ignore"):
        w = np.exp(np.where(v == v[0], 0.0, v - v[0]) / float(temp))
    sums = np.cumsum(w)
    kept, near = n, math.inf

    def reach(target, upto):
        nonlocal near
        i = int(np.searchsorted(sums[:upto], target, side="left"))
        near = min([near] + [abs(sums[j] - target) for j in (i - 1, i) if 0 <= j < upto and target > 0])
        return min(i, upto - 1) + 1

    if top_k > 0:
        kept = min(kept, top_k)
    if top_p < TOP_P_OFF:
        kept = min(kept, reach(max(0.0, float(top_p)) * sums[-1], n))
    if min_p > 0:
        likely = int((w >= float(min_p)).sum())
        near = min([near] + [abs(w[j] - float(min_p)) for j in (likely - 1, likely) if 0 <= j < n and 0 < j])
        kept = min(kept, likely)
    kept = max(kept, 1)
    u = 0.0 if math.isnan(u) else min(max(float(u), 0.0), 1.0)
    if u == 1.0:  # the kept sum itself, whichever way it is added: the last token that weighs anything
        at = int(np.searchsorted(sums[:kept], sums[kept - 1], side="left"))
    else:
        at = reach(u * sums[kept - 1], kept) - 1
    return int(order[at]), w[at] / sums[kept - 1], kept, near


def check(paged, logits, u, temp=None, top_k=None, top_p=None, min_p=None):
    to = lambda v, t: None if v is None else torch.as_tensor(np.asarray(v), dtype=t).cuda()  # noqa: E731
    r = paged.sample(logits, to(u, torch.float32), temperature=to(temp, torch.float32), top_k=to(top_k, torch.int32),
                     top_p=to(top_p, torch.float32), min_p=to(min_p, torch.float32))
    again = paged.sample(logits, to(u, torch.float32), temperature=to(temp, torch.float32), top_k=to(top_k, torch.int32),
                         top_p=to(top_p, torch.float32), min_p=to(min_p, torch.float32))
    assert all(torch.equal(a, b) for a, b in zip(r, again))
    x = logits.double().cpu().numpy()
    f = lambda v, off: np.full(len(x), off) if v is None else np.asarray(v, np.float32)  # noqa: E731
    temp, top_p, min_p = f(temp, 1.0), f(top_p, 1.0), f(min_p, 0.0)
    top_k = np.zeros(len(x), int) if top_k is None else np.asarray(top_k)
    vocab = x.shape[1]
    off = vocab * 2.0 ** -(min(50, 62 - math.ceil(math.log2(vocab))) + 1) if vocab > 1 else 2.0 ** -51
    token, prob, kept = (t.cpu().numpy() for t in r)
    for b in range(len(x)):
        t, p, k, near = reference(x[b], np.float32(u[b]), temp[b], int(top_k[b]), top_p[b], min_p[b])
        assert near > off / 1000, "this seed puts a border on its target: choose another"
        assert (token[b], kept[b]) == (t, k), (b, token[b], t, kept[b], k)
        # the sum's error moves the share by at most its own relative size; the share's f32 rounding adds 2^-24
        assert abs(prob[b] - p) <= (2.0 ** -24 + off + 2.0 ** -50) * p + 1e-45


def logits_of(kind, B, V, dtype, seed, stride=None):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(B, V, generator=g, device="cuda")
    if kind == "likely":
        x = 2 * x
        x[torch.arange(B, device="cuda")[:, None], torch.randint(0, V, (B, 9), generator=g, device="cuda")] += 8
    elif kind == "flat":
        x = 0.01 * x
    elif kind == "steep":
        x = 30 * x
    elif kind == "ties":
        x = (2 * x).round()
    elif kind == "equal":
        x = torch.full_like(x, 1.25)
    elif kind == "masked":
        x = torch.where(torch.rand(B, V, generator=g, device="cuda") < 0.97, -math.inf, x)
        x[:, V // 2] = torch.finfo(DT[dtype]).min
        x[:, V // 3] = 0.5
    x = x.to(DT[dtype])
    if stride:
        wide = torch.full((B, stride), math.nan, device="cuda").to(DT[dtype])
        wide[:, :V] = x
        x = wide[:, :V]
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kind", ["normal", "likely", "flat", "steep", "ties", "equal", "masked"])
@pytest.mark.parametrize("B, V, stride", [(5, 1, None), (7, 37, 41), (3, 4096, None), (12, 50001, None), (4, 151936, 151944)])
def test_matches_the_definition(pkg, dtype, kind, B, V, stride):
    from minicpmo_b200 import paged

    x = logits_of(kind, B, V, dtype, V + B, stride)
    rng = np.random.default_rng(V)
    u = rng.random(B).astype(np.float32)
    check(paged, x, u)  # the whole distribution
    check(paged, x, u, temp=rng.choice([0.3, 1.0, 1.7], B))
    check(paged, x, u, temp=rng.choice([0.5, 1.0], B), top_k=rng.choice([0, 1, 2, 50, 1500, V], B))
    check(paged, x, u, temp=rng.choice([0.5, 1.0], B), top_p=rng.choice([0.1, 0.77, 0.93], B))
    check(paged, x, u, temp=rng.choice([0.5, 1.0], B), min_p=rng.choice([0.013, 0.37], B))
    check(paged, x, u, temp=rng.choice([0.0, 0.7, 1.0], B), top_k=rng.choice([0, 40, 3000], B),
          top_p=rng.choice([0.83, 0.97, 1.0], B), min_p=rng.choice([0.0, 0.003], B))


@pytest.mark.gpu
def test_values_at_the_edges(pkg):
    """Ends of the uniform range, infinities, NaN, rows with nothing left, parameters at and beyond their ends."""
    from minicpmo_b200 import paged

    inf, nan = math.inf, math.nan
    rows = [[nan, 1, 2, -inf], [-inf] * 4, [nan] * 4, [inf, 3, inf, nan], [-3e38, -inf, nan, -3e38], [0.0, -0.0, -1, -2],
            [5, 1e-40, -1e-40, 5], [-inf, -inf, -inf, 7]]
    x = torch.tensor(rows, device="cuda")
    B = len(rows)
    for u in (0.0, 0.25, 0.99, 1.0, -1.0, 2.0, nan):
        check(paged, x, [u] * B)
        check(paged, x, [u] * B, top_p=[0.6] * B, temp=[2.0] * B)
    check(paged, x, [0.3] * B, temp=[nan] * B)
    check(paged, x, [0.3] * B, temp=[-1.0] * B)
    check(paged, x, [0.9] * B, top_k=[-5] * B, top_p=[-0.5] * B)
    check(paged, x, [0.9] * B, top_k=[1000] * B, min_p=[2.0] * B)
    check(paged, x, [0.9] * B, min_p=[-1.0] * B, top_p=[1.5] * B)


@pytest.mark.gpu
def test_more_kept_than_one_block_sorts(pkg):
    """Nuclei of tens of thousands of tokens: every cut is narrowed by histograms, down to equal logits."""
    from minicpmo_b200 import paged

    rng = np.random.default_rng(3)
    for dtype in DT:
        for kind in ("normal", "flat", "ties"):
            x = logits_of(kind, 6, 120007, dtype, 17)
            u = rng.random(6).astype(np.float32)
            check(paged, x, u, top_p=[0.9, 0.99, 0.5, 0.995, 0.8, 0.97], temp=[1, 2, 5, 1, 50, 1])
            check(paged, x, u, top_k=[2000, 30000, 1025, 119999, 5000, 64], min_p=[0, 1e-4, 1e-9, 0, 0.01, 0])
            check(paged, x, u, top_k=[0, 90000, 0, 70000, 1024, 2], top_p=[0.9, 0.7, 0.999, 0.6, 0.9, 0.9],
                  min_p=[1e-5, 0, 1e-3, 0, 0, 1e-6])


@pytest.mark.gpu
def test_many_rows_and_the_largest_vocabulary(pkg):
    from minicpmo_b200 import paged

    rng = np.random.default_rng(4)
    x = logits_of("likely", 200, 3001, "bf16", 5)
    check(paged, x, rng.random(200).astype(np.float32), top_p=rng.choice([0.5, 0.9, 1.0], 200))
    x = logits_of("normal", 2, 1 << 19, "f32", 6)
    check(paged, x, [0.21, 0.83], top_p=[0.9, 1.0], top_k=[0, 60])
