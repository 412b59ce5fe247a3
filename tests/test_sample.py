"""The sampler against its definition in 64 bits.

A drawn id must be the definition's, unless the uniform number or a limit lies so near a border that the roundings decide: the kernel's
weights are fp32 exponentials (2^-22 relative, at worst all in one direction) in steps of 2^-40 (2^-23 of the sum over 2^17 tokens at
worst), so a border moves by at most 2^-21 of the row's weight against u times the sum: a draw is only compared where u's distance
from the borders of the chosen token, and the limits' distance from theirs, is above that (the inputs are drawn by
seed; how many rows that leaves out is bounded below)."""
import math
import os

import numpy as np
import pytest
import torch

gpu = pytest.mark.gpu
DEV = "cuda"
NEAR = 2.0 ** -21


@pytest.fixture(scope="module")
def sctx(pkg):
    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    c = pkg.Ctx(0, pdl=os.environ.get("DSUF_TEST_PDL", "0") == "1")
    yield c
    c.close()


def sample64(x, u, temp, top_k, top_p, min_p):
    """(id, log-probability, is near a border) of one row, from the definition."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    best = x.max()
    if best == -np.inf:
        return -1, -np.inf, False
    with np.errstate(invalid="ignore"):
        raw = np.where(x == best, 1.0, np.exp(np.where(x == best, 0.0, x - best)))
    if not temp > 0:
        i = int(np.flatnonzero(x == best)[0])
        return i, -math.log(raw.sum()), False
    with np.errstate(invalid="ignore"):
        w = np.where(x == best, 1.0, np.exp(np.where(x == best, 0.0, (x - best) / temp)))
    by = np.lexsort((np.arange(x.size), -x))
    by = by[x[by] > -np.inf]
    near = False
    if top_k > 0:
        by = by[:top_k]
    if top_p < 1:
        mass = np.concatenate([[0.0], np.cumsum(w[by])])
        target = top_p * mass[-1]
        n = max(1, int((mass[:-1] < target).sum()))
        near |= bool(np.abs(mass[[n - 1, n]] - target).min() < NEAR * mass[-1]) and target > 0
        by = by[:n]
    near |= bool((np.abs(w[by] - min_p) < NEAR * max(min_p, 0)).any()) and min_p < 1
    by = np.sort(by[(w[by] >= min(min_p, 1.0)) | (x[by] == best)])
    mass = np.cumsum(w[by])
    at = int(np.flatnonzero(mass > u * mass[-1])[0])
    border = [mass[at]] + ([mass[at - 1]] if at else [])
    near |= min(abs(b - u * mass[-1]) for b in border) < NEAR * mass[-1]
    i = int(by[at])
    return i, (0.0 if x[i] == best else x[i] - best) - math.log(raw.sum()), near


def check(pkg, ctx, logits, u, temp, top_k, top_p, min_p, most_near=0.25):
    m = logits.shape[0]
    col = lambda v, dt: v.to(DEV) if isinstance(v, torch.Tensor) else torch.full((m,), v, dtype=dt, device=DEV)   # noqa: E731
    args = dict(temperature=col(temp, torch.float32), top_k=col(top_k, torch.int32), top_p=col(top_p, torch.float32), min_p=col(min_p, torch.float32))
    ids, lp = pkg.sample(ctx, logits, u, return_logprobs=True, **args)
    again, _ = pkg.sample(ctx, logits, u, return_logprobs=True, **args)
    torch.cuda.synchronize()
    assert torch.equal(ids, again)
    x, uu = logits.cpu().numpy(), u.cpu().numpy()
    cols = [args[k].cpu().numpy() for k in ("temperature", "top_k", "top_p", "min_p")]
    left_out = 0
    for r in range(m):
        i, p, near = sample64(x[r], float(uu[r]), *(float(c[r]) if j != 1 else int(c[r]) for j, c in enumerate(cols)))
        if near:
            left_out += 1
            continue
        assert int(ids[r]) == i, f"row {r}: {int(ids[r])}, wanted {i}"
        if i >= 0:   # two fp32 roundings of a sum of at most 2^22 terms and a logarithm
            assert abs(float(lp[r]) - p) <= 2 ** -18 + 2 ** -22 * abs(p)
        else:
            assert float(lp[r]) == -math.inf
    assert left_out <= max(1, most_near * m)
    return ids


def inputs(seed, m, n, ld=None, std=2.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.empty(m, ld or n, device=DEV).normal_(0, std, generator=g)
    return x[:, :n], torch.rand(m, generator=g, device=DEV), g


@gpu
@pytest.mark.parametrize("m,n,ld", [(1, 1, 1), (3, 2, 5), (2, 31, 31), (5, 1000, 1003), (1, 129280, 129280), (40, 50021, 50022), (7, 4096, 4096), (300, 777, 777), (600, 64, 64)])
@pytest.mark.parametrize("temp,top_k,top_p,min_p", [(1.0, 0, 1.0, 0.0), (0.7, 40, 1.0, 0.0), (1.0, 0, 0.9, 0.0), (0.9, 50, 0.8, 0.05), (1.5, 1, 0.5, 0.0), (0.0, 5, 0.5, 0.1),
                                                    (1.0, 0, 1.0, 0.2), (1.0, 700, 0.999, 1.5), (0.01, 30, 0.9, 0.0), (100.0, 5000, 0.7, 0.0), (1.0, 3, 0.0, 0.0),
                                                    (1.0, 2 ** 31 - 1, 0.5, 0.0)])
def test_settings(pkg, sctx, m, n, ld, temp, top_k, top_p, min_p):
    x, u, _ = inputs(n + m, m, n, ld)
    check(pkg, sctx, x, u, temp, top_k, top_p, min_p)


@gpu
@pytest.mark.parametrize("m,n", [(64, 129280), (9, 20000)])
def test_rows_of_their_own(pkg, sctx, m, n):
    x, u, g = inputs(5, m, n)
    pick = lambda v, dt: torch.tensor([v[i % len(v)] for i in range(m)], dtype=dt)   # noqa: E731
    check(pkg, sctx, x, u, pick([0.8, 1.0, 0.0, 1.3, 0.5], torch.float32), pick([50, 0, 1, 20, 1000, 30000], torch.int32),
          pick([0.95, 1.0, 0.9, 0.5], torch.float32), pick([0.02, 0.0, 0.1], torch.float32))


@gpu
@pytest.mark.parametrize("n", [5000, 100003])
@pytest.mark.parametrize("levels", [1, 2, 7])
def test_many_equal_logits(pkg, sctx, n, levels):
    """Bins that no split can thin out: the id decides."""
    g = torch.Generator(device=DEV).manual_seed(n)
    x = torch.randint(0, levels, (6, n), generator=g, device=DEV).float() * 0.5
    x[:, 17] = torch.where(x[:, 17] == 0, -0.0, x[:, 17])
    u = torch.tensor([0.0, 0.25, 0.5, 0.9, 0.999, 1 - 2 ** -24], device=DEV)
    for top_k, top_p in ((n // 3, 1.0), (0, 0.4), (n // 3, 0.5), (2000, 0.999), (n, 1.0)):
        # equal weights: the borders lie w / total apart, u and the limits exactly on one at worst, so compare the neighbours as well
        ids = pkg.sample(sctx, x, u, top_k=torch.full((6,), top_k, dtype=torch.int32, device=DEV), top_p=torch.full((6,), top_p, device=DEV))
        for r in range(6):
            xs = x[r].cpu().numpy()
            near = {sample64(xs, min(max(float(u[r]) + d, 0.0), 1 - 2 ** -30), 1.0, top_k, top_p + e, 0.0)[0] for d in (-1e-6, 0, 1e-6) for e in (-1e-6, 0, 1e-6)}
            near |= {i + j for i in near for j in (-1, 1)} if levels == 1 else set()
            assert int(ids[r]) in near


@gpu
def test_clustered_logits_are_split_again(pkg, sctx):
    """Far outliers leave most tokens in one bin of the first histogram."""
    x, u, g = inputs(3, 8, 60000, std=0.001)
    x[:, 7] = -1e30
    x[:, 9] += 0.01
    for top_k, top_p in ((3000, 1.0), (0, 0.3), (3000, 0.6), (50000, 0.9)):
        check(pkg, sctx, x, u, 1.0, top_k, top_p, 0.0, most_near=0.5)
        check(pkg, sctx, x * 1e4, u, 50.0, top_k, top_p, 0.0, most_near=0.5)


@gpu
def test_infinite_and_missing_logits(pkg, sctx):
    x, u, _ = inputs(8, 8, 3000)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 1:] = -math.inf
    x[3, 5], x[3, 2000] = math.inf, math.inf
    x[4, ::2] = math.nan
    x[5, :2990] = -math.inf
    x[6] = torch.finfo(torch.float32).min
    x[7, 100] = torch.finfo(torch.float32).max
    for top_k, top_p, min_p, temp in ((0, 1.0, 0.0, 1.0), (20, 0.9, 0.0, 1.0), (0, 0.5, 0.1, 1.0), (1500, 0.9, 0.0, 2.0), (0, 1.0, 0.0, 0.0)):
        ids = check(pkg, sctx, x, u, temp, top_k, top_p, min_p, most_near=0.5)
        assert int(ids[0]) == -1 and int(ids[1]) == -1 and int(ids[2]) == 0 and int(ids[3]) in (5, 2000)


@gpu
@pytest.mark.parametrize("gap,tied", [(2.0, 1), (9.0, 1), (14.0, 1), (9.0, 3)])
@pytest.mark.parametrize("kw", [{}, dict(top_k=5), dict(top_p=0.5), dict(temperature=0.0)])
def test_log_probability_of_a_near_certain_token(pkg, sctx, gap, tied, kw):
    """log(1 / (1 + s)) keeps s's precision however small s is."""
    x, u, _ = inputs(12, 3, 5000)
    x = x.clone()
    x[:, 100:100 + tied] = x.amax(1, keepdim=True) + gap
    full = lambda v: torch.full((3,), v, dtype=torch.int32 if isinstance(v, int) else torch.float32, device=DEV)
    ids, lp = pkg.sample(sctx, x, u * 0.1, return_logprobs=True, **{k: full(v) for k, v in kw.items()})
    assert ids.tolist() == [100] * 3
    others = torch.cat([x[:, :100], x[:, 101:]], 1).double() - x[:, 100:101].double()
    want = -torch.log1p(others.exp().sum(1))
    # l - top (below 32) and its product with log2(e) are rounded once each, the exponential is good to 2^-22, and a sum of at most 5 terms per thread,
    # 5 shuffles, 16 warps and 2 CTAs rounds 28 times: 2^-20 + 2^-19 ln 2 + 2^-22 + 28 2^-24, and log1p
    assert ((lp.double() - want).abs() <= 2 ** -18 * want.abs()).all()


@gpu
@pytest.mark.parametrize("temp", [1.4e-45, 1e-40, 4e-39, 1.2e-38, 1e-30])
@pytest.mark.parametrize("kw", [{}, dict(top_k=3), dict(top_k=2000), dict(top_p=0.7), dict(min_p=0.5)])
def test_temperatures_next_to_nothing(pkg, sctx, temp, kw):
    """Only the largest logits are left, as likely as each other, down to the smallest temperature that fp32 has."""
    x = torch.randn(4, 5000, generator=torch.Generator(device=DEV).manual_seed(3), device=DEV)
    x[:, 700] = x[:, 4100] = 9.0
    u = torch.tensor([0.0, 0.2, 0.9, 0.999], device=DEV)
    full = lambda v: torch.full((4,), v, dtype=torch.int32 if isinstance(v, int) else torch.float32, device=DEV)
    got = torch.full((4,), -7, dtype=torch.int32, device=DEV)
    pkg.sample(sctx, x, u, temperature=full(temp), ids=got, **{k: full(v) for k, v in kw.items()})
    assert got.tolist() == [700, 700, 4100, 4100]


@gpu
def test_defaults_and_frequencies(pkg, sctx):
    """Without settings the draw follows softmax(logits): one row drawn with a lattice of uniforms meets its expectation to one."""
    g = torch.Generator(device=DEV).manual_seed(1)
    row = torch.randn(50, generator=g, device=DEV)
    m = 4000
    u = (torch.arange(m, device=DEV, dtype=torch.float32) + 0.5) / m
    ids = pkg.sample(sctx, row.expand(m, 50).contiguous(), u)
    count = torch.bincount(ids.long(), minlength=50).double()
    assert ((count - torch.softmax(row.double(), 0) * m).abs() <= 1.0).all()


@gpu
def test_refusals(pkg, sctx):
    E = pkg.DsufError
    x, u = torch.zeros(3, 100, device=DEV), torch.zeros(3, device=DEV)
    f, i = torch.zeros(3, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    pkg.sample(sctx, x, u)
    for logits, uu, kw in [(x.half(), u, {}), (x.cpu(), u, {}), (x, u[:2], {}), (x, u.double(), {}), (x[0], u, {}), (x.t(), u, {}), (x, u, dict(temperature=i)), (x, u, dict(top_k=f)),
                           (x, u, dict(top_p=f[:2])), (x, u, dict(min_p=f.cpu())), (x, u, dict(ids=f)), (x, u, dict(logprobs=i)), (x[:, :0], u, {}), (None, u, {})]:
        with pytest.raises(E):
            pkg.sample(sctx, logits, uu, **kw)
    assert pkg.sample(sctx, x[:0], u[:0]).shape == (0,)


@gpu
def test_head_and_sampler_together(pkg, sctx):
    """The output head's logits, their padding columns included, straight into the sampler; greedy rows agree with the head's records."""
    g = torch.Generator(device=DEV).manual_seed(2)
    w = torch.empty(1024, 256, device=DEV).normal_(0, 0.1, generator=g).bfloat16()
    h = torch.empty(9, 256, device=DEV).normal_(0, 1, generator=g).bfloat16()
    logits, rec = pkg.lm_head(sctx, w, h, temperature=1.0)
    ids = pkg.sample(sctx, logits, torch.zeros(9, device=DEV), temperature=torch.zeros(9, device=DEV))
    best = rec[:, :, 0].argmax(1)
    assert torch.equal(ids, rec[torch.arange(9), best, 11].contiguous().view(torch.int32))
