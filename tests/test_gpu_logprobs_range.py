"""Token log probabilities and their gradient over the whole range of finite
logits, on the GPU: tokens masked with a large negative number, rows far from
zero, rows of one certain token.

The definition takes a row's maximum m off before it scales, so that it is exact
in 64 bits at any size: d = (x - m) / temperature, log p = d - log sum exp d.

Tolerances, u = 2^-24 (half a step of f32, relative). The temperature, its
reciprocal's product and the result are rounded to f32, u of |log p| (of |lse|)
each; the sum of exponentials is off by less than 80 u (64 terms a lane in two
chains, a tree of 6, exponentials and their arguments).
  logprobs u (80 + 4 |log p|), lse u (80 + 4 |lse|)
  entropy  u (80 (2 + H) + 4 sum p (|d| + d^2)): a term p d is off by what its
           exponential's argument is, 3 u |d|, and by its own roundings
No log probability is above 0 and no entropy below: the largest term is exactly 1,
so the sum is at least 1, and every other step keeps the sign."""
import numpy as np
import pytest
import torch

from test_gpu_logprobs import BF, F32, U, ids_for, make

pytestmark = pytest.mark.gpu

V, ROWS, K = 40000, 3, 20
MASKS = [-1e9, -1e10, -1e20, -1e30]


def exact(logits, temp):
    x = logits.detach().float().cpu().double().numpy()
    m = x.max(1, keepdims=True)
    d = (x - m) / temp
    ls = np.log(np.exp(d).sum(1, keepdims=True))
    logp = d - ls
    p = np.exp(logp)
    H = -(p * np.where(p > 0, logp, 0)).sum(1)
    return dict(d=d, logp=logp, p=p, H=H, lse=(m / temp + ls)[:, 0])


def rows_of(name, value, dtype):
    x = make(ROWS, V, dtype, 41)
    if name == "part":       # whole wavefronts and pieces are masked, parts of others
        x[:, 9000:31000] = value
    elif name == "most":     # five tokens are allowed
        keep = x[:, 7::8000].clone()
        x[:] = value
        x[:, 7::8000] = keep
    elif name == "row":      # a row whose mask leaves nothing, between ordinary ones
        x[1] = value
    elif name == "offset":   # ordinary rows far from zero
        x = (x.float() * 1000 + value).to(dtype)
    return x


CASES = [(n, v) for n in ("part", "most", "row") for v in MASKS] + [("offset", s * v) for v in (1e10, 1e20) for s in (1, -1)]


def check_forward(logits, ids, temp, k):
    from glt_amd import ops
    got = ops.token_logprobs(logits, ids, top_k=k, temperature=temp)
    torch.cuda.synchronize()
    w = exact(logits, temp)
    i = ids.cpu().numpy()
    order = np.argsort(-logits.float().cpu().numpy(), 1, kind="stable")[:, :k]
    assert np.array_equal(got["top_ids"].cpu().numpy(), order)
    tol_h = U * (80 * (2 + w["H"]) + 4 * (w["p"] * (np.abs(w["d"]) + w["d"] ** 2)).sum(1))
    for name, want, tol in [
            ("lse", w["lse"], U * (80 + 4 * np.abs(w["lse"]))), ("entropy", w["H"], tol_h),
            ("logprobs", np.take_along_axis(w["logp"], i, 1), None),
            ("top_logprobs", np.take_along_axis(w["logp"], order, 1), None)]:
        g = got[name].double().cpu().numpy()
        tol = U * (80 + 4 * np.abs(want)) if tol is None else tol
        assert np.isfinite(g).all() and (np.abs(g - want) <= tol).all(), (name, g, want)
    assert bool((got["logprobs"] <= 0).all()) and bool((got["top_logprobs"] <= 0).all())
    assert bool((got["entropy"] >= 0).all())
    return got, w


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("temp", [0.7, 1.0, 1.3])
@pytest.mark.parametrize("name,value", CASES)
def test_statistics_of_large_logits(dev, dtype, temp, name, value):
    check_forward(rows_of(name, value, dtype), ids_for(ROWS, V, 4, 42), temp, K)


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("temp", [0.7, 1.0])
def test_certain_tokens_have_no_positive_log_probability(dev, dtype, temp):
    """One token has all the weight: its logit 14 to 86 temperatures above the
    rest."""
    rows, v = 300, 9000
    x = make(rows, v, dtype, 43, std=0.5).float()
    at = ids_for(rows, v, 1, 44)
    x.scatter_(1, at.long(), temp * torch.linspace(14, 86, rows, device="cuda")[:, None])
    x = x.to(dtype)
    check_forward(x, at, temp, 5)


def check_gradient(logits, ids, temp, ent, place=False):
    """Against the formula. p is off by u (100 + 8 min(|d|, 110)) relative where
    it is formed from d (past 110 it is 0), and by 8 u |lse| more where from z and
    the rounded lse, which rows of |lse| of 4096 and more do not use."""
    from glt_amd import ops
    n = ids.shape[1]
    g = torch.randn((ROWS, n), generator=torch.Generator().manual_seed(1)).cuda()
    ge = torch.randn((ROWS,), generator=torch.Generator().manual_seed(2)).cuda() if ent else None
    r = ops.token_logprobs(logits, ids, temperature=temp)
    w = exact(logits, temp)
    got = ops.token_logprobs_bwd(logits, ids, r["lse"], g, r["entropy"], ge, temp, grad=logits if place else None)
    torch.cuda.synchronize()
    gn = g.cpu().double().numpy()
    gh = ge.cpu().double().numpy()[:, None] if ent else np.zeros((ROWS, 1))
    p, H = w["p"], w["H"][:, None]
    lp_h = np.where(p > 0, w["logp"] + H, 0)
    want = -p * (gn.sum(1, keepdims=True) + gh * lp_h)
    size = p * (np.abs(gn).sum(1, keepdims=True) + np.abs(gh) * (np.abs(lp_h) + H))
    i = ids.cpu().numpy()
    for j in range(n):
        np.add.at(want, (np.arange(ROWS), i[:, j]), gn[:, j])
        np.add.at(size, (np.arange(ROWS), i[:, j]), np.abs(gn[:, j]))
    want, size = want / temp, size / temp
    near = 8 * np.minimum(np.abs(w["d"]), 110) + np.where(np.abs(w["lse"]) < 4096, 8 * np.abs(w["lse"]), 0)[:, None]
    half = 2.0 ** -8 if logits.dtype == BF else 2.0 ** -24
    tol = U * (100 + near) * size + half * np.abs(want) + 2.0 ** -133
    d = np.abs(got.double().cpu().numpy() - want)
    assert np.isfinite(d).all() and (d <= tol).all(), (d.max(), (d / tol).max())
    return got


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("temp", [0.7, 1.0, 1.3])
@pytest.mark.parametrize("name,value", CASES)
def test_gradient_of_large_logits(dev, dtype, temp, name, value):
    ids = ids_for(ROWS, V, 4, 45)
    ids[:, 1] = ids[:, 0]    # the same token twice
    x = rows_of(name, value, dtype)
    got = check_gradient(x, ids, temp, True)
    y = x.clone()
    assert torch.equal(check_gradient(y, ids, temp, True, place=True), got) and torch.equal(y, got)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_gradient_where_lse_passes_the_range(dev, dtype):
    """Rows masked with the type's lowest value, whose scaled lse is -inf in f32:
    every token has its share. A row of -inf has none, and no other row's
    gradient changes."""
    x = rows_of("row", torch.finfo(dtype).min, dtype)
    ids = ids_for(ROWS, V, 2, 46)
    got = check_gradient(x, ids, 0.7, True)
    assert bool(got[1].any())
    from glt_amd import ops
    x[1] = -np.inf
    g = torch.ones((ROWS, 2), device="cuda")
    r = ops.token_logprobs(x, ids, temperature=0.7)
    a = ops.token_logprobs_bwd(x, ids, r["lse"], g, temperature=0.7)
    b = ops.token_logprobs_bwd(x[::2], ids[::2].contiguous(), r["lse"][::2].contiguous(), g[::2].contiguous(), temperature=0.7)
    assert not a[1].any() and torch.equal(a[::2], b)


@pytest.mark.parametrize("v,n", [(1, 1), (37, 3), (4097, 64), (1 << 20, 2)])
def test_gradient_far_from_zero_of_any_width(dev, v, n):
    """One logit to the largest vocabulary, rows of large lse beside one of
    ordinary lse, with padding and foreign ids."""
    from glt_amd import ops
    x = make(3, v, F32, 47)
    x[1] += 30000
    x[2] -= 30000
    ids = ids_for(3, v, n, 48)
    r = ops.token_logprobs(x, ids)
    g = torch.full((3, n), 0.25, device="cuda")
    got = ops.token_logprobs_bwd(x, ids, r["lse"], g)
    for i in range(3):
        w = exact(x[i:i + 1], 1.0)
        want = -w["p"][0] * 0.25 * n
        np.add.at(want, ids[i].cpu().numpy(), 0.25)
        size = w["p"][0] * 0.25 * n
        np.add.at(size, ids[i].cpu().numpy(), 0.25)
        tol = U * (100 + 8 * np.minimum(np.abs(w["d"][0]), 110) + 60) * size + U * np.abs(want) + 2.0 ** -133
        assert (np.abs(got[i].double().cpu().numpy() - want) <= tol).all(), i
    ids[:, 0] = -1
    a = ops.token_logprobs_bwd(x, ids, r["lse"], g)
    assert bool(torch.isfinite(a).all()) and a.any() == (n > 1 and v > 1)
    ids[:, 0] = v
    assert bool(torch.isnan(ops.token_logprobs_bwd(x, ids, r["lse"], g)).all())


def test_entropy_gradient_without_tokens_far_from_zero(dev):
    """No given tokens: the entropy's gradient alone, of rows either side of zero
    and of the lse from which a row is formed again."""
    from glt_amd import ops
    x = make(4, V, F32, 49)
    x += torch.tensor([0.0, 4000.0, 4100.0, -1e6], device="cuda")[:, None]
    r = ops.token_logprobs(x, temperature=1.0)
    ge = torch.tensor([1.0, -2.0, 0.5, 3.0], device="cuda")
    got = ops.token_logprobs_bwd(x, None, r["lse"], None, r["entropy"], ge)
    w = exact(x, 1.0)
    gh, H = ge.cpu().double().numpy()[:, None], w["H"][:, None]
    lp_h = np.where(w["p"] > 0, w["logp"] + H, 0)
    want, size = -w["p"] * gh * lp_h, w["p"] * np.abs(gh) * (np.abs(lp_h) + H)
    assert (np.abs(w["lse"])[:2] < 4096).all() and (np.abs(w["lse"])[2:] > 4096).all()
    far = np.where(np.abs(w["lse"]) < 4096, 8 * np.abs(w["lse"]), 0)[:, None]
    tol = U * (100 + 8 * np.minimum(np.abs(w["d"]), 110) + far) * (size + w["p"] * np.abs(gh)) + U * np.abs(want) + 2.0 ** -133
    assert (np.abs(got.double().cpu().numpy() - want) <= tol).all()
