"""Token log probabilities, entropy, top alternatives and their gradient on
the GPU, against the definition in 64 bits.

Tolerances, u = 2^-24 (half a step of f32, relative). The sum of exponentials
of a wavefront: 64 terms a lane in two chains and a tree of 6, each addition u,
the exponential 2 u, its argument's rounding |a| 2^a u below u: s is off by
less than 80 u relative, so lse by 80 u; the scale's rounding moves z by u |z|,
results in f32 round by u of themselves. lse, logprobs: u (80 + 4 max |z|).
Entropy = lse - E[z]: its second sum has the same relative error of a size of
at most H + max shift: u (80 (2 + H) + 4 max |z|).
Gradient: p is off by u (84 + 4 max |z|) relative (lse's error, the difference
and its product with log2 e, the exponential), what multiplies it by three
roundings; and the result's own rounding to its type."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32
U = 2.0 ** -24


def make(rows, V, dtype, seed, ld=None, std=3.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.empty((rows, ld or V), device="cuda").normal_(0, std, generator=g)
    return x.to(dtype)[:, :V]


def ids_for(rows, V, n, seed):
    return torch.from_numpy(np.random.RandomState(seed).randint(0, V, (rows, n)).astype(np.int32)).cuda()


def definition(logits, ids, k, temp):
    """lse, logprobs, entropy in 64 bits; ids of the k largest, lower index first."""
    x = logits.detach().float().cpu().double().numpy()
    z = x / temp
    m = z.max(1, keepdims=True)
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.where(z == -np.inf, 0.0, np.exp(z - np.where(np.isfinite(m), m, 0)))
        s = e.sum(1, keepdims=True)
        lse = np.where(s > 0, np.where(np.isfinite(m), m, 0) + np.log(s), -np.inf)[:, 0]
        logp = np.where(z == -np.inf, -np.inf, z - lse[:, None])
        p = np.where(s > 0, e / np.where(s > 0, s, 1), 0)
        H = -np.where(p > 0, p * logp, 0).sum(1)
    i = ids.cpu().numpy()
    lp = np.take_along_axis(logp, np.clip(i, 0, x.shape[1] - 1), 1)
    lp = np.where(i < 0, 0.0, np.where(i >= x.shape[1], np.nan, lp))
    order = np.argsort(-x, 1, kind="stable")[:, :k]
    return dict(lse=lse, logprobs=lp, entropy=H, top_ids=order, top_logprobs=np.take_along_axis(logp, order, 1)), p, logp


def close(name, got, want, tol):
    got = got.cpu().double().numpy()
    fin = np.isfinite(want)
    assert got.shape == want.shape and np.array_equal(np.isnan(got), np.isnan(want)), name
    assert np.array_equal(got[~fin & ~np.isnan(want)], want[~fin & ~np.isnan(want)]), name
    d = np.abs(got[fin] - want[fin])
    assert d.size == 0 or d.max() <= tol, (name, d.max(), tol)


def check(logits, ids, k, temp=1.0, what=""):
    from glt_amd import ops
    got = ops.token_logprobs(logits, ids, top_k=k, temperature=temp)
    torch.cuda.synchronize()
    want, p, logp = definition(logits, ids, k, temp)
    z = logits.float().cpu().numpy() / temp
    zmax = float(np.abs(z[np.isfinite(z)]).max()) if np.isfinite(z).any() else 0.0
    tol = U * (80 + 4 * zmax)
    close(what + " lse", got["lse"], want["lse"], tol)
    close(what + " logprobs", got["logprobs"], want["logprobs"], tol)
    close(what + " entropy", got["entropy"], want["entropy"], U * (80 * (2 + float(want["entropy"].max())) + 4 * zmax))
    if k:
        assert np.array_equal(got["top_ids"].cpu().numpy(), want["top_ids"]), what
        close(what + " top", got["top_logprobs"], want["top_logprobs"], tol)
    return got, p, logp


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,V,ld,n,k,temp", [
    (1, 1, None, 1, 1, 1.0),                  # one logit
    (2, 37, None, 3, 20, 0.7),                # fewer logits than threads
    (3, 301, 302, 1, 64, 1.0),                # rows at odd places, k of a short row
    (5, 2048, None, 2, 0, 1.3),
    (2, 8191, None, 1, 5, 1.0),               # pieces: 8192 (f32) and 16384 (bf16) logits
    (3, 8193, 8200, 1, 33, 1.0),
    (2, 16384, None, 64, 1, 1.0),
    (2, 16385, 16387, 1, 20, 2.5),
    (4, 50257, None, 4, 20, 0.7),
    (9, 128256, None, 1, 5, 1.0),
    (1, 300001, None, 2, 64, 1.0),
])
def test_statistics_and_alternatives(dev, dtype, rows, V, ld, n, k, temp):
    check(make(rows, V, dtype, V + k, ld), ids_for(rows, V, n, V), k, temp)


def _special(name, V, k, dtype):
    x = make(3, V, dtype, 5)
    if name == "constant":                    # equal everywhere: the lowest indices
        x[:] = 1.25
    elif name == "masked":                    # three tokens are allowed
        keep = x[:, [7, V // 2, V - 1]].clone()
        x[:] = -math.inf
        x[:, [7, V // 2, V - 1]] = keep
    elif name == "nothing":                   # a row whose mask leaves nothing
        x[1] = -math.inf
    elif name == "lowest":                    # masked with the type's lowest value
        x[0, 5:] = torch.finfo(dtype).min
        x[1] = torch.finfo(dtype).min
    elif name == "zeros":                     # both zeros are one value
        x[:] = -1.0
        x[:, 3::5] = -0.0
        x[:, 10::7] = 0.0
    elif name == "falling":                   # sorted: the largest lie together
        x = torch.sort(x.float(), 1, descending=True)[0].to(dtype)
    elif name == "clustered":                 # more large values than a piece's list holds, on fewer lanes than k
        e = torch.arange(V, device="cuda")
        per = 8 if dtype == BF else 4
        lane = (e // per) % 64
        x = torch.where((lane < k - 1)[None], x + 40, x).to(dtype).contiguous()
    elif name == "ties":                      # a few values, each many times, more above the bound than the list holds
        x = torch.round(x.float() / 2).to(dtype)
        x[:, ::3] = 9.0
    elif name == "large":
        x = (x.float() * 1e37).to(dtype)
    return x


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("V,k", [(500, 20), (40000, 20), (40000, 64), (40000, 1)])
@pytest.mark.parametrize("name", ["constant", "masked", "nothing", "lowest", "zeros", "falling", "clustered", "ties"])
def test_special_rows(dev, dtype, V, k, name):
    check(_special(name, V, k, dtype), ids_for(3, V, 2, 3), k, 1.0, name)


def test_logits_near_the_end_of_the_range(dev):
    """Logits of 1e37: one token has everything; alternatives and the
    certain token's log probability 0."""
    x = _special("large", 3000, 5, F32)
    ids = x.argmax(1, keepdim=True).to(torch.int32)
    from glt_amd import ops
    got = ops.token_logprobs(x, ids, top_k=5)
    want, _, _ = definition(x, ids, 5, 1.0)
    assert np.array_equal(got["top_ids"].cpu().numpy(), want["top_ids"])
    assert not got["logprobs"].any() and not got["entropy"].any()
    assert bool((got["top_logprobs"][:, 1:] < -1e30).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_nan_and_inf_rows(dev, dtype):
    """A NaN or +inf makes its row's statistics NaN, no other row's; the
    alternatives stay valid and distinct ids."""
    from glt_amd import ops
    V = 20000
    x = make(4, V, dtype, 6)
    clean = ops.token_logprobs(x.clone(), ids_for(4, V, 1, 1), top_k=20)
    x[1, 12345] = math.nan
    x[2, 19999] = math.inf
    got = ops.token_logprobs(x, ids_for(4, V, 1, 1), top_k=20)
    torch.cuda.synchronize()
    for name in ("lse", "entropy", "logprobs"):
        assert bool(torch.isnan(got[name][1:3]).all()), name
    for name in got:
        assert torch.equal(got[name][[0, 3]], clean[name][[0, 3]]), name
    for r in (1, 2):
        ids = got["top_ids"][r].cpu().numpy()
        assert len(set(ids)) == 20 and ids.min() >= 0 and ids.max() < V
    assert int(got["top_ids"][2, 0]) == 19999


@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_nan_among_masked_logits(dev, dtype):
    """A NaN counts where all logits near it are -inf or NaN too, wherever it
    stands in its row; a row of NaN alone is no row without tokens."""
    from glt_amd import ops
    V = 50001
    x = torch.full((9, V), -math.inf, dtype=dtype, device="cuda")
    for r, at in enumerate((0, 1, 7777, 16384, 40000, V - 1)):
        x[r, at] = math.nan
    x[6] = math.nan
    x[7] = make(1, V, dtype, 3)[0]
    x[7, 30000:40000] = -math.inf
    x[7, 35000] = math.nan
    x[8] = make(1, V, dtype, 4)[0]
    x[8, 16384:32768] = math.nan
    got = ops.token_logprobs(x, ids_for(9, V, 2, 1), top_k=20)
    for name in ("lse", "entropy", "logprobs"):
        assert bool(torch.isnan(got[name]).all()), name
    for r in range(9):
        ids = got["top_ids"][r].cpu().numpy()
        assert len(set(ids)) == 20 and ids.min() >= 0 and ids.max() < V
    grad = ops.token_logprobs_bwd(x, ids_for(9, V, 2, 1), got["lse"], torch.ones(9, 2, device="cuda"))
    assert bool(torch.isnan(grad.float()).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_the_largest_vocabulary(dev, dtype):
    """2^20 tokens and 64 alternatives: the most that a row's workgroup holds."""
    x = make(2, 1 << 20, dtype, 21)
    check(x, ids_for(2, 1 << 20, 64, 5), 64)


def test_padding_and_foreign_ids(dev):
    from glt_amd import ops
    V = 1000
    x = make(3, V, BF, 7)
    ids = torch.tensor([[-1, 5, -7], [999, 1000, 5], [5, 5, -2 ** 31]], dtype=torch.int32, device="cuda")
    got, p, _ = check(x, ids, 0)
    g = torch.tensor([[3.0, 0.5, 2.0], [1.0, 1.0, 1.0], [0.25, 0.5, 9.0]], device="cuda")
    grad = ops.token_logprobs_bwd(x, ids, got["lse"], g).float().cpu().numpy()
    assert np.isnan(grad[1]).all()
    for r, G, at in ((0, 0.5, 0.5), (2, 0.75, 0.75)):
        want = -G * p[r]
        want[5] += at
        assert np.abs(grad[r] - want).max() <= 2.0 ** -8 * np.abs(want).max() + 1e-6


def test_a_row_does_not_depend_on_its_call(dev):
    """Rows alone, in a batch and at another alignment: the same bits."""
    from glt_amd import ops
    V = 50257
    x = make(9, V, BF, 8, V + 4)
    ids = ids_for(9, V, 2, 9)
    whole = ops.token_logprobs(x, ids, top_k=10)
    dense = ops.token_logprobs(x.contiguous(), ids, top_k=10)
    for name in whole:
        assert torch.equal(whole[name], dense[name]), name
        for r in (0, 4, 8):
            one = ops.token_logprobs(x[r:r + 1], ids[r:r + 1], top_k=10)
            assert torch.equal(one[name], whole[name][r:r + 1]), name


def grad_check(logits, ids, g, ge, temp, got, what=""):
    _, p, logp = definition(logits, ids, 0, temp)
    x = logits.float().cpu().numpy().astype(np.float64)
    logp = np.where(p > 0, logp, 0)
    H = -(p * logp).sum(1, keepdims=True)
    gn = g.cpu().double().numpy()
    G = gn.sum(1, keepdims=True)
    gh = ge.cpu().double().numpy()[:, None] if ge is not None else np.zeros_like(G)
    lpH = np.where(p > 0, logp + H, 0)
    want = -p * (G + gh * lpH)
    size = p * (np.abs(gn).sum(1, keepdims=True) + np.abs(gh) * (np.abs(lpH) + H))
    i = ids.cpu().numpy()
    for j in range(i.shape[1]):
        np.add.at(want, (np.arange(len(i)), i[:, j]), gn[:, j])
        np.add.at(size, (np.arange(len(i)), i[:, j]), np.abs(gn[:, j]))
    want, size = want / temp, size / temp
    zmax = np.abs(x[np.isfinite(x)]).max() / temp
    half = 2.0 ** -8 if logits.dtype == BF else 2.0 ** -24
    tol = U * (100 + 8 * zmax) * size + half * np.abs(want) + 2.0 ** -133  # (and a step of the smallest values)
    d = np.abs(got.float().cpu().numpy() - want)
    assert np.isfinite(d).all() and (d <= tol).all(), (what, d.max(), (d / tol).max())


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,V,ld,n,temp,ent,place", [
    (1, 1, None, 1, 1.0, True, False),
    (2, 37, 41, 3, 0.7, True, False),
    (3, 8193, None, 2, 1.0, False, True),
    (2, 16385, 16387, 64, 1.0, True, True),
    (5, 50257, None, 4, 1.3, False, False),
    (4, 128256, None, 1, 1.0, True, True),
])
def test_gradient_against_the_formula(dev, dtype, rows, V, ld, n, temp, ent, place):
    from glt_amd import ops
    x, ids = make(rows, V, dtype, V + 1, ld), ids_for(rows, V, n, V)
    if n > 1:
        ids[:, 1] = ids[:, 0]                 # the same token twice
    g = torch.randn((rows, n), generator=torch.Generator().manual_seed(1)).cuda()
    ge = torch.randn((rows,), generator=torch.Generator().manual_seed(2)).cuda() if ent else None
    r = ops.token_logprobs(x, ids, temperature=temp)
    keep = x.clone()
    got = ops.token_logprobs_bwd(x, ids, r["lse"], g, r["entropy"], ge, temp, grad=x if place else None)
    torch.cuda.synchronize()
    assert (got.data_ptr() == x.data_ptr()) == place
    grad_check(keep, ids, g, ge, temp, got)


def test_gradient_of_masked_logits_and_rows(dev):
    """-inf logits get 0, a row that allows nothing zeros, a row without
    upstream gradient zeros though it holds NaN."""
    from glt_amd import ops
    V = 20000
    x, ids = make(4, V, BF, 11), ids_for(4, V, 1, 12)
    x[0, 100:] = -math.inf
    ids[0] = 50
    x[1] = -math.inf
    x[2, 77] = math.nan
    g, ge = torch.tensor([[1.0], [1.0], [0.0], [1.0]], device="cuda"), torch.tensor([0.5, 0.5, 0.0, 0.5], device="cuda")
    r = ops.token_logprobs(x, ids)
    got = ops.token_logprobs_bwd(x, ids, r["lse"], g, r["entropy"], ge)
    torch.cuda.synchronize()
    assert not got[0, 100:].any() and bool(got[0, :100].any()) and not got[1].any() and not got[2].any()
    for i in (0, 3):
        grad_check(x[i:i + 1], ids[i:i + 1], g[i:i + 1], ge[i:i + 1], 1.0, got[i:i + 1])


def test_gradient_against_differences(dev):
    """Directional differences of the 64-bit objective against the kernel's
    f32 gradient: its error bound (1e-5 relative) times the norms, and a step
    of 1e-4's curvature."""
    from glt_amd import ops
    V, n = 300, 2
    x, ids = make(2, V, F32, 13, std=1.0), ids_for(2, V, n, 14)
    g, ge = torch.tensor([[1.0, -0.5], [0.3, 2.0]]).cuda(), torch.tensor([0.7, -1.1]).cuda()
    r = ops.token_logprobs(x, ids, temperature=0.8)
    grad = ops.token_logprobs_bwd(x, ids, r["lse"], g, r["entropy"], ge, 0.8).cpu().double()

    def f(y):
        lp = torch.log_softmax(y / 0.8, -1)
        return float((g.cpu().double() * lp.gather(1, ids.cpu().long())).sum()
                     - (ge.cpu().double() * (lp.exp() * lp).sum(1)).sum())

    y = x.cpu().double()
    for seed in range(3):
        u = torch.randn(y.shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)
        u /= u.norm()
        slope = (f(y + 1e-4 * u) - f(y - 1e-4 * u)) / 2e-4
        assert abs(slope - float((grad * u).sum())) <= 1e-5 * float(grad.norm()) + 1e-6


def test_values_outside_the_rows_are_left(dev):
    from glt_amd import ops
    buf = torch.full((4, 107), 3.0, dtype=BF, device="cuda")
    x, ids = make(4, 100, BF, 15), ids_for(4, 100, 1, 16)
    r = ops.token_logprobs(x, ids)
    g = torch.ones((4, 1), device="cuda")
    got = ops.token_logprobs_bwd(x, ids, r["lse"], g, grad=buf[:, 3:103])
    assert torch.equal(got, ops.token_logprobs_bwd(x, ids, r["lse"], g))
    assert bool((buf[:, :3] == 3.0).all()) and bool((buf[:, 103:] == 3.0).all())


def test_captured_and_on_streams(dev):
    """Captured twice and replayed with eager work between, and two calls at
    once on two streams: the eager results."""
    from glt_amd import ops
    V = 33000
    x, ids = make(6, V, BF, 17), ids_for(6, V, 2, 18)
    g = torch.ones((6, 2), device="cuda")

    def step():
        r = ops.token_logprobs(x, ids, top_k=7)
        r["grad"] = ops.token_logprobs_bwd(x, ids, r["lse"], g)
        return r

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            r = step()
        graphs.append((gr, r))
    for rep in range(3):
        print("replay", rep, flush=True)
        x.copy_(make(6, V, BF, 30 + rep))
        eager = step()
        for gr, _ in graphs:
            gr.replay()
        s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(s1):
            a = step()
        with torch.cuda.stream(s2):
            b = step()
        torch.cuda.synchronize()
        for r in [r for _, r in graphs] + [a, b]:
            for name in eager:
                assert torch.equal(r[name], eager[name]), (rep, name)


def test_python_refusals(dev):
    from glt_amd import _ffi as F
    from glt_amd import ops
    x, ids = make(3, 50, BF, 19), ids_for(3, 50, 1, 20)
    r = ops.token_logprobs(x, ids)
    g = torch.ones((3, 1), device="cuda")
    bad = [
        lambda: ops.token_logprobs(x[0], ids),
        lambda: ops.token_logprobs(x.t(), ids),
        lambda: ops.token_logprobs(x[:1].expand(3, 50), ids),
        lambda: ops.token_logprobs(x, ids.long()),
        lambda: ops.token_logprobs(x, ids[:2]),
        lambda: ops.token_logprobs(x, ids.cpu()),
        lambda: ops.token_logprobs(x.cpu(), ids),
        lambda: ops.token_logprobs(x, ids, workspace=torch.empty(8, dtype=torch.uint8, device="cuda")),
        lambda: ops.token_logprobs_bwd(x, ids, r["lse"].double(), g),
        lambda: ops.token_logprobs_bwd(x, ids, r["lse"], g[:2]),
        lambda: ops.token_logprobs_bwd(x, ids, r["lse"], g, grad_entropy=g[:, 0].contiguous()),
        lambda: ops.token_logprobs_bwd(x, ids, r["lse"], g, grad=x.float()),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(TypeError):
        ops.token_logprobs(x.half(), ids)
    for f in (lambda: ops.token_logprobs(x, ids, top_k=51), lambda: ops.token_logprobs(x, ids, temperature=0.0)):
        with pytest.raises(F.GltError):
            f()


def test_offsets_past_32_bits(dev):
    """20000 rows of 128256 logits (5.1 GB): the last rows as on their own, the
    gradient in place."""
    from glt_amd import ops
    rows, V = 20000, 128256
    x = torch.zeros((rows, V), dtype=BF, device=dev)
    tail = make(3, V, BF, 31)
    x[-3:] = tail
    ids, few = torch.full((rows, 1), 5, dtype=torch.int32, device=dev), ids_for(3, V, 1, 2)
    ids[-3:] = few
    got, want = ops.token_logprobs(x, ids, top_k=3), ops.token_logprobs(tail, few, top_k=3)
    for name, w in want.items():
        assert torch.equal(got[name][-3:], w), name
    assert float((got["lse"][:-3] - math.log(V)).abs().max()) <= U * (80 + 4 * math.log(V))
    g = torch.ones((rows, 1), device=dev)
    w = ops.token_logprobs_bwd(tail, few, want["lse"], g[-3:])
    grad = ops.token_logprobs_bwd(x, ids, got["lse"], g, grad=x)
    assert grad.data_ptr() == x.data_ptr() and torch.equal(x[-3:], w)
    assert bool((x[:-3, 5] > 0.99).all()) and bool((x[:-3, 6] < 0).all())


def test_gradient_beside_the_logits_in_one_buffer(dev):
    """Gradients in the columns behind the logits do not overlap them; one that is
    shifted over them is refused and leaves them alone."""
    from glt_amd import _ffi as F
    from glt_amd import ops
    buf = torch.full((4, 207), 3.0, dtype=BF, device="cuda")
    x, ids = buf[:, :100], ids_for(4, 100, 1, 16)
    x.copy_(make(4, 100, BF, 15))
    r = ops.token_logprobs(x, ids)
    g = torch.ones((4, 1), device="cuda")
    want = ops.token_logprobs_bwd(x, ids, r["lse"], g)
    assert torch.equal(ops.token_logprobs_bwd(x, ids, r["lse"], g, grad=buf[:, 101:201]), want)
    keep = buf.clone()
    for at in (1, 99):
        with pytest.raises(F.GltError, match="overlap"):
            ops.token_logprobs_bwd(x, ids, r["lse"], g, grad=buf[:, at:at + 100])
    assert torch.equal(buf, keep)
