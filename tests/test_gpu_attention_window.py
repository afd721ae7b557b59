"""Attention for training with a sliding window and sinks against the formula in
64 bits, with the tolerances of test_gpu_attention_train.py, and a generation
over the 8-bit cache that sees what training sees."""
import math

import pytest
import torch

import kv8_ref as R
from test_gpu_attention_train import BF, BOUND, F64, HD, check, lse_bound, make, run

pytestmark = pytest.mark.gpu


def visible(n, window, sinks):
    t = torch.arange(n)
    back = t[:, None] - t[None]
    return (back >= 0) & ((back < window) | (t[None] < sinks))


def formula(q, k, v, dout, scale, lens, window, sinks):
    q, k, v, dout = (t.detach().cpu().double() for t in (q, k, v, dout))
    B, T, Hq, _ = q.shape
    rep = Hq // k.shape[2]
    r = dict(out=torch.zeros_like(q), lse=torch.full((B, Hq, T), -math.inf, dtype=F64), dq=torch.zeros_like(q),
             dk=torch.zeros_like(k), dv=torch.zeros_like(v))
    for b in range(B):
        n = lens[b]
        see = visible(n, window, sinks)
        for h in range(Hq if n else 0):
            g = h // rep
            Q, K, V, dO = q[b, :n, h], k[b, :n, g], v[b, :n, g], dout[b, :n, h]
            s = (Q @ K.t() * scale).masked_fill(~see, -math.inf)
            r["lse"][b, h, :n] = torch.logsumexp(s, -1)
            p = torch.softmax(s, -1)
            dp = dO @ V.t()
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            r["out"][b, :n, h] = p @ V
            r["dq"][b, :n, h] = scale * ds @ K
            r["dk"][b, :n, g] += scale * ds.t() @ Q
            r["dv"][b, :n, g] += p.t() @ dO
    return r


CASES = [
    # B, T, Hq, Hkv, window, sinks, lens, fused
    (1, 2, 2, 1, 1, 0, None, False),               # each row sees itself alone
    (1, 130, 2, 2, 1, 0, None, True),
    (1, 200, 4, 2, 1, 1, None, False),             # and the first one
    (2, 65, 2, 1, 2, 0, None, False),
    (1, 300, 2, 1, 31, 0, None, True),             # below, at and past a wavefront's rows
    (1, 300, 4, 4, 32, 3, None, False),
    (1, 300, 6, 2, 33, 33, None, True),
    (1, 400, 2, 1, 64, 0, None, False),            # a tile
    (1, 400, 2, 1, 65, 64, None, False),
    (2, 450, 4, 2, 127, 65, None, True),           # a workgroup's rows
    (1, 515, 2, 2, 128, 128, None, False),
    (1, 515, 3, 1, 129, 129, None, False),         # sinks in two blocks
    (1, 1500, 2, 1, 70, 4, None, True),            # sinks' queries in cuts of eight tiles
    (1, 3300, 4, 2, 200, 4, None, False),
    (1, 2500, 2, 1, 90, 300, None, False),         # of three blocks
    (1, 2300, 1, 1, 1000, 1024, None, False),
    (2, 2900, 4, 2, 500, 200, (2777, 700), False), # cuts of ten
    (5, 300, 4, 2, 50, 2, (300, 0, 1, 64, 201), True),
    (3, 1700, 2, 1, 64, 4, (1300, 1700, 17), False),
    (2, 100, 2, 1, 99, 0, None, False),            # all but one key
]


@pytest.mark.parametrize("B,T,Hq,Hkv,window,sinks,lens,fused", CASES)
def test_forward_and_backward_against_the_formula(dev, B, T, Hq, Hkv, window, sinks, lens, fused):
    q, k, v, dout = make(B, T, Hq, Hkv, 200 + T, fused, 2.0)
    sl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    got = run(q, k, v, dout, seq_lens=sl, window=window, sinks=sinks)
    torch.cuda.synchronize()
    want = formula(q, k, v, dout, HD ** -0.5, lens or [T] * B, window, sinks)
    if window == 1 and sinks == 0:                 # one key a row: no gradient on the scores, exactly
        assert not got.pop("dq").any() and not got.pop("dk").any()
    for name in got:
        check(name, got[name], want[name], lse_bound(q, k, HD ** -0.5, want["lse"]))
    for b, n in enumerate(lens or []):
        for name in got:
            assert name == "lse" or not got[name][b, n:].any(), name


@pytest.mark.parametrize("B,T,Hq,Hkv,window,sinks,fused", [
    (12, 1400, 16, 4, 100, 4, True),      # key blocks that fill the chip: a kv head's query heads in one workgroup
    (12, 1400, 16, 4, 700, 0, False),
    (12, 1400, 16, 4, 701, 0, False),     # in parts again
    (6, 1400, 16, 4, 64, 130, False),     # in two parts
    (24, 700, 6, 3, 90, 1, True),
])
def test_batches_that_fill_the_chip(dev, B, T, Hq, Hkv, window, sinks, fused):
    q, k, v, dout = make(B, T, Hq, Hkv, 31, fused, 2.0)
    lens = [T - (137 * i) % 900 if i % 3 else T for i in range(B)]
    got = run(q, k, v, dout, seq_lens=torch.tensor(lens, dtype=torch.int32, device=dev), window=window, sinks=sinks)
    lens = [max(n, 0) for n in lens]
    for b in (1, B - 1):
        one = [t[b:b + 1] for t in (q, k, v, dout)]
        want = formula(*one, HD ** -0.5, lens[b:b + 1], window, sinks)
        for name in want:
            check(name, got[name][b:b + 1], want[name], lse_bound(one[0], one[1], HD ** -0.5, want["lse"]))


@pytest.mark.parametrize("window", [333, 334, 5000, 2 ** 31 - 1])
@pytest.mark.parametrize("sinks", [0, 7])
def test_a_window_that_hides_nothing(dev, window, sinks):
    q, k, v, dout = make(2, 333, 4, 2, 3)
    a, b = run(q, k, v, dout), run(q, k, v, dout, window=window, sinks=sinks)
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_many_sinks_where_nothing_is_hidden(dev):
    q, k, v, dout = make(1, 200, 4, 2, 3)
    a, b = run(q, k, v, dout), run(q, k, v, dout, window=200, sinks=5000)
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_what_no_row_of_the_tile_sees_takes_no_part(dev):
    """NaN and infinity in keys and values that lie whole tiles before every
    window, behind the sinks' tile, and in the padding."""
    q, k, v, dout = make(1, 700, 2, 1, 4)
    lens = torch.tensor([650], dtype=torch.int32, device=dev)
    last = slice(512, 700)
    res = []
    for fill in (0.0, math.nan, math.inf):
        for t in (k, v):
            t[:, 64:320] = fill
            t[:, 650:] = fill
        q[:, 64:320], dout[:, 64:320] = fill, fill
        res.append(run(q, k, v, dout, seq_lens=lens, window=100, sinks=5))
    for r in res[1:]:
        for name in ("out", "dq"):
            assert torch.equal(r[name][:, last], res[0][name][:, last]), name
        for name in ("dk", "dv"):
            assert torch.equal(r[name][:, last], res[0][name][:, last]), name


def test_repeats_and_batches(dev):
    q, k, v, dout = make(4, 1400, 4, 2, 9)
    lens = torch.tensor((1400, 1, 1250, 64), dtype=torch.int32, device=dev)
    kw = dict(window=100, sinks=4)
    whole, again = run(q, k, v, dout, seq_lens=lens, **kw), run(q, k, v, dout, seq_lens=lens, **kw)
    for name in whole:
        assert torch.equal(whole[name], again[name]), name
    for b in range(4):
        one = run(q[b:b + 1], k[b:b + 1], v[b:b + 1], dout[b:b + 1], seq_lens=lens[b:b + 1], **kw)
        for name in whole:
            assert torch.equal(one[name], whole[name][b:b + 1]), (name, b)


@pytest.mark.parametrize("T,window,sinks,sharpness", [(700, 600, 0, 16), (1500, 300, 4, 8), (1500, 1000, 4, 16)])
def test_peaked_rows(dev, T, window, sinks, sharpness):
    q, k, v, dout = make(1, T, 2, 1, 5)
    scale = sharpness * HD ** -0.5
    got = run(q, k, v, dout, scale=scale, window=window, sinks=sinks)
    want = formula(q, k, v, dout, scale, [T], window, sinks)
    for name in want:
        check(name, got[name], want[name], lse_bound(q, k, scale, want["lse"]))


@pytest.mark.parametrize("B,T,Hq,Hkv,window,sinks,lens", [
    (1, 2, 8, 1, 2, 0, None),
    (1, 7, 6, 2, 3, 0, None),
    (3, 11, 6, 2, 672, 0, None),                   # a window that hides nothing
    (2, 65, 4, 4, 20, 3, (65, 30)),
    (2, 128, 4, 1, 128, 0, None),
    (1, 128, 2, 1, 127, 9, None),
])
def test_short_calls_round_once(dev, B, T, Hq, Hkv, window, sinks, lens):
    """Up to 128 tokens p and ds go in two bf16 parts: the gradients are off by the
    result's half step and what the rest leaves. e, the relative error of p: its
    score's and lse's (a bound each), and the exponential's. dp and D are f32 sums of
    at most 128 products of 16 bits, D's with p's error too; the parts hold 2^-16. The last
    sum has as many terms as rows and heads, and 64 at most of rest and rounding each."""
    q, k, v, dout = make(B, T, Hq, Hkv, 7, False, 2.0)
    sl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    got = run(q, k, v, dout, seq_lens=sl, window=window, sinks=sinks)
    torch.cuda.synchronize()
    scale, rep = HD ** -0.5, Hq // Hkv
    lens = lens or [T] * B
    want = formula(q, k, v, dout, scale, lens, window, sinks)
    e = 2 * lse_bound(q, k, scale, want["lse"]) + 2.0 ** -20
    q, k, v, dout = (t.detach().cpu().double() for t in (q, k, v, dout))
    names = ("dq", "dk", "dv")
    tol, once = ({n: torch.zeros_like(want[n]) for n in names} for _ in range(2))
    for b, n in enumerate(lens):
        for h in range(Hq):
            g = h // rep
            Q, K, V, dO = q[b, :n, h], k[b, :n, g], v[b, :n, g], dout[b, :n, h]
            p = torch.softmax((Q @ K.t() * scale).masked_fill(~visible(n, window, sinks), -math.inf), -1)
            dp = dO @ V.t()
            dp = dp - (p * dp).sum(-1, keepdim=True)
            f32 = 127 * 2.0 ** -24 * (dO.abs() @ V.abs().t())
            D = e * (p * dp.abs()).sum(-1, keepdim=True) + 2 * (p * f32).sum(-1, keepdim=True)
            ds, sums = p * dp, 2.0 ** -16 + 2 * rep * n * 2.0 ** -24
            eds, ep = ds.abs() * (e + sums) + p * (f32 + D), p * (e + sums)
            tol["dq"][b, :n, h] = scale * eds @ K.abs()
            tol["dk"][b, :n, g] += scale * eds.t() @ Q.abs()
            tol["dv"][b, :n, g] += ep.t() @ dO.abs()
            p, ds = p.to(BF).double(), ds.to(BF).double()
            once["dq"][b, :n, h] = scale * ds @ K
            once["dk"][b, :n, g] += scale * ds.t() @ Q
            once["dv"][b, :n, g] += p.t() @ dO
    for name in names:
        tol[name] += (want[name].abs() + tol[name]).frexp().exponent.sub(9).double().exp2()
        assert bool(((got[name].cpu().double() - want[name]).abs() <= tol[name]).all()), name
        # one part does not hold that
        assert T < 7 or not bool(((once[name].to(BF).double() - want[name]).abs() <= tol[name]).all()), name


def test_long_rows_dq_in_two_parts(dev):
    """dq takes ds in two parts at every length: in the 2-norm the result's rounding, 2^-9
    as above, and D's share of out's, which adds in squares: a row's D is off by less than
    half of what ds's own rounding would be, 2^-10 (a quarter of the square)."""
    q, k, v, dout = make(1, 1500, 4, 2, 8, False, 2.0)
    got = run(q, k, v, dout, window=600, sinks=4)
    want = formula(q, k, v, dout, HD ** -0.5, [1500], 600, 4)["dq"]
    assert float((got["dq"].cpu().double() - want).norm()) <= (2.0 ** -9) * 1.25 ** 0.5 * float(want.norm())


def test_gradient_against_differences(dev):
    T, window, sinks = 150, 40, 3
    q, k, v, dout = make(1, T, 4, 2, 11)
    got = run(q, k, v, dout, window=window, sinks=sinks)
    x = dict(q=q.cpu().double(), k=k.cpu().double(), v=v.cpu().double())
    loss = lambda t: float((formula(t["q"], t["k"], t["v"], dout, HD ** -0.5, [T], window, sinks)["out"]
                            * dout.cpu().double()).sum())
    g = torch.Generator()
    g.manual_seed(3)
    for name in ("q", "k", "v"):
        grad = got["d" + name].cpu().double()
        u = torch.randn(x[name].shape, generator=g, dtype=F64)
        u /= u.norm()
        h = 1e-4
        up, down = dict(x), dict(x)
        up[name], down[name] = x[name] + h * u, x[name] - h * u
        slope = (loss(up) - loss(down)) / (2 * h)
        assert abs(slope - float((grad * u).sum())) <= BOUND["d" + name] * float(grad.norm()) + 1e-6, name


def test_captured_in_a_graph(dev):
    q, k, v, dout = make(2, 1300, 8, 2, 13)
    lens = torch.tensor((1300, 90), dtype=torch.int32, device=dev)
    kw = dict(seq_lens=lens, window=64, sinks=4)
    run(q, k, v, dout, **kw)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = run(q, k, v, dout, **kw)
        graphs.append((g, r))
    for rep in range(3):
        for t, x in zip((q, k, v, dout), make(2, 1300, 8, 2, 20 + rep)):
            t.copy_(x)
        eager = run(q, k, v, dout, **kw)
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, r in graphs:
            for name in r:
                assert torch.equal(r[name], eager[name]), (rep, name)


def test_refusals(dev):
    from glt_amd import ops
    q, k, v, dout = make(2, 20, 4, 2, 19)
    out, lse = ops.attention_train(q, k, v, window=3)
    for kw, err in ((dict(window=3, sinks=1025), ops.F.GltError), (dict(window=3, causal=False), ops.F.GltError),
                    (dict(window=0), ValueError), (dict(window=-1), ValueError), (dict(window=2 ** 32 + 5), ValueError),
                    (dict(window=3, sinks=-1), ValueError), (dict(window=3, sinks=2 ** 32), ValueError),
                    (dict(sinks=3), ValueError)):
        with pytest.raises(err):
            ops.attention_train(q, k, v, **kw)
        with pytest.raises(err):
            ops.attention_bwd(q, k, v, out, lse, dout, **kw)


# ------------------------------------------------------- the set together
@pytest.mark.parametrize("window,sinks", [(None, 0), (70, 4)])
def test_generating_sees_what_training_sees(dev, window, sinks):
    """A prompt of 300 tokens shared by 4 answers of up to 40 that are generated token by
    token over the cache, then the same sequences in one training pass on the values that the cache
    holds. Both round p (and its step) and out: twice 2^-8 of out and of the sums of p |v|."""
    from glt_amd import ops
    P, N, B, Hq, Hkv = 300, 40, 4, 8, 2
    g = torch.Generator().manual_seed(1)
    n = lambda *s: torch.randn(*s, generator=g).to(BF).cuda()
    pk, pv, xk, xv, xq = n(1, P, Hkv, HD), n(1, P, Hkv, HD), n(B, N, Hkv, HD), n(B, N, Hkv, HD), n(B, N, Hq, HD)
    steps = [40, 1, 25, 40]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")
    cache = ops.Kv8Cache(12, Hkv)
    table = torch.randperm(12, generator=g).to(torch.int32).cuda()
    prefix, pages = table[None, :5].contiguous(), table[5:9].view(4, 1).contiguous()
    cache.write(pk, pv, prefix, ints([P]))
    outs = torch.zeros_like(xq)
    for t in range(N):
        new = ints([int(t < s) for s in steps])
        lens = ints([min(t + 1, s) for s in steps])
        cache.write(xk[:, t:t + 1], xv[:, t:t + 1], pages, lens, new)
        o, _ = cache.attention(xq[:, t:t + 1], pages, lens, new, window=window, sinks=sinks, prefix=(prefix, ints([P])))
        outs[:, t] = o[:, 0]
    k0, v0 = cache.read(prefix, ints([P]), P)
    k1, v1 = cache.read(pages, ints(steps), N, ints(steps))
    k, v = (torch.cat([a.expand(B, P, Hkv, HD), b], 1).contiguous() for a, b in ((k0, k1), (v0, v1)))
    q = torch.cat([torch.zeros(B, P, Hq, HD, dtype=BF, device="cuda"), xq], 1)
    out, lse = ops.attention_train(q, k, v, seq_lens=ints([P + s for s in steps]), window=window, sinks=sinks)
    whole = ops.attention_train(q, k, v.abs(), seq_lens=ints([P + s for s in steps]), window=window, sinks=sinks)[0]
    # bf16 values of the cache: k is off by 2^-8, a score by 2^-8 of sum |q k|
    for b, s in enumerate(steps):
        a, c, m = (x[b].double() for x in (outs[:, :s], out[:, P:P + s], whole[:, P:P + s]))
        big = (q[b, P:P + s].float().abs().transpose(0, 1) @ k[b].float().abs().repeat_interleave(Hq // Hkv, 1).permute(1, 2, 0))
        off = 2 * 2.0 ** -8 * big.amax(-1).t()[..., None].double() * HD ** -0.5
        assert ((a - c).abs() <= (5 * 2.0 ** -8 + off) * m + 2 * 2.0 ** -8 * c.abs()).all()
    # and the gradients of the answers go back through the same rows
    dout = torch.randn(q.shape, generator=g).to(BF).cuda()
    dout[:, :P] = 0
    dq, dk, dv = ops.attention_bwd(q, k, v, out, lse, dout, seq_lens=ints([P + s for s in steps]), window=window, sinks=sinks)
    assert not dq[:, :P].any() and dk[:, :P].any() and torch.isfinite(dv.float()).all()
    if window:
        assert not dv[1, sinks:P - window].any()  # one answer of one token
