"""Attention for training on the GPU: the forward with log-sum-exp and the
backward, against the formulas in 64 bits on the same inputs.

Tolerances. A rounding to bf16 is off by at most 2^-8 of the value, and in the
2-norm over values whose mantissas are spread by about 2^-8 / sqrt(3) * 0.72 =
1.7e-3, less than 2^-9. Relative to an output's 2-norm:
  out, dv  two such roundings (of p, and of the result): 2 * 2^-9 if they add
       outright, 3 * 2^-9 with half as much again for sums that cancel.
  dq, dk  ds and the result, and D's share of out's rounding: 4 * 2^-9.
  lse  off by no more than the scores are, and roundings of its own. A score is
       an f32 sum of 128 products (exact in f32: 8 x 8 bits): in any order at
       most 127 roundings of half a step of a partial sum, 127 * 2^-24 *
       sum |q k|, times scale. The shift, the logarithm and the last sum round
       values of at most max |lse| + 8: four times 2^-24 of that.
Every element: within 8 times the 2-norm bound of max(|value|, rms)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F64 = torch.bfloat16, torch.float64
HD = 128


def make(B, T, Hq, Hkv, seed, fused=False, qstd=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n = lambda *s, std=1.0: torch.empty(s, device="cuda").normal_(0, std, generator=g).to(BF)
    if fused:
        qkv = n(B, T, Hq + 2 * Hkv, HD)
        q, k, v = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    else:
        q, k, v = n(B, T, Hq, HD, std=qstd), n(B, T, Hkv, HD), n(B, T, Hkv, HD)
    return q, k, v, n(B, T, Hq, HD)


def formula(q, k, v, dout, scale, causal, lens):
    """out, lse, dq, dk, dv in 64 bits, on the CPU, sequence by sequence."""
    q, k, v, dout = (t.detach().cpu().double() for t in (q, k, v, dout))
    B, T, Hq, _ = q.shape
    rep = Hq // k.shape[2]
    out, lse = torch.zeros_like(q), torch.full((B, Hq, T), -math.inf, dtype=F64)
    dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for b in range(B):
        n = lens[b]
        for h in range(Hq if n else 0):
            g = h // rep
            Q, K, V, dO = q[b, :n, h], k[b, :n, g], v[b, :n, g], dout[b, :n, h]
            s = Q @ K.t() * scale
            if causal:
                s = s.masked_fill(torch.ones(n, n, dtype=torch.bool).triu(1), -math.inf)
            lse[b, h, :n] = torch.logsumexp(s, -1)
            p = torch.exp(s - lse[b, h, :n, None])
            out[b, :n, h] = p @ V
            dp = dO @ V.t()
            ds = p * (dp - (p * dp).sum(-1, keepdim=True))
            dq[b, :n, h] = scale * ds @ K
            dk[b, :n, g] += scale * ds.t() @ Q
            dv[b, :n, g] += p.t() @ dO
    return dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)


BOUND = {"out": 3 * 2.0 ** -9, "dv": 3 * 2.0 ** -9, "dq": 4 * 2.0 ** -9, "dk": 4 * 2.0 ** -9}


def lse_bound(q, k, scale, want):
    rep = q.shape[2] // k.shape[2]
    aq, ak = q.cpu().double().abs(), k.cpu().double().abs().repeat_interleave(rep, 2)
    terms = float((aq.transpose(1, 2) @ ak.permute(0, 2, 3, 1)).max())
    live = torch.isfinite(want)
    return 127 * 2.0 ** -24 * scale * terms + 4 * 2.0 ** -24 * (float(want[live].abs().max()) + 8 if live.any() else 8)


def check(name, got, want, tol=None):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    if name == "lse":
        live = torch.isfinite(want)
        assert torch.equal(live, torch.isfinite(got)) and bool((got[~live] == -math.inf).all())
        assert not live.any() or float((got - want)[live].abs().max()) <= tol
        return
    assert bool(torch.isfinite(got).all()), name
    d, norm = got - want, float(want.norm())
    assert float(d.norm()) <= BOUND[name] * norm, (name, float(d.norm()) / norm)
    rms = norm / math.sqrt(want.numel())
    worst = float((d.abs() / want.abs().clamp(min=rms)).max()) if norm else float(d.abs().max())
    assert worst <= 8 * BOUND[name], (name, worst)


def run(q, k, v, dout, **kw):
    from glt_amd import ops
    out, lse = ops.attention_train(q, k, v, **kw)
    dq, dk, dv = ops.attention_bwd(q, k, v, out, lse, dout, **kw)
    return dict(out=out, lse=lse, dq=dq, dk=dk, dv=dv)


CASES = [
    # B, T, Hq, Hkv, causal, lens, fused
    (1, 1, 4, 1, True, None, False),              # a single token: dq = dk = 0
    (3, 2, 2, 2, False, None, True),
    (1, 31, 2, 1, True, None, False),             # below, at and past a wavefront's 32 rows
    (1, 32, 2, 2, False, None, False),
    (1, 33, 6, 2, True, None, True),
    (2, 64, 4, 4, True, None, False),             # a tile
    (2, 65, 8, 1, False, None, True),
    (2, 127, 2, 1, False, None, False),           # a workgroup's 128 rows
    (1, 128, 4, 1, True, None, False),
    (1, 129, 3, 3, True, None, True),
    (1, 255, 2, 1, True, None, False),
    (1, 256, 4, 2, True, None, True),
    (1, 257, 3, 1, False, None, False),
    (2, 513, 4, 2, True, None, False),            # either side of the rows that take D from p
    (1, 700, 2, 1, False, None, True),
    (5, 130, 4, 2, True, (130, 0, 1, 64, 65), True),
    (4, 300, 2, 2, False, (0, 300, 33, 256), False),
    (3, 600, 8, 2, True, (599, 600, 17), False),
    (1, 5003, 2, 1, True, None, False),           # a long sequence
]


@pytest.mark.parametrize("B,T,Hq,Hkv,causal,lens,fused", CASES)
def test_forward_and_backward_against_the_formula(dev, B, T, Hq, Hkv, causal, lens, fused):
    q, k, v, dout = make(B, T, Hq, Hkv, 100 + T, fused, 2.0)
    sl = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    got = run(q, k, v, dout, causal=causal, seq_lens=sl)
    torch.cuda.synchronize()
    want = formula(q, k, v, dout, HD ** -0.5, causal, lens or [T] * B)
    if fused:
        assert got["dq"].stride() == q.stride() and got["dk"].data_ptr() - got["dq"].data_ptr() == 2 * Hq * HD
    for name, w in want.items():
        if name in ("dq", "dk") and max(lens or [T]) == 1:
            assert not got[name].any()            # one key: no gradient on the scores, exactly
            continue
        check(name, got[name], w, lse_bound(q, k, HD ** -0.5, want["lse"]))
    for b, n in enumerate(lens or []):            # rows past a sequence's end
        for name in ("out", "dq", "dk", "dv"):
            assert not got[name][b, n:].any(), name


def test_nan_and_inf_past_the_end_take_no_part(dev):
    """A padded batch whose padding holds NaN and inf: every result is bit for
    bit the one with zeros there."""
    B, T, Hq, Hkv = 3, 150, 4, 2
    lens = (150, 70, 0)
    q, k, v, dout = make(B, T, Hq, Hkv, 7)
    sl = torch.tensor(lens, dtype=torch.int32, device=dev)
    res = []
    for fill in (0.0, math.nan, math.inf):
        for t in (q, k, v, dout):
            for b, n in enumerate(lens):
                t[b, n:] = fill
        res.append(run(q, k, v, dout, seq_lens=sl))
    for r in res[1:]:
        for name in r:
            assert torch.equal(r[name], res[0][name]), name


def test_rows_of_a_single_key_have_no_score_gradient(dev):
    """The first row under the causal mask and sequences of one token: exact
    zeros, in dk too; a NaN of theirs is passed on."""
    q, k, v, dout = make(3, 90, 4, 2, 6)
    got = run(q, k, v, dout)
    assert not got["dq"][:, 0].any() and got["dq"][:, 1:].any()
    one = torch.tensor([1, 90, 1], dtype=torch.int32, device=dev)
    for causal in (True, False):
        got = run(q, k, v, dout, seq_lens=one, causal=causal)
        for name in ("dq", "dk"):
            assert not got[name][[0, 2]].any() and got[name][1].any(), (name, causal)
        assert torch.equal(got["dv"][0, 0].float(), dout[0, 0].float().view(2, 2, HD).sum(1).to(BF).float())
    dout[0, 0, 3, 5] = math.nan
    got = run(q, k, v, dout, seq_lens=one)
    for name in ("dq", "dk", "dv"):
        assert bool(torch.isnan(got[name][0, 0].float()).any()) and not bool(torch.isnan(got[name][1:].float()).any())


def test_lengths_outside_the_batch_are_clamped(dev):
    q, k, v, dout = make(3, 90, 2, 1, 8)
    a = run(q, k, v, dout, seq_lens=torch.tensor((-5, 90, 40), dtype=torch.int32, device=dev))
    b = run(q, k, v, dout, seq_lens=torch.tensor((0, 2 ** 31 - 1, 40), dtype=torch.int32, device=dev))
    for name in a:
        assert torch.equal(a[name], b[name]), name


def test_a_sequence_does_not_depend_on_the_batch(dev):
    """Each sequence alone gives the bits that it has in the batch, and a run
    again too."""
    q, k, v, dout = make(6, 320, 8, 2, 9)
    lens = torch.tensor((320, 1, 200, 64, 320, 77), dtype=torch.int32, device=dev)
    whole = run(q, k, v, dout, seq_lens=lens)
    again = run(q, k, v, dout, seq_lens=lens)
    for name in whole:
        assert torch.equal(whole[name], again[name]), name
    for b in range(6):
        one = run(q[b:b + 1], k[b:b + 1], v[b:b + 1], dout[b:b + 1], seq_lens=lens[b:b + 1])
        for name in whole:
            assert torch.equal(one[name], whole[name][b:b + 1]), (name, b)


def test_forward_against_the_inference_forward(dev):
    """The same output as glt_attention_fwd up to roundings of p and out."""
    from glt_amd import ops
    q, k, v, _ = make(2, 500, 8, 2, 10)
    out, _ = ops.attention_train(q, k, v)
    ref = ops.attention(q, k, v).double()
    assert float((out.double() - ref).norm() / ref.norm()) < 3 * 2.0 ** -9


def test_gradient_against_differences(dev):
    """Directional differences of the 64-bit loss sum(out * dout) along random
    directions in q, k and v against the kernels' gradients: the gradient's
    tolerance times its norm, as the directions have unit norm per element,
    and the curvature of a step of 1e-4."""
    T, Hq, Hkv = 50, 4, 2
    q, k, v, dout = make(1, T, Hq, Hkv, 11)
    got = run(q, k, v, dout)
    x = dict(q=q.cpu().double(), k=k.cpu().double(), v=v.cpu().double())
    loss = lambda **t: float((formula(t["q"], t["k"], t["v"], dout, HD ** -0.5, True, [T])["out"]
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
        slope = (loss(**up) - loss(**down)) / (2 * h)
        # an error of 2-norm e projects on a unit direction to at most e
        assert abs(slope - float((grad * u).sum())) <= BOUND["d" + name] * float(grad.norm()) + 1e-6, name


def test_scale_and_peaked_rows(dev):
    """A scale that makes most rows one key: p is 0 or 1 nearly everywhere, and
    dp - D cancels. Held to the bounds of the other cases (the scores' f32
    roundings move p by some 2^-17 relative, far below the others)."""
    q, k, v, dout = make(1, 200, 2, 1, 12)
    got = run(q, k, v, dout, scale=1.5)
    want = formula(q, k, v, dout, 1.5, True, [200])
    for name in want:
        check(name, got[name], want[name], lse_bound(q, k, 1.5, want["lse"]))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("T,sharpness", [(700, 4), (700, 16), (1500, 8), (1500, 16)])
def test_peaked_rows_of_many_keys(dev, T, sharpness, causal):
    """Rows of more than 512 keys of which one has nearly all the weight: dp - D
    cancels, and out's rounding in D would show (twice the bounds' elements
    without the second walk of such rows)."""
    q, k, v, dout = make(1, T, 2, 1, 5)
    scale = sharpness * HD ** -0.5
    got = run(q, k, v, dout, scale=scale, causal=causal)
    want = formula(q, k, v, dout, scale, causal, [T])
    for name in want:
        check(name, got[name], want[name], lse_bound(q, k, scale, want["lse"]))


def test_captured_in_a_graph_with_two_workspaces(dev):
    """Forward and backward captured twice, each with a workspace of its own,
    replayed several times with eager work between on new inputs in the
    captured buffers: every replay against the eager call."""
    from glt_amd import ops
    q, k, v, dout = make(2, 200, 8, 2, 13)
    lens = torch.tensor((200, 90), dtype=torch.int32, device=dev)
    run(q, k, v, dout, seq_lens=lens)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            r = run(q, k, v, dout, seq_lens=lens)
        graphs.append((g, r))
    for rep in range(3):
        print("replay", rep, flush=True)
        for t, x in zip((q, k, v, dout), make(2, 200, 8, 2, 20 + rep)):
            t.copy_(x)
        eager = run(q, k, v, dout, seq_lens=lens)
        for g, r in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, r in graphs:
            for name in r:
                assert torch.equal(r[name], eager[name]), (rep, name)


def test_on_another_stream_and_overlapping_calls(dev):
    """Two calls at once on two streams, each with its own workspace, give the
    results of the calls alone."""
    a, b = make(2, 400, 8, 2, 14), make(1, 333, 4, 4, 15)
    ra, rb = run(*a), run(*b)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(sa):
            xa = run(*a)
        with torch.cuda.stream(sb):
            xb = run(*b)
    torch.cuda.synchronize()
    for r, x in ((ra, xa), (rb, xb)):
        for name in r:
            assert torch.equal(r[name], x[name]), name


def test_rows_outside_the_tensors_are_left(dev):
    """A fused gradient buffer with a margin of columns: what is not dq, dk or
    dv keeps its values."""
    from glt_amd import ops
    B, T, Hq, Hkv, pad = 2, 70, 4, 2, 3
    heads = Hq + 2 * Hkv + pad
    buf = torch.full((B, T, heads, HD), 7.0, dtype=BF, device=dev)
    grad = torch.full((B, T, heads, HD), 7.0, dtype=BF, device=dev)
    cut = lambda t: (t[:, :, :Hq], t[:, :, Hq:Hq + Hkv], t[:, :, Hq + Hkv:Hq + 2 * Hkv])
    q, k, v, dout = make(B, T, Hq, Hkv, 16)
    for t, x in zip(cut(buf), (q, k, v)):
        t.copy_(x)
    out, lse = ops.attention_train(*cut(buf))
    r = ops.attention_bwd(*cut(buf), out, lse, dout, grads=cut(grad))
    want = run(q, k, v, dout)
    for t, n in zip(r, ("dq", "dk", "dv")):
        assert torch.equal(t, want[n]), n
    assert bool((grad[:, :, Hq + 2 * Hkv:] == 7.0).all())


def test_one_tensor_as_keys_and_values(dev):
    """q, k and v the same tensor: gradients are three, not one."""
    x = make(1, 60, 2, 2, 17)[0]
    dout = make(1, 60, 2, 2, 18)[0]
    got = run(x, x, x, dout)
    want = formula(x, x, x, dout, HD ** -0.5, True, [60])
    assert len({got[n].data_ptr() for n in ("dq", "dk", "dv")}) == 3
    for name in want:
        check(name, got[name], want[name], lse_bound(x, x, HD ** -0.5, want["lse"]))


def test_python_refusals(dev):
    from glt_amd import ops
    q, k, v, dout = make(2, 20, 4, 2, 19)
    out, lse = ops.attention_train(q, k, v)
    bad = [
        lambda: ops.attention_train(q.float(), k, v),
        lambda: ops.attention_train(q, k[:, :10], v[:, :10]),
        lambda: ops.attention_train(q.transpose(1, 2), k, v),
        lambda: ops.attention_train(q, k, v[:, :, :1]),
        lambda: ops.attention_train(q, k, v, seq_lens=torch.tensor((20, 20), device=dev)),
        lambda: ops.attention_train(q, k, v, seq_lens=torch.tensor((20, 20), dtype=torch.int32)),
        lambda: ops.attention_train(q.cpu(), k, v),
        lambda: ops.attention_bwd(q, k, v, out, lse.double(), dout),
        lambda: ops.attention_bwd(q, k, v, out, lse[:, :, :10], dout),
        lambda: ops.attention_bwd(q, k, v, out, lse, dout[:, :, :2]),
        lambda: ops.attention_bwd(q, k, v, out, lse, dout, grads=(k, q, v)),
        lambda: ops.attention_bwd(q, k, v, out, lse, dout, workspace=torch.empty(16, dtype=torch.uint8, device=dev)),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    from glt_amd import _ffi as F
    with pytest.raises(F.GltError):
        ops.attention_train(q, k, v, scale=0.0)


def test_offsets_past_32_bits(dev):
    """Sequences of nearly 2 GiB of strided rows each, 6 GB in all: the same
    bits as from dense tensors."""
    B, T, ld = 3, 20000, 49152
    q, k, v, dout = make(B, T, 1, 1, 9)
    big = torch.empty((B, T, ld // HD, HD), dtype=BF, device=dev)
    Q, K, V, O = (big[:, :, i:i + 1] for i in (0, 100, 382, 383))
    Q.copy_(q)
    K.copy_(k)
    V.copy_(v)
    lens = torch.tensor([17, 300, T], dtype=torch.int32, device=dev)
    want, got = run(q, k, v, dout, seq_lens=lens), run(Q, K, V, dout, seq_lens=lens)
    for name, w in want.items():
        assert torch.equal(got[name], w), name
    assert got["dq"].stride() == Q.stride()
    # out and dout at the same stride, through the entry points
    from glt_amd import _ffi as F
    import ctypes
    d = F.AttnDesc(B, T, 1, 1, HD, HD ** -0.5, 1, ld, ld, ld, ld, lens.data_ptr())
    lse = torch.empty((B, 1, T), device=dev)
    st = torch.cuda.current_stream().cuda_stream
    F.call("glt_attention_train_fwd", ctypes.byref(d), Q.data_ptr(), K.data_ptr(), V.data_ptr(), O.data_ptr(),
           lse.data_ptr(), st)
    assert torch.equal(O, want["out"]) and torch.equal(lse, want["lse"])
    assert torch.equal(Q, q) and torch.equal(V, v)


def test_gradients_beside_their_inputs_in_one_buffer(dev):
    """q, k, v, dout and dq, dk, dv as columns of one buffer, which do not overlap;
    gradients over their inputs are refused and leave them alone."""
    from glt_amd import _ffi as F
    from glt_amd import ops
    B, T, Hq, Hkv = 2, 70, 4, 2
    heads = Hq + 2 * Hkv
    buf = torch.full((B, T, 2 * heads + Hq, HD), 7.0, dtype=BF, device=dev)
    cut = lambda t: (t[:, :, :Hq], t[:, :, Hq:Hq + Hkv], t[:, :, Hq + Hkv:heads])
    x, grads, dout = cut(buf), cut(buf[:, :, heads:]), buf[:, :, 2 * heads:]
    for t, src in zip(x + (dout,), make(B, T, Hq, Hkv, 23)):
        t.copy_(src)
    dense = dout.contiguous()
    out, lse = ops.attention_train(*x)
    want = run(*(t.contiguous() for t in x), dense)
    for t, n in zip(ops.attention_bwd(*x, out, lse, dense, grads=grads), ("dq", "dk", "dv")):
        assert torch.equal(t, want[n]), n
    keep = buf.clone()
    for bad in (x, (grads[0], x[1], grads[2]), (grads[0], grads[1], grads[1])):
        with pytest.raises(F.GltError, match="overlap"):
            ops.attention_bwd(*x, out, lse, dense, grads=bad)
    assert torch.equal(buf, keep)


def test_output_over_the_queries(dev):
    """out may be q itself: the same bits as apart from it."""
    import ctypes

    from glt_amd import _ffi as F
    q, k, v, dout = make(3, 300, 4, 2, 24)
    lens = torch.tensor((300, 130, 1), dtype=torch.int32, device=dev)
    want = run(q, k, v, dout, seq_lens=lens)
    d = F.AttnDesc(3, 300, 4, 2, HD, HD ** -0.5, 1, 4 * HD, 2 * HD, 2 * HD, 4 * HD, lens.data_ptr())
    lse = torch.empty((3, 4, 300), device=dev)
    F.call("glt_attention_train_fwd", ctypes.byref(d), q.data_ptr(), k.data_ptr(), v.data_ptr(), q.data_ptr(),
           lse.data_ptr(), torch.cuda.current_stream().cuda_stream)
    assert torch.equal(q, want["out"]) and torch.equal(lse, want["lse"])
