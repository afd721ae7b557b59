"""8-bit checkpoints on the GPU: codes and restored values exactly as defined
(every operation is exact but the rounding to the nearest step), the MLP's
activations from them, and the MLP backward that reads them."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def definition(x):
    """Restored values of x [rows, cols] in 64 bits: block by block the smallest
    power of two step with rint(max / step) <= 127 (2^-133 at least, as f32's
    exponents end; 2^121 at most)."""
    a = x.detach().float().cpu().double().numpy()
    rows, cols = a.shape
    out = np.zeros_like(a)
    for b in range(0, cols, 32):
        t = a[:, b:b + 32]
        top = np.abs(t).max(1, keepdims=True)
        ok = np.isfinite(top)
        e = np.frexp(np.where(ok & (top > 0), top, 2.0 ** -140))[1].astype(np.float64)  # top = f 2^e, f in [1/2, 1)
        step = 2.0 ** np.clip(e - 7, -133, 121)
        with np.errstate(invalid="ignore"):
            step = np.where((np.rint(top / step) > 127) & (step < 2.0 ** 121), 2 * step, step)
            v = np.clip(np.rint(t / step), -127, 127) * step
        out[:, b:b + 32] = np.where(ok, v, np.nan)
    return out


def same(got, want):
    g = got.detach().float().cpu().double().numpy()
    assert np.array_equal(np.isnan(g), np.isnan(want))
    assert np.array_equal(g[~np.isnan(g)], want[~np.isnan(want)])


def make(rows, cols, dtype, seed, ld=None):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.empty((rows, ld or cols), device="cuda").normal_(0, 1, generator=g)
    x *= torch.exp2(torch.empty((rows, ld or cols), device="cuda").normal_(0, 3, generator=g))
    return x.to(dtype)[:, :cols]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("rows,cols,ld", [
    (1, 1, None), (1, 15, None), (3, 16, None), (2, 17, 19), (5, 31, None), (4, 32, 40), (7, 33, None), (3, 96, 97),
    (511, 1409, None), (64, 4096, None), (1000, 40, 41),
])
def test_saved_and_restored_as_defined(dev, dtype, rows, cols, ld):
    from glt_amd import ops
    x = make(rows, cols, dtype, rows * cols, ld)
    c = ops.ckpt8_save(x)
    want = definition(x)
    same(c.load(), want)
    same(c.load(BF), want)       # exact in both types
    same(c.load(F32), want)
    again = ops.ckpt8_save(c.load(F32))
    assert torch.equal(again.load(F32), c.load(F32))


def test_error_is_at_most_half_a_step(dev):
    """The step is the smallest power of two for which the largest magnitude
    rounds to at most 127 steps; half that step would give more than 127, so the
    largest is at least 127.5 half steps: half a step is at most 1 / 127.5 of
    it."""
    from glt_amd import ops
    x = make(300, 4096, F32, 2)
    d = (ops.ckpt8_save(x).load(F32) - x).abs().view(300, 128, 32)
    top = x.abs().view(300, 128, 32).amax(2, keepdim=True)
    assert bool((127.5 * d.double() <= top.double()).all())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_borders(dev, dtype):
    """127.5 steps and either side of it, ties, the ends of the range, zeros,
    subnormal values, NaN and infinities: one block each, beside blocks that
    they must not touch."""
    from glt_amd import ops
    tops = [0.0, -0.0, 1.0, 127.0, 127.5, 126.5, 255.0, 254.0, 63.75, 2.0 ** -126, 2.0 ** -133, 3 * 2.0 ** -133,
            torch.finfo(dtype).max, -torch.finfo(dtype).max, 2.0 ** 127, math.nan, math.inf, -math.inf]
    if dtype == F32:
        tops += [float(np.nextafter(np.float32(127.5), np.float32(0))), 2.0 ** -149, 127.49, 1.9999999]
    x = torch.zeros((2 * len(tops), 64), dtype=dtype)
    fill = torch.tensor([0.5, -0.25, 1.5, 2.5, -3.5, 0.0, 60.5, -61.5, 2.0 ** -133, 0.49], dtype=F32)
    for i, t in enumerate(tops):
        x[2 * i, :10] = fill.to(dtype)
        x[2 * i, 11] = t                      # the largest of its block, or not
        x[2 * i + 1, 40] = t                  # alone in its block
        x[2 * i + 1, 3] = 1.0
    x = x.cuda()
    got = ops.ckpt8_save(x).load()
    torch.cuda.synchronize()
    same(got, definition(x))


def test_what_lies_outside_is_left(dev):
    from glt_amd import ops
    x = make(9, 50, BF, 3)
    buf = torch.full((9, 70), 5.0, dtype=BF, device=dev)
    c = ops.ckpt8_save(x)
    c.load(out=buf[:, 11:61])
    same(buf[:, 11:61], definition(x))
    assert bool((buf[:, :11] == 5).all()) and bool((buf[:, 61:] == 5).all())
    size = c.buf.numel()
    big = torch.full((size + 512,), 0xAB, dtype=torch.uint8, device=dev)
    ops.ckpt8_save(x, big[:size])
    assert torch.equal(ops.Ckpt8(big[:size], 9, 50, BF).load(), c.load()) and bool((big[size:] == 0xAB).all())


@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 40), (77, 1100), (130, 704)])
def test_swiglu_from_checkpoints(dev, rows, cols):
    """gate and up exactly; inter within its rounding (2^-8) and the hardware's
    exponential and reciprocal (an ulp of f32 each, times |g|)."""
    from glt_amd import ops
    g, u = make(rows, cols, BF, 4), make(rows, cols, BF, 5)
    g = (g / 8).clamp(-30, 30)
    gate, up, inter = ops.ckpt8_swiglu(ops.ckpt8_save(g), ops.ckpt8_save(u))
    wg, wu = definition(g), definition(u)
    same(gate, wg)
    same(up, wu)
    want = wg / (1 + np.exp(-wg)) * wu
    d = np.abs(inter.double().cpu().numpy() - want)
    assert (d <= np.abs(want) * (2.0 ** -8 + 64 * 2.0 ** -23) + 2.0 ** -133).all()


def _layer(D, I, N, slices, seed):
    from glt_amd import ops
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    n = lambda *s, std=0.02, dt=BF: torch.empty(s, device="cuda").normal_(0, std, generator=g).to(dt)
    base = ops.BaseMLP(n(I, D), n(I, D), n(D, I))
    sl = [ops.GraftSlice(i0, s, h0, h, *[n(s, h, dt=F32) if p in keep else None for p in range(3)]).pack()
          for i0, s, h0, h, keep in slices]
    return base, sl, n


@pytest.mark.parametrize("M,D,I,N,slices", [
    (70, 128, 192, 256, [(192, 64, 0, 128, (0, 1, 2))]),                              # MFMA path, ragged tokens
    (64, 128, 256, 256, [(64, 64, 0, 128, (0, 1, 2)), (128, 64, 64, 64, (2,))]),      # in place, a down slice alone
    (33, 128, 192, 192, [(0, 64, 0, 128, (0, 1))]),                                   # no down graft: inter is not needed
    (19, 100, 60, 75, [(60, 15, 10, 50, (0, 1, 2))]),                                 # odd sizes: the strided path
])
def test_mlp_backward_from_checkpoints(dev, M, D, I, N, slices):
    """The backward from checkpoints is, bit for bit, the backward from the
    activations that they restore to."""
    from glt_amd import ops
    base, sl, n = _layer(D, I, N, slices, 7)
    x, dy = n(M, D, std=1.0), n(M, D, std=1.0, dt=F32)
    _, g, u, _ = ops.mlp_forward(base, sl, x, N)
    g8, u8 = ops.ckpt8_save(g), ops.ckpt8_save(u)
    gr, ur, ir = ops.ckpt8_swiglu(g8, u8)
    want_dx, want = ops.mlp_backward(base, sl, x, dy, N, gr, ur, ir)
    dx, grads = ops.mlp_backward(base, sl, x, dy, N, g8, u8)
    torch.cuda.synchronize()
    assert torch.equal(dx, want_dx) and float(dx.norm()) > 0
    for a, b in zip(grads, want):
        for s, t in zip(a, b):
            assert (s is None) == (t is None)
            assert s is None or (torch.equal(s, t) and float(s.norm()) > 0)


def test_mlp_rmsnorm_backward_from_checkpoints(dev):
    from glt_amd import ops
    M, D, I = 96, 128, 192
    base, sl, n = _layer(D, I, I + 64, [(I, 64, 0, D, (0, 1, 2))], 8)
    xr, w, dy = n(M, D, std=1.0), n(D, std=1.0), n(M, D, std=1.0, dt=F32)
    x, var = ops.rms_norm(xr, w, 1e-5)
    _, g, u, _ = ops.mlp_forward(base, sl, x, I + 64)
    g8, u8 = ops.ckpt8_save(g), ops.ckpt8_save(u)
    gr, ur, ir = ops.ckpt8_swiglu(g8, u8)
    a = ops.mlp_backward(base, sl, x, dy, I + 64, gr, ur, ir, norm=(xr, w, var, 1e-5))
    b = ops.mlp_backward(base, sl, x, dy, I + 64, g8, u8, norm=(xr, w, var, 1e-5))
    torch.cuda.synchronize()
    assert torch.equal(a[0], b[0]) and torch.equal(a[2], b[2])
    for s, t in zip(a[1][0], b[1][0]):
        assert torch.equal(s, t)


def test_captured_and_on_streams(dev):
    from glt_amd import ops
    x, y = make(100, 500, BF, 9), make(100, 500, BF, 10)

    def step():
        return ops.ckpt8_swiglu(ops.ckpt8_save(x), ops.ckpt8_save(y)) + (ops.ckpt8_save(x).load(),)

    step()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r = step()
    for rep in range(3):
        print("replay", rep, flush=True)
        x.copy_(make(100, 500, BF, 20 + rep))
        eager = step()
        g.replay()
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            other = step()
        again = step()
        torch.cuda.synchronize()
        for t in (r, other, again):
            for a, b in zip(t, eager):
                assert torch.equal(a, b), rep


def test_python_refusals(dev):
    from glt_amd import ops
    x = make(4, 64, BF, 11)
    c = ops.ckpt8_save(x)
    base, sl, n = _layer(64, 64, 64, [], 12)
    bad = [
        lambda: ops.ckpt8_save(x[0]),
        lambda: ops.ckpt8_save(x.cpu()),
        lambda: ops.ckpt8_save(x.t()),
        lambda: ops.ckpt8_save(x, torch.empty(10, dtype=torch.uint8, device=dev)),
        lambda: c.load(out=torch.empty((4, 63), dtype=BF, device=dev)),
        lambda: c.load(F32, out=torch.empty((4, 64), dtype=BF, device=dev)),
        lambda: ops.ckpt8_swiglu(c, ops.ckpt8_save(x[:2])),
        lambda: ops.mlp_backward(base, sl, x, x, 64, c, x),
        lambda: ops.mlp_backward(base, sl, x[:2], x[:2], 64, c, c),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was taken")
    with pytest.raises(TypeError):
        ops.ckpt8_save(x.half())


def test_offsets_past_32_bits(dev):
    """4.5 * 10^9 values, 9 GB: the last rows as on their own, and what lies
    before them."""
    from glt_amd import ops
    rows, cols = 275000, 16384
    x = torch.full((rows, cols), 0.75, dtype=BF, device=dev)
    tail = make(5, cols, BF, 77)
    x[-5:] = tail
    y = ops.ckpt8_save(x).load()
    assert torch.equal(y[-5:], ops.ckpt8_save(tail).load())
    assert torch.equal(y[:-5], x[:-5])          # 0.75 is 96 steps of 2^-7
    gate, up, inter = ops.ckpt8_swiglu(ops.ckpt8_save(x), ops.ckpt8_save(x))
    w = ops.ckpt8_swiglu(ops.ckpt8_save(tail), ops.ckpt8_save(tail))
    for a, b in zip((gate, up, inter), w):
        assert torch.equal(a[-5:], b)
