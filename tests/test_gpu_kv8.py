"""The 8-bit cache of keys and values and attention over it against 64-bit results."""
import pytest
import torch

import kv8_ref as R
from glt_amd import ops

pytestmark = pytest.mark.gpu
BF, I32 = torch.bfloat16, torch.int32
HD, PAGE = R.HD, R.PAGE


def ints(v, dev="cuda"):
    return torch.tensor(v, dtype=I32, device=dev)


def rows(shape, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g) * std
    return (x * torch.exp(torch.randn(shape[-1], generator=g) * 0.5)).to(BF)


def stale(cache):
    """Every byte as some other use might have left it: steps NaN, codes -1."""
    cache.data.fill_(0xFF)
    return cache


# --------------------------------------------------------- write and read
@pytest.mark.parametrize("B,T,Hkv,lens,new", [
    (1, 1, 1, [1], None),
    (3, 1, 8, [64, 65, 128], None),          # the last of a page, the first of the next
    (2, 5, 2, [70, 66], [5, 3]),             # over a page's end
    (2, 64, 2, [64, 128], None),             # whole pages
    (3, 64, 1, [100, 63, 0], [64, 63, 0]),
    (2, 200, 4, [200, 333], [200, 77]),
    (4, 3, 3, [2, 1, 0, 9], None),           # fewer tokens than new ones
    (1, 700, 1, [1000], None),
])
def test_tokens_come_back_as_whole_steps(dev, B, T, Hkv, lens, new):
    k, v = rows((B, T, Hkv, HD), 1), rows((B, T, Hkv, HD), 2, 3.0)
    pages = R.tables(lens, 64, 3)
    cache = stale(ops.Kv8Cache(64, Hkv))
    args = pages.cuda(), ints(lens)
    nl = None if new is None else ints(new)
    cache.write(k.cuda(), v.cuda(), *args, new_lens=nl)
    gk, gv = cache.read(*args, T, new_lens=nl)
    n = [min(T if new is None else new[b], T, lens[b]) for b in range(B)]
    for b in range(B):
        for got, x in ((gk, k), (gv, v)):
            assert torch.equal(got[b, :n[b]].cpu(), R.values(x[b, :n[b]]).to(BF))
            assert not got[b, n[b]:].any()


def test_only_the_tokens_bytes_are_written(dev):
    Hkv, lens, new = 2, [70, 130, 64], [9, 66, 2]
    cache = ops.Kv8Cache(12, Hkv)
    before = torch.randint(0, 256, cache.data.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(0))
    cache.data.copy_(before)
    pages = R.tables(lens, 12, 1)
    cache.write(rows((3, 66, Hkv, HD), 4).cuda(), rows((3, 66, Hkv, HD), 5).cuda(), pages.cuda(), ints(lens), ints(new))
    touched = torch.zeros(12, Hkv, R.HEAD_B, dtype=torch.bool)
    for b in range(3):
        for i in range(lens[b] - new[b], lens[b]):
            touched[pages[b, i // PAGE], :, R.token_bytes(i % PAGE)] = True
    same = cache.data.cpu() == before
    assert same[~touched.flatten()].all()
    assert (~same).sum() > touched.sum() * 0.9  # and those are


def test_rows_of_every_kind(dev):
    """Zeros, ties between two codes, the ends of the exponents, NaN and infinity."""
    x = rows((10, HD), 7)
    x[0] = 0
    x[1] = torch.arange(128).to(BF) - 64.5
    x[1, 0] = 127.0                      # step 1: halves are ties
    x[2] = torch.arange(128).to(BF) * 2.0 ** -133
    x[3] = 3.3895e38
    x[4, 5] = float("nan")
    x[5, 6] = float("inf")
    x[6] *= 2.0 ** -100
    x[7] *= 2.0 ** 120
    x[8, :64] *= 1e-30
    x[9] = -x[1]
    k = x.view(1, 10, 1, HD)
    cache = stale(ops.Kv8Cache(1, 1))
    cache.write(k.cuda(), (-k).cuda(), ints([[0]]), ints([10]))
    gk, gv = cache.read(ints([[0]]), ints([10]), 10)
    for got, y in ((gk, k), (gv, -k)):
        want = R.values(y).to(BF)
        assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want))
        assert torch.equal(got.cpu().nan_to_num(0.0), want.nan_to_num(0.0))


def test_parts_of_a_projection(dev):
    B, T, Hq, Hkv = 2, 77, 6, 2
    qkv = rows((B, T, Hq + 2 * Hkv, HD), 8).cuda()
    k, v = qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    lens, pages = ints([77, 90]), R.tables([77, 90], 8, 2).cuda()
    a, b = ops.Kv8Cache(8, Hkv), ops.Kv8Cache(8, Hkv)
    for c, kk, vv in ((a, k, v), (b, k.contiguous(), v.contiguous())):
        c.data.zero_()
        c.write(kk, vv, pages, lens)
    assert torch.equal(a.data, b.data)
    to = torch.full((B, T, 2 * Hkv + 1, HD), 7.0, dtype=BF, device="cuda")
    a.read(pages, lens, T, out=(to[:, :, :Hkv], to[:, :, Hkv:2 * Hkv]))
    gk, gv = a.read(pages, lens, T)
    assert torch.equal(to[:, :, :Hkv], gk) and torch.equal(to[:, :, Hkv:2 * Hkv], gv) and (to[:, :, 2 * Hkv:] == 7).all()


def test_pages_outside_the_pool(dev):
    """Dropped on writing, NaN on reading; a table row longer than what is held is not looked at."""
    cache = ops.Kv8Cache(4, 1)
    cache.data.zero_()
    k, v = rows((1, 150, 1, HD), 1).cuda(), rows((1, 150, 1, HD), 2).cuda()
    pages, lens = ints([[2, -1, 4, 1 << 30]]), ints([150])
    cache.write(k, v, pages, lens)
    assert not cache.data.view(4, -1)[[0, 1, 3]].any()
    gk, gv = cache.read(pages, lens, 150)
    for got, x in ((gk, k), (gv, v)):
        assert torch.equal(got[0, :64].cpu(), R.values(x[0, :64]).to(BF))
        assert torch.isnan(got[0, 64:]).all()
    q = rows((1, 150, 2, HD), 3).cuda()
    out, lse = cache.attention(q, pages, lens)
    assert torch.isfinite(out[0, :64]).all() and torch.isfinite(lse[..., :64]).all()
    assert torch.isnan(out[0, 64:]).all() and torch.isnan(lse[..., 64:]).all()
    out, _ = cache.attention(q[:, :1], pages, ints([64]))
    assert torch.isfinite(out).all()


# -------------------------------------------------------------- attention
class Setup:
    """A cache with sequences (and prefixes), what it holds, and the call's q."""

    def __init__(self, T, Hq, Hkv, lens, new=None, plens=(), seed=0, n_pages=None, bad=(), q_std=2.0, extra=1):
        B = len(lens)
        self.B, self.T, self.Hq, self.Hkv, self.lens, self.plens = B, T, Hq, Hkv, list(lens), list(plens)
        self.new = [min(T if new is None else new[b], T, lens[b]) for b in range(B)]
        width = max([-(-n // PAGE) for n in list(lens) + list(plens)] + [1]) + extra
        n_pages = n_pages or (B + len(plens)) * width + 3
        table = R.tables(list(lens) + list(plens), n_pages, seed, extra)
        self.cache = stale(ops.Kv8Cache(n_pages, Hkv))
        self.table = table.cuda()
        self.pages = self.table[:B]
        self.prefix = (self.table[B:], ints(self.plens)) if plens else None
        self.k, self.v = [], []
        for i, n in enumerate(self.lens + self.plens):
            k, v = rows((n, Hkv, HD), 100 * seed + 2 * i), rows((n, Hkv, HD), 100 * seed + 2 * i + 1)
            for s, t in bad:
                if s == i:
                    v[t, 0, 3] = float("nan")
            if n:
                self.cache.write(k[None].cuda(), v[None].cuda(), self.table[i:i + 1], ints([n]))
            self.k.append(R.values(k))
            self.v.append(R.values(v))
        self.q = rows((B, T, Hq, HD), 100 * seed + 99, q_std).cuda()
        self.new_t = None if new is None else ints(new)

    def run(self, **kw):
        return self.cache.attention(self.q, self.pages, ints(self.lens), new_lens=self.new_t, prefix=self.prefix, **kw)

    def check(self, window=None, sinks=0, scale=None, **kw):
        out, lse = self.run(window=window, sinks=sinks, scale=scale, **kw)
        for b in range(self.B):
            k, v, P = self.k[b], self.v[b], 0
            if self.plens:
                i = self.B + b // (self.B // len(self.plens))
                P = self.plens[i - self.B]
                k, v = torch.cat([self.k[i], k]), torch.cat([self.v[i], v])
            m, n = self.new[b], self.lens[b]
            ref = R.attend(self.q[b, :m], k, v, torch.arange(P + n - m, P + n), HD ** -0.5 if scale is None else scale,
                           window, sinks)
            R.check(out[b, :m], lse[b, :, :m], ref)
            assert not out[b, m:].any() and (lse[b, :, m:] == -torch.inf).all()
        return out, lse


@pytest.mark.parametrize("T,Hq,Hkv,lens,new", [
    (1, 1, 1, [1], None),
    (1, 32, 8, [300], None),
    (1, 8, 8, [64, 63, 65, 1, 0, 128], None),
    (1, 6, 2, [2000, 3, 700], None),
    (2, 8, 1, [5, 257], None),               # 16 rows
    (5, 12, 3, [5, 70, 333], [5, 0, 3]),     # 20 rows of one block of 32
    (4, 8, 1, [900, 64], [4, 1]),            # 32 rows
    (11, 6, 2, [130, 11], None),             # 33 rows
    (100, 4, 1, [100, 500, 164], [100, 77, 100]),
    (130, 2, 2, [130, 700], None),
    (1, 40, 1, [100, 900], None),            # many heads of one kv head
])
def test_attention(dev, T, Hq, Hkv, lens, new):
    Setup(T, Hq, Hkv, lens, new).check()


@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (64, 0), (100, 4), (257, 64), (63, 100), (1000, 1), (5000, 4),
                                          (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("T,Hq,Hkv,lens,new", [
    (1, 8, 2, [2000, 300, 1], None),
    (3, 8, 2, [700, 2, 66], [3, 2, 0]),
    (90, 4, 2, [1500, 90, 333], [90, 20, 77]),
])
def test_windows_and_sinks(dev, T, Hq, Hkv, lens, new, window, sinks):
    Setup(T, Hq, Hkv, lens, new, seed=1).check(window, sinks)


@pytest.mark.parametrize("T,Hq,Hkv,lens,new,plens", [
    (1, 8, 2, [1, 70, 300], None, [200]),                    # 12 rows share a prefix
    (1, 8, 1, [1, 70, 300, 64], None, [200, 65]),            # 16
    (3, 16, 4, [3, 60, 9, 70], [3, 0, 2, 3], [1000, 0]),     # 24; a group without prefix
    (2, 8, 2, [1, 70, 0, 64, 2, 9, 130, 33], None, [640]),   # 64 rows
    (40, 4, 1, [40, 99, 200], [40, 7, 40], [333]),
    (1, 4, 2, [0, 0], None, [100]),                          # nothing new: no rows
])
@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3), (150, 70), (300, 0)])
def test_prefixes(dev, T, Hq, Hkv, lens, new, plens, window, sinks):
    Setup(T, Hq, Hkv, lens, new, plens, seed=2).check(window, sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 70)])
@pytest.mark.parametrize("T,Hq,Hkv,lens,new,plens", [
    (300, 4, 1, [300, 777, 512], [300, 77, 0], None),        # five row blocks, in runs that end anywhere
    (500, 8, 2, [1500], None, None),
    (70, 12, 2, [70, 400, 90, 71], [70, 64, 1, 0], [900, 63]),
    (33, 8, 1, [33, 200], None, [4000, 4000]),
])
def test_many_rows(dev, T, Hq, Hkv, lens, new, plens, window, sinks):
    Setup(T, Hq, Hkv, lens, new, plens or (), seed=12).check(window, sinks)


def test_many_sequences_of_many_rows(dev):
    """More columns than workgroups: most rows are written as their only piece."""
    lens = [40 + (97 * i) % 300 for i in range(70)]
    Setup(40, 16, 4, lens, [(11 * i) % 41 for i in range(70)], seed=13, extra=0).check()


@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 70)])
@pytest.mark.parametrize("T,Hq,Hkv,lens,new", [
    (413, 30, 2, [1500], None),                                  # five pieces a row, 12390 rows
    (413, 30, 2, [1500, 500, 0], [413, 100, 0]),
    (1, 28, 4, [1 + (613 * i) % 3000 for i in range(450)], [i % 7 != 0 for i in range(450)]),
    (9, 32, 16, [9 + (613 * i) % 2500 for i in range(50)], [i % 10 for i in range(50)]),
])
def test_joins_of_many_rows(dev, T, Hq, Hkv, lens, new, window, sinks):
    """More than 12288 rows: a wavefront joins eight, of pieces of several numbers, written
    ones and padding."""
    Setup(T, Hq, Hkv, lens, None if new is None else [int(n) for n in new], seed=15).check(window, sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 70)])
@pytest.mark.parametrize("T,Hq,Hkv,lens,new,plens", [
    (100, 32, 2, [150, 220, 101, 300], [100, 1, 60, 0], [700, 64]),
    (100, 33, 3, [150, 220, 0, 3000], None, [5000]),
    (1, 28, 4, [(61 * i) % 400 for i in range(500)], None, [(331 * i) % 1500 for i in range(10)]),
    (1, 32, 4, [1 + (7 * i) % 90 for i in range(400)], [int(i % 9 != 0) for i in range(400)], [(77 * i) % 300 for i in range(100)]),
])
def test_joins_of_many_rows_with_prefixes(dev, T, Hq, Hkv, lens, new, plens, window, sinks):
    Setup(T, Hq, Hkv, lens, new, plens, seed=17).check(window, sinks)


@pytest.mark.parametrize("plens", [(), (900,)])
def test_a_bad_query_row_stays_alone_among_many(dev, plens):
    s = Setup(120, 64, 1, [3000, 2000], [120, 50], plens, seed=16)
    a, al = s.run()
    for bad in (float("nan"), float("inf")):
        q = s.q.clone()
        s.q[1, 50:] = bad                       # padding
        s.q[0, 1, 0] = bad
        b, bl = s.run()
        s.q.copy_(q)
        assert torch.isnan(b[0, 1, 0]).all()
        b[0, 1, 0], bl[0, 0, 1] = a[0, 1, 0], al[0, 0, 1]
        assert torch.equal(a, b) and torch.equal(al, bl)


@pytest.mark.parametrize("T,Hq,lens,new,plens", [
    (4, 4, [300, 90], [4, 2], None), (4, 4, [3000, 90], [4, 2], None), (6, 8, [3000, 90], [6, 2], None),
    (60, 8, [300, 90], [60, 2], None), (4, 4, [300, 90], [4, 2], [200]), (20, 8, [300, 90], [20, 2], [500]),
])
def test_a_bad_query_row_stays_alone(dev, T, Hq, lens, new, plens):
    """NaN and infinity in padding and in one row: the other rows keep their bits."""
    s = Setup(T, Hq, 1, lens, new, plens or (), seed=14)
    a, al = s.run(window=200, sinks=3)
    for bad in (float("nan"), float("inf"), -3e38):
        q = s.q.clone()
        s.q[1, 2:] = bad                    # padding
        s.q[0, 1, 0] = bad
        b, bl = s.run(window=200, sinks=3)
        s.q.copy_(q)
        assert torch.isnan(b[0, 1, 0]).all() or bad == -3e38
        b[0, 1, 0], bl[0, 0, 1] = a[0, 1, 0], al[0, 0, 1]
        assert torch.equal(a, b) and torch.equal(al, bl)


@pytest.mark.parametrize("T,Hq", [(3, 2), (70, 4)])
def test_lengths_outside_the_tables_are_clamped(dev, T, Hq):
    s = Setup(T, Hq, 2, [128, 128, 30], extra=0, seed=15)
    q, p = s.q, s.pages
    a = s.cache.attention(q, p, ints([128, 0, 30]), new_lens=ints([T, 0, 2]))
    b = s.cache.attention(q, p, ints([2 ** 31 - 1, -5, 30]), new_lens=ints([2 ** 31 - 1, T, 2]))
    c = s.cache.attention(q, p, ints([500, 128, 30]), new_lens=ints([T + 1, -3, 2]))
    for x in (b, c):
        assert torch.equal(a[0], x[0]) and torch.equal(a[1], x[1])
    k0, _ = s.cache.read(p, ints([128, 0, 30]), T, ints([T, 0, 2]))
    k1, _ = s.cache.read(p, ints([2 ** 31 - 1, -5, 30]), T, ints([2 ** 31 - 1, T, 2]))
    assert torch.equal(k0, k1)
    pre = (s.table[:1], ints([2 ** 31 - 1]))
    x = s.cache.attention(q, p, ints([128, 0, 30]), new_lens=ints([T, 0, 2]), prefix=pre)
    y = s.cache.attention(q, p, ints([128, 0, 30]), new_lens=ints([T, 0, 2]), prefix=(s.table[:1], ints([128])))
    assert torch.equal(x[0], y[0])
    z = s.cache.attention(q, p, ints([128, 0, 30]), new_lens=ints([T, 0, 2]), prefix=(s.table[:1], ints([-1])))
    R.check(z[0][2, :2], z[1][2, :, :2], R.attend(q[2, :2], s.k[2], s.v[2], torch.arange(28, 30), HD ** -0.5))


def test_calls_at_once_on_two_streams(dev):
    """Each with its own workspace, over one cache."""
    s = Setup(1, 8, 2, [5000, 333, 64], seed=16)
    t = Setup(50, 8, 2, [700, 90], plens=[900], seed=17)
    want = s.run(), t.run()
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(5):
        with torch.cuda.stream(sa):
            a = s.run(), s.run(window=200, sinks=4)
        with torch.cuda.stream(sb):
            b = t.run()
        got.append((a[0], b))
    torch.cuda.synchronize()
    for a, b in got:
        for x, y in zip(a + b, want[0] + want[1]):
            assert torch.equal(x, y)


def test_no_sequences(dev):
    cache = ops.Kv8Cache(2, 1)
    none, q = torch.empty(0, 3, dtype=I32, device="cuda"), torch.empty(0, 1, 2, HD, dtype=BF, device="cuda")
    out, lse = cache.attention(q, none, ints([]))
    assert out.shape == (0, 1, 2, HD) and lse.shape == (0, 2, 1)
    k = torch.empty(0, 1, 1, HD, dtype=BF, device="cuda")
    cache.write(k, k, none, ints([]))
    assert cache.read(none, ints([]), 1)[0].shape == (0, 1, 1, HD)


@pytest.mark.parametrize("T,lens,window,sinks", [(1, [400, 100], 60, 2), (1, [400, 300], None, 0), (40, [400, 100], 60, 2)])
def test_a_bad_token_reaches_the_rows_that_see_it(dev, T, lens, window, sinks):
    """Values of NaN at token 341 of the first sequence, and at one that no row sees."""
    s = Setup(T, 4, 2, lens, seed=3, bad=[(0, 341), (0, 100)])
    out, lse = s.run(window=window, sinks=sinks)
    for b in range(2):
        m = s.new[b]
        ref = R.attend(s.q[b, :m], s.k[b], s.v[b], torch.arange(lens[b] - m, lens[b]), HD ** -0.5, window, sinks)
        got, want = out[b, :m].cpu(), ref[0]
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        ok = ~torch.isnan(want)
        assert ((got.double() - want)[ok].abs() <= 2.0 ** -8 * (1 + 2.0 ** -6) * (want.abs() + ref[2])[ok]).all()


@pytest.mark.parametrize("scale,q_std", [(1.0, 4.0), (1e-6, 1.0), (0.05, 100.0)])
@pytest.mark.parametrize("T", [1, 50])
def test_flat_and_peaked_rows(dev, T, scale, q_std):
    Setup(T, 4, 2, [700, 90], seed=4, q_std=q_std).check(scale=scale)


def test_a_long_cache(dev):
    """70,001 tokens: pieces of more pages."""
    s = Setup(1, 4, 1, [70001], seed=5)
    s.check()
    s.check(window=66000, sinks=100)


@pytest.mark.parametrize("T", [1, 40])
def test_offsets_past_32_bits(dev, T):
    """A pool of 4.4 GB; its last pages."""
    n = 262144
    s = Setup(T, 2, 1, [200], seed=6)
    big = ops.Kv8Cache(n, 1)
    w = s.pages.shape[1]
    top = torch.arange(n - w, n, dtype=I32, device="cuda").flip(0)[None].contiguous()
    big.data[(n - w) * R.HEAD_B:].fill_(0xFF)
    k, v = s.cache.read(s.pages, ints([200]), 200)
    big.write(k, v, top, ints([200]))
    k2, v2 = big.read(top, ints([200]), 200)
    small = stale(ops.Kv8Cache(w, 1))
    low = torch.arange(w, dtype=I32, device="cuda")[None].contiguous()
    small.write(k, v, low, ints([200]))
    k3, v3 = small.read(low, ints([200]), 200)
    assert torch.equal(k2, k3) and torch.equal(v2, v3)
    for x, y in zip(big.attention(s.q, top, ints([200])), small.attention(s.q, low, ints([200]))):
        assert torch.equal(x, y)


@pytest.mark.parametrize("T", [2, 40])
def test_results_repeat(dev, T):
    """The same call twice gives the same bits."""
    s = Setup(T, 8, 2, [900, 5, 333, 64], plens=[500, 30], seed=7)
    a, b = s.run(), s.run()
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_more_sequences_than_a_workgroup_has_threads(dev):
    lens = [1 + (37 * i) % 90 for i in range(300)]
    s = Setup(1, 2, 1, lens, seed=8, extra=0)
    s.check()
    lens = [1 + i % 3 for i in range(600)]
    Setup(1, 2, 1, lens, seed=9, plens=[1 + i % 70 for i in range(300)], extra=0).check(window=64, sinks=1)


@pytest.mark.parametrize("B,n", [(3, 5000), (40, 700)])
def test_runs_that_cross_segments_and_heads(dev, B, n):
    """More pages than wavefronts: their runs end in other segments than they start in."""
    lens = [n - (n * 7 * i) % n // 2 if i % 5 else i % 2 for i in range(B)]
    Setup(1, 16, 16, lens, seed=11).check(window=n // 2, sinks=65)


def test_no_tables_no_tokens(dev):
    cache = ops.Kv8Cache(2, 1)
    none = torch.empty(2, 0, dtype=I32, device="cuda")
    q = rows((2, 1, 2, HD), 1).cuda()
    out, lse = cache.attention(q, none, ints([5, 0]))
    assert not out.any() and (lse == -torch.inf).all()
    k, _ = cache.read(none, ints([5, 0]), 1)
    assert not k.any()
    out, lse = cache.attention(q, none, ints([5, 0]), prefix=(ints([[1]]), ints([3])))
    assert not out.any() and (lse == -torch.inf).all()


def test_strided_q_tables_and_a_given_workspace(dev):
    s = Setup(3, 6, 2, [70, 200], seed=10)
    want = s.run()
    qkv = torch.zeros(2, 3, 10, HD, dtype=BF, device="cuda")
    qkv[:, :, :6] = s.q
    wide = torch.full((2, s.pages.shape[1] + 5), -7, dtype=I32, device="cuda")
    wide[:, :s.pages.shape[1]] = s.pages
    ws = torch.empty(1 << 24, dtype=torch.uint8, device="cuda")
    got = s.cache.attention(qkv[:, :, :6], wide[:, :s.pages.shape[1]], ints(s.lens), workspace=ws)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = s.cache.attention(s.q, wide, ints(s.lens))  # pages past the sequences' ends are never looked at
    R.check(got[0][0], got[1][0], R.attend(s.q[0], s.k[0], s.v[0], torch.arange(67, 70), HD ** -0.5))


# ------------------------------------------------- streams, graphs, devices
def test_another_stream_and_a_graph(dev):
    """A generation step captured once: new tokens into the cache, attention, the
    lengths counted up; each replay against the eager call."""
    B, Hq, Hkv, steps = 3, 8, 2, 70
    start = [1, 60, 127]
    cache, eager = stale(ops.Kv8Cache(24, Hkv)), stale(ops.Kv8Cache(24, Hkv))
    pages = R.tables([n + steps for n in start], 24, 1).cuda()
    k0, v0 = rows((B, 127, Hkv, HD), 1).cuda(), rows((B, 127, Hkv, HD), 2).cuda()
    for c in (cache, eager):
        c.write(k0, v0, pages, ints(start), ints(start))
    toks = rows((steps, B, 1, Hq + 2 * Hkv, HD), 3).cuda()
    x, lens = torch.zeros_like(toks[0]), ints(start)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()

    def step():
        lens.add_(1)
        cache.write(x[:, :, Hq:Hq + Hkv], x[:, :, Hq + Hkv:], pages, lens)
        return cache.attention(x[:, :, :Hq], pages, lens, window=100, sinks=4)

    with torch.cuda.stream(side):
        cache.read(pages, lens, 1)
        cache.attention(x[:, :, :Hq], pages, lens)  # the kernels' limits are set before the capture
    side.synchronize()
    with torch.cuda.graph(graph, stream=side):
        out, lse = step()
    lens.copy_(ints(start))
    n = ints(start)
    for i in range(steps):
        x.copy_(toks[i])
        graph.replay()
        n = n + 1
        y = toks[i]
        eager.write(y[:, :, Hq:Hq + Hkv], y[:, :, Hq + Hkv:], pages, n)
        a, b = eager.attention(y[:, :, :Hq], pages, n, window=100, sinks=4)
        torch.cuda.synchronize()
        assert torch.equal(out, a) and torch.equal(lse, b), i


def test_refusals(dev):
    cache = ops.Kv8Cache(4, 2)
    k = torch.zeros(2, 3, 2, HD, dtype=BF, device="cuda")
    q = torch.zeros(2, 3, 4, HD, dtype=BF, device="cuda")
    pages, lens = ints([[0, 1], [2, 3]]), ints([3, 3])
    for bad in (dict(k=k[:, :, :1]), dict(k=k.float()), dict(k=k.cpu()), dict(v=k[:1]), dict(pages=pages.long()),
                dict(pages=pages[:1]), dict(pages=pages.t()), dict(lens=lens.long()), dict(lens=lens[:1]),
                dict(lens=lens.cpu()), dict(new_lens=ints([1])), dict(k=k.transpose(0, 1))):
        a = dict(k=k, v=k.clone(), pages=pages, lens=lens)
        a.update(bad)
        with pytest.raises(ValueError):
            cache.write(**a)
    for bad in (dict(q=q[..., :64]), dict(q=q.float()), dict(window=0), dict(window=-1),
                dict(window=2 ** 32 + 5), dict(sinks=-1), dict(sinks=2 ** 32),
                dict(prefix=(pages[:0], lens[:0])), dict(prefix=(pages, lens.long())),
                dict(prefix=(pages, lens), workspace=torch.empty(16, dtype=torch.uint8, device="cuda"))):
        a = dict(q=q, pages=pages, lens=lens)
        a.update(bad)
        with pytest.raises(ValueError):
            cache.attention(**a)
    for bad in (dict(q=q[:, :, :3].contiguous()), dict(scale=0.0), dict(scale=float("nan")),
                dict(prefix=(ints([[0]] * 3), ints([1] * 3)))):
        a = dict(q=q, pages=pages, lens=lens)
        a.update(bad)
        with pytest.raises(ops.F.GltError):
            cache.attention(**a)
    with pytest.raises(ValueError):
        ops.Kv8Cache(4, 2, head_dim=64)
    with pytest.raises(ValueError):
        ops.Kv8Cache(0, 2)


@pytest.mark.parametrize("sinks", [1, 3, 2 ** 31 - 1])
def test_sinks_are_refused_without_a_window(dev, sinks):
    """As in training: they say nothing where every token is seen, so the window was forgotten."""
    s = Setup(1, 4, 2, [300], seed=18)
    with pytest.raises(ValueError, match="sinks"):
        s.run(sinks=sinks)
    s.check(window=20, sinks=sinks)


@pytest.mark.parametrize("T", [1, 5, 40])
def test_no_tables_behind_prefixes(dev, T):
    """Few, some and many rows that all come to nothing."""
    s = Setup(1, 8, 2, [3, 3, 3, 3], plens=[500, 70], seed=19)
    none = torch.empty(4, 0, dtype=I32, device="cuda")
    q = rows((4, T, 8, HD), 1).cuda()
    out, lse = s.cache.attention(q, none, ints([5, 0, 1, T]), prefix=s.prefix)
    assert not out.any() and (lse == -torch.inf).all()


@pytest.mark.parametrize("window,sinks", [(None, 0), (50, 3), (150, 70), (300, 0)])
@pytest.mark.parametrize("T,Hq,Hkv,lens,new,plens", [
    (5, 8, 2, [5, 60, 9, 370], [5, 0, 2, 4], [1000]),           # 80 rows of a prefix, 20 of a sequence
    (5, 8, 2, [5, 60, 9, 370], None, [1000, 64, 0, 333]),       # 20 and 20
    (8, 12, 3, [8, 300, 70, 64, 9, 200], [8, 3, 0, 8, 1, 7], [130, 700]),  # 96, 32
    (4, 8, 1, [700, 4], [4, 2], [63, 2000]),                    # 32, 32
    (8, 4, 1, [20 + 3 * i for i in range(70)], [i % 9 for i in range(70)], [257]),  # more sequences than lanes
])
def test_two_row_blocks_behind_a_prefix(dev, T, Hq, Hkv, lens, new, plens, window, sinks):
    """17 to 32 own rows a sequence and head beside a prefix's few or many."""
    Setup(T, Hq, Hkv, lens, new, plens, seed=20).check(window, sinks)


@pytest.mark.parametrize("window,sinks", [(None, 0), (150, 70)])
@pytest.mark.parametrize("T,plens", [
    (5, [(97 * i) % 900 for i in range(20)]),                   # 200 rows of a prefix
    (5, [(31 * i) % 400 for i in range(200)]),                  # 20
])
def test_joins_of_two_row_blocks_behind_a_prefix(dev, T, plens, window, sinks):
    """16000 rows: eight joined by a wavefront."""
    lens = [T + (53 * i) % 300 for i in range(200)]
    Setup(T, 16, 4, lens, [i % (T + 1) for i in range(200)], plens, seed=21).check(window, sinks)


@pytest.mark.parametrize("T,Hq,lens,new,plens", [
    (6, 4, [3000, 90], [6, 2], None), (8, 4, [300, 90], [8, 2], None),      # 24, 32 rows
    (6, 4, [300, 90], [6, 2], [200]), (8, 4, [300, 90], [8, 3], [500, 70]),  # beside 48 and 32 of a prefix
])
def test_a_bad_query_row_stays_alone_in_two_row_blocks(dev, T, Hq, lens, new, plens):
    """NaN and infinity in padding and in a row of either block of 16."""
    s = Setup(T, Hq, 1, lens, new, plens or (), seed=22)
    a, al = s.run(window=200, sinks=3)
    assert torch.isfinite(a).all()
    for bad in (float("nan"), float("inf")):
        for t, h in ((1, 0), (5, 3)):
            q = s.q.clone()
            s.q[1, 3:] = bad                    # padding
            s.q[0, t, h] = bad
            b, bl = s.run(window=200, sinks=3)
            s.q.copy_(q)
            assert torch.isnan(b[0, t, h]).all() and torch.isnan(bl[0, h, t])
            b[0, t, h], bl[0, h, t] = a[0, t, h], al[0, h, t]
            assert torch.equal(a, b) and torch.equal(al, bl)


@pytest.mark.parametrize("q_std", [1e8, 1e10, 1e20, 1e30])
@pytest.mark.parametrize("T,lens,plens", [(1, [700], ()), (1, [3000], ()), (8, [700], ()), (100, [700, 164], ()),
                                          (100, [5000], ()), (60, [700], [500])])
def test_scores_of_any_size(dev, T, lens, plens, q_std):
    """Past 2^24 a step of f32 between two scores is more than a whole power of e: the weights
    are those of a few keys (whichever rounding leaves in front), finite and no larger than the values."""
    s = Setup(T, 4, 1, lens, None, plens, seed=23, q_std=q_std)
    top = max(float(v.abs().max()) for v in s.v)
    for sign in (1, -1):
        s.q *= sign
        out, lse = s.check(scale=1.0)
        assert float(out.abs().max()) <= top * (1 + 2.0 ** -7)  # two roundings, of p and of the result


@pytest.mark.parametrize("T,n", [(1, 1), (1, 40), (1, 3000), (8, 700), (100, 100), (100, 5000)])
def test_scores_near_the_lowest_f32(dev, T, n):
    """Every score the same, -3.2e38 in units of log2: the mean of the values."""
    cache = stale(ops.Kv8Cache(80, 1))
    pages = torch.arange(80, dtype=I32, device="cuda")[None]
    k, v = torch.full((1, n, 1, HD), 8128.0, dtype=BF), rows((1, n, 1, HD), 24)  # 127 steps of 64
    cache.write(k.cuda(), v.cuda(), pages, ints([n]))
    q = torch.full((1, T, 4, HD), -2.0 ** 111, dtype=BF)
    out, lse = cache.attention(q.cuda(), pages, ints([n]), scale=0.082)
    R.check(out[0], lse[0], R.attend(q[0], R.values(k)[0], R.values(v)[0], torch.arange(n - T, n), 0.082))


@pytest.mark.parametrize("window,sinks", [(1, 1), (33, 64), (64, 4), (128, 0), (128, 4), (100, 200), (500, 65), (600, 1000),
                                          (128, 2 ** 31 - 1), (5000, 3)])
@pytest.mark.parametrize("T,Hq,Hkv,lens,new,plens", [
    (700, 4, 1, [2000, 701, 900], [700, 699, 3], ()),
    (300, 6, 2, [1900], None, ()),
    (300, 4, 2, [1500, 310], [300, 40], [50]),      # sinks of the prefix and behind it
])
def test_sinks_before_the_windows_of_many_rows(dev, T, Hq, Hkv, lens, new, plens, window, sinks):
    """Row blocks whose windows start pages behind the sinks, on them, and before them."""
    Setup(T, Hq, Hkv, lens, new, plens, seed=25).check(window, sinks)


def test_sinks_leave_a_window_its_savings(dev):
    """4096 new tokens with a window of 128: a few sinks are a page more for each row block (four
    for three), not every page between them and its window as well (up to 65)."""
    s = Setup(4096, 32, 8, [4096 + 64], seed=26)

    def least(**kw):
        t = []
        for _ in range(6):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in "ab")
            a.record()
            for _ in range(4):
                s.run(**kw)
            b.record()
            torch.cuda.synchronize()
            t.append(a.elapsed_time(b))
        return min(t)
    assert least(window=128, sinks=4) < 3 * least(window=128)
