"""The 8-bit cache of keys and values and attention over it in 64 bits (CPU)."""
import torch

HD, PAGE, HEAD_B = 128, 64, 16640


def held(x):
    """(codes, steps) f64 of rows [..., 128]: whole steps of bf16(max |x| / 127)."""
    x = x.double().cpu()
    top = x.abs().amax(-1)
    # f32 holds the quotient to 2^-24; no bf16 over 127 lies that close to the middle of two bf16
    step = (top / 127).float().bfloat16().double().clamp(2.0 ** -100, 2.0 ** 121)
    bad = ~torch.isfinite(top)
    step = torch.where(bad, torch.nan, step)
    codes = torch.where(bad[..., None], 0.0, torch.round(x / step[..., None]).clamp(-127, 127))
    return codes, step


def values(x):
    codes, step = held(x)
    return codes * step[..., None]


def tables(lens, n_pages, seed, extra=0):
    """A page table of `lens` tokens a row (and `extra` pages), pages in no order and of no two rows."""
    g = torch.Generator().manual_seed(seed)
    width = max([-(-n // PAGE) for n in lens] + [1]) + extra
    ids = torch.randperm(n_pages, generator=g)[:len(lens) * width].to(torch.int32)
    return ids.view(len(lens), width)


def v_byte(t):
    return (t & 0x33) | ((t & 4) << 1) | ((t & 8) >> 1)


def token_bytes(t):
    """Offsets in a page's head that hold token t of the page."""
    k = [t * HD + d for d in range(HD)]
    v = [8192 + d * PAGE + v_byte(t) for d in range(HD)]
    return k + v + [16384 + 2 * t, 16384 + 2 * t + 1, 16512 + 2 * t, 16512 + 2 * t + 1]


def attend(q, k, v, pos, scale, window=None, sinks=0):
    """One sequence: q [m, Hq, 128] at positions pos [m], k and v [n, Hkv, 128].
    Returns out, lse, the sums of p |v| that the roundings scale with, and the
    largest sum of |q k| of a row's keys, f64."""
    q, k, v = q.double().cpu(), k.double().cpu(), v.double().cpu()
    m, Hq, n, Hkv = q.shape[0], q.shape[1], k.shape[0], k.shape[1]
    j = torch.arange(n)
    see = j[None] <= pos[:, None]
    if window:
        see = see & ((j[None] > pos[:, None] - window) | (j[None] < sinks))
    out, mag = torch.zeros(m, Hq, HD, dtype=torch.float64), torch.zeros(m, Hq, HD, dtype=torch.float64)
    lse, big = torch.full((Hq, m), -torch.inf, dtype=torch.float64), torch.zeros(Hq, m, dtype=torch.float64)
    if n == 0 or m == 0:
        return out, lse, mag, big
    for h in range(Hq):
        kh, vh = k[:, h // (Hq // Hkv)], v[:, h // (Hq // Hkv)]
        s = torch.where(see, q[:, h] @ kh.t() * scale, -torch.inf)
        some = see.any(-1)
        lse[h] = torch.logsumexp(s, -1)
        p = torch.where(see, torch.exp(s - torch.where(some, lse[h], 0.0)[:, None]), 0.0)
        # what a row does not see counts for nothing, NaN included
        bad = torch.isnan(vh).any(-1) | torch.isnan(kh).any(-1)
        p0, v0 = torch.where(bad[None], 0.0, p), torch.where(bad[:, None], 0.0, vh)
        hit = (see & bad[None]).any(-1)
        out[:, h], mag[:, h] = p0 @ v0, p0 @ v0.abs()
        out[hit, h], lse[h, hit] = torch.nan, torch.nan
        big[h] = torch.where(see, q[:, h].abs() @ torch.where(bad[:, None], 0.0, kh).abs().t() * scale, 0.0).amax(-1)
    return out, lse, mag, big


def check(out, lse, ref):
    """Half a step of bf16 of out, as much of the sums of p |v| (p times the
    step, rounded before the product), and 128 f32 roundings of the scores, which
    change weights and lse by as much. bf16 has 8 significant bits: values from 1 to 2
    are 2^-7 apart, so half a step is at most 2^-8 of the value."""
    r_out, r_lse, mag, big = ref
    out, lse = out.double().cpu(), lse.double().cpu()
    assert torch.equal(torch.isnan(out), torch.isnan(r_out)) and torch.equal(torch.isnan(lse), torch.isnan(r_lse))
    assert torch.equal(torch.isinf(lse), torch.isinf(r_lse))
    eps = 128 * 2.0 ** -24 * big + 2.0 ** -20  # of a score; exp2 and the sums' orders
    d = (out - r_out).nan_to_num(0.0).abs()
    # the bf16 exponent's lower end apart
    lim = 2.0 ** -8 * (1 + 2.0 ** -8) * (r_out.abs() + mag).nan_to_num(0.0) + 2 * eps.t()[..., None] * mag + 2.0 ** -126
    assert (d <= lim).all(), f"out off by {(d / lim).max():.3f} of its bound"
    fin = torch.isfinite(r_lse)
    dl = (lse - r_lse)[fin].abs()
    ll = (eps + 2.0 ** -21 * r_lse.abs())[fin]
    assert (dl <= ll).all(), f"lse off by {(dl / ll).max():.3f} of its bound"
