"""Operators that produce answers and train with limited sight: what a call of
each takes and gives, its plain form in torch, and its 64-bit result.

* kv8       new tokens' keys and values into a paged 8-bit cache and back.
* decode    attention of new tokens over that cache: one token a sequence or
            several, with a sliding window and first tokens that stay visible
            (sinks), with a prefix that a group of sequences shares.
* win_fwd   attention for training with such a window and sinks: output and
            log-sum-exp of each row.
* win_bwd   its backward from q, k, v, out, lse and dout.

listed() holds sizes of each, draw() spreads over the ranges they stand for.
`own` selects the framework's entry points, otherwise run() computes the plain
form.
"""
import math

import torch

own = False

DEV = "cuda"
BF, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
HD = 128
PAGE = 64  # tokens of a page of the cache
NEG = float("-inf")


# ------------------------------------------------------------------ cases
def listed():
    """Cache cases: B sequences, each holding lo to hi tokens with its new ones
    counted; T new tokens a sequence, fewer where ragged (`new` from 0 to T).
    group: consecutive sequences that share a prefix (0 = none) of plo to phi
    tokens. window 0 = none. Training cases: B sequences padded to T, `lens`
    their true lengths ("" = all T); fused = views of one projection output."""
    return [
        # one generation step of a batch of 64: each sequence's new token into its last page
        dict(name="kv8_64x1", kind="kv8", B=64, T=1, Hkv=8, lo=1, hi=4096, ragged=False),
        # a batch of prompts of odd lengths into the cache
        dict(name="kv8_8x4096_ragged", kind="kv8", B=8, T=4096, Hkv=8, lo=4096, hi=4096, ragged=True),
        # a single short conversation: latency
        dict(name="decode_1x300", kind="decode", B=1, T=1, Hq=32, Hkv=8, lo=300, hi=300, ragged=False, group=0, plo=0,
             phi=0, window=0, sinks=0),
        # a serving step of 32 sequences from short to long
        dict(name="decode_32_to_32768", kind="decode", B=32, T=1, Hq=32, Hkv=8, lo=1, hi=32768, ragged=False, group=0,
             plo=0, phi=0, window=0, sinks=0),
        # long conversations of a model with a window
        dict(name="decode_48_window", kind="decode", B=48, T=1, Hq=32, Hkv=8, lo=900, hi=16000, ragged=False, group=0,
             plo=0, phi=0, window=1024, sinks=4),
        # two prompts continued in pieces: 512 and fewer new tokens over what is cached
        dict(name="decode_2x512_pieces", kind="decode", B=2, T=512, Hq=32, Hkv=8, lo=5000, hi=8704, ragged=True, group=0,
             plo=0, phi=0, window=0, sinks=0),
        # 64 answers sampled from one long prompt, for training on them
        dict(name="prefix_64_of_16384", kind="decode", B=64, T=1, Hq=32, Hkv=8, lo=1, hi=512, ragged=False, group=64,
             plo=16384, phi=16384, window=0, sinks=0),
        # four prompts of odd lengths, eight answers each, up to three proposed tokens checked at once
        dict(name="prefix_4x8_of_1999", kind="decode", B=32, T=3, Hq=16, Hkv=4, lo=3, hi=700, ragged=True, group=8,
             plo=77, phi=1999, window=0, sinks=0),
        # the benchmark's decoder layer (2 x 4096 tokens, 32/8 heads) with a window
        dict(name="win_fwd_2x4096", kind="win_fwd", B=2, T=4096, Hq=32, Hkv=8, lens="", window=1024, sinks=4, fused=False),
        # a padded batch out of a fused projection, no sinks, an odd window
        dict(name="win_fwd_5x701_padded", kind="win_fwd", B=5, T=701, Hq=16, Hkv=4, lens="701,600,1,333,0", window=129,
             sinks=0, fused=True),
        # the same layer's backward
        dict(name="win_bwd_2x4096", kind="win_bwd", B=2, T=4096, Hq=32, Hkv=8, lens="", window=1024, sinks=4, fused=False),
        # one long document with a short window and many visible first tokens
        dict(name="win_bwd_1x12001", kind="win_bwd", B=1, T=12001, Hq=16, Hkv=4, lens="", window=500, sinks=70, fused=True),
    ]


def _log_int(rng, lo, hi):
    """Log-uniform whole number in [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["kv8", "decode", "decode", "decode", "win_fwd", "win_bwd"])
    Hq, Hkv = rng.choice([(32, 8), (16, 4), (8, 8), (32, 4), (6, 2), (8, 1)])
    if kind == "kv8":
        B = _log_int(rng, 1, 64)
        T = _log_int(rng, 1, max(1, 8 * 4096 * 8 // (B * Hkv)) if B * Hkv > 64 else 4096)
        lo = rng.choice([T, T, T + rng.randint(0, 200)])
        return dict(kind=kind, B=B, T=T, Hkv=Hkv, lo=lo, hi=lo + rng.choice([0, rng.randint(0, 500)]),
                    ragged=rng.random() < 0.5)
    if kind == "decode":
        B, T = _log_int(rng, 1, 64), rng.choice([1, 1, 1, 2, 5, _log_int(rng, 1, 512)])
        B = max(1, min(B, 1024 * 32 // (T * Hq)))
        hi = max(T + 1, _log_int(rng, 1, max(2, min(32768, 32 * 13000 * 8 // (B * Hkv), 2 * 512 * 32 * 7000 // (B * T * Hq)))))
        c = dict(kind=kind, B=B, T=T, Hq=Hq, Hkv=Hkv, lo=rng.randint(T, hi), hi=hi, ragged=rng.random() < 0.4, group=0,
                 plo=0, phi=0, window=0, sinks=0)
        if rng.random() < 0.4:
            c["group"] = rng.choice([g for g in range(1, B + 1) if B % g == 0])
            c["phi"] = _log_int(rng, 1, min(16384, 64 * 16384 * 32 // (B * T * Hq)))
            c["plo"] = rng.randint(0, c["phi"])
        if rng.random() < 0.4:
            c["window"], c["sinks"] = _log_int(rng, 1, 4096), rng.choice([0, 1, 4, 64, 100])
        return c
    B = rng.randint(1, 6)
    W = _log_int(rng, 1, 4096)
    # no more pairs than the listed layer has, nor more columns than the long document
    T = _log_int(rng, 1, min(12000, 2 * 32 * 4096 * 900 // (B * Hq * W), math.isqrt(16 * 12001 ** 2 // (B * Hq))))
    lens = ""
    if rng.random() < 0.5:
        lens = ",".join(str(rng.randint(0, T) if rng.random() < 0.8 else T) for _ in range(B))
        if not any(int(v) for v in lens.split(",")):
            lens = ""
    return dict(kind=kind, B=B, T=T, Hq=Hq, Hkv=Hkv, lens=lens, window=W, sinks=rng.choice([0, 1, 4, 64, 100]),
                fused=rng.random() < 0.5)


def _spread(lo, hi, n):
    """n whole numbers from hi down to lo, in a mixed order."""
    return [hi - (hi - lo) * ((5 * i) % n) // max(n - 1, 1) for i in range(n)]


def _own_lens(case):
    """Tokens that each sequence holds, and how many of them are new."""
    B, T = case["B"], case["T"]
    new = _spread(0, T, B) if case["ragged"] and B > 1 else [T] * B
    return [max(n, m) for n, m in zip(_spread(case["lo"], case["hi"], B), new)], new


def _prefix_lens(case):
    return _spread(case["plo"], case["phi"], case["B"] // case["group"]) if case.get("group") else []


def _lens(case):
    return [int(v) for v in case["lens"].split(",")] if case["lens"] else [case["T"]] * case["B"]


# ---------------------------------------------------------------- prepare
class _Draw:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV)
        self.g.manual_seed(int(seed) & 0x7FFFFFFFFFFFFFFF)

    def normal(self, shape, std=1.0, dtype=BF):
        t = torch.empty(shape, dtype=F32, device=DEV)
        t.normal_(0.0, std, generator=self.g)
        return t if dtype == F32 else t.to(dtype)

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device=DEV)


def _keys_values(d, tokens, Hkv):
    """Keys whose channels differ in size, as trained ones do, and values."""
    k = d.normal((tokens, Hkv, HD), dtype=F32)
    k *= torch.exp(d.normal((Hkv, HD), 0.5, dtype=F32))
    return k.to(BF), d.normal((tokens, Hkv, HD))


def _cache_inputs(case, seed):
    """Tokens of the sequences and then of the prefixes, packed, q, and the
    tables of the pages that hold them, in no order."""
    d = _Draw(seed)
    lens, new = _own_lens(case)
    plens = _prefix_lens(case)
    s = dict(lens=lens, new=new, plens=plens)
    if case["kind"] == "kv8":  # padded batch of the new tokens
        k, v = _keys_values(d, case["B"] * case["T"], case["Hkv"])
        s["k"], s["v"] = (t.view(case["B"], case["T"], case["Hkv"], HD) for t in (k, v))
    else:
        s["k"], s["v"] = _keys_values(d, sum(lens) + sum(plens), case["Hkv"])
        s["q"] = d.normal((case["B"], case["T"], case["Hq"], HD), 2.0)
    tables, n_pages = [], 1
    for ls in (lens, plens):
        width = max([-(-n // PAGE) for n in ls] + [1])
        tables.append((len(ls), width))
        n_pages += len(ls) * width
    ids = d.perm(n_pages).to(I32)
    s["pages"] = ids[:tables[0][0] * tables[0][1]].view(tables[0])
    s["ppages"] = ids[tables[0][0] * tables[0][1]:n_pages - 1].view(tables[1])
    s["n_pages"] = n_pages
    return s


def _ints(v):
    return torch.tensor(v, dtype=I32, device=DEV)


def _train_inputs(case, seed):
    """q of twice the keys' size: rows between flat and peaked. What lies past
    a sequence's end is finite and arbitrary."""
    d = _Draw(seed)
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    s = dict(scale=HD ** -0.5, window=case["window"], sinks=case["sinks"])
    if case["fused"]:
        qkv = d.normal((B, T, Hq + 2 * Hkv, HD))
        qkv[:, :, :Hq] *= 2
        s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    else:
        s["q"], s["k"], s["v"] = d.normal((B, T, Hq, HD), 2.0), d.normal((B, T, Hkv, HD)), d.normal((B, T, Hkv, HD))
    s["seq_lens"] = _ints(_lens(case)) if case["lens"] else None
    if case["kind"] == "win_bwd":
        s["dout"] = d.normal((B, T, Hq, HD))
    return s


def prepare(case, seed):
    kind = case["kind"]
    if kind in ("win_fwd", "win_bwd"):
        s = _train_inputs(case, seed)
        if kind == "win_bwd":
            s["out"], s["lse"] = _plain_win_fwd(s)  # what the forward left
        s["kind"] = kind
        return s
    x = _cache_inputs(case, seed)
    B, T, Hkv = case["B"], case["T"], case["Hkv"]
    s = dict(kind=kind, B=B, T=T, pages=x["pages"], lens=_ints(x["lens"]), new=_ints(x["new"]) if case["ragged"] else None)
    if case.get("group"):
        s["prefix"] = (x["ppages"], _ints(x["plens"]))
    else:
        s["prefix"] = None
    if own:
        from glt_amd import ops
        s["cache"] = ops.Kv8Cache(x["n_pages"], Hkv, device=DEV)
    else:
        s["k_codes"], s["v_codes"] = (torch.zeros((x["n_pages"] * PAGE, Hkv, HD), dtype=torch.int8, device=DEV) for _ in "kv")
        s["k_step"], s["v_step"] = (torch.zeros((x["n_pages"] * PAGE, Hkv), dtype=F32, device=DEV) for _ in "kv")
    if kind == "kv8":
        s["k"], s["v"] = x["k"], x["v"]
        return s
    # the cache as the steps before left it, the new tokens written too
    s.update(q=x["q"], window=case["window"], sinks=case["sinks"], scale=HD ** -0.5)
    at = 0
    for pages, lens in ((x["pages"], x["lens"]), (x["ppages"], x["plens"])):
        for b, n in enumerate(lens):
            k, v = x["k"][at:at + n], x["v"][at:at + n]
            at += n
            if n == 0:
                continue
            if own:
                s["cache"].write(k[None], v[None], pages[b:b + 1], _ints([n]))
            else:
                _plain_write(s, _slots(pages[b], torch.arange(n, device=DEV)), k, v)
    return s


# -------------------------------------------------------------------- run
def run(s):
    return (_OWN if own else _PLAIN)[s["kind"]](s)


def _own_kv8(s):
    s["cache"].write(s["k"], s["v"], s["pages"], s["lens"], new_lens=s["new"])
    k, v = s["cache"].read(s["pages"], s["lens"], s["T"], new_lens=s["new"])
    return dict(k=k, v=v)


def _own_decode(s):
    out, lse = s["cache"].attention(s["q"], s["pages"], s["lens"], new_lens=s["new"], scale=s["scale"],
                                    window=s["window"] or None, sinks=s["sinks"], prefix=s["prefix"])
    return dict(out=out, lse=lse)


def _own_win_fwd(s):
    from glt_amd import ops
    out, lse = ops.attention_train(s["q"], s["k"], s["v"], scale=s["scale"], seq_lens=s["seq_lens"], window=s["window"],
                                   sinks=s["sinks"])
    return dict(out=out, lse=lse)


def _own_win_bwd(s):
    from glt_amd import ops
    dq, dk, dv = ops.attention_bwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], scale=s["scale"],
                                   seq_lens=s["seq_lens"], window=s["window"], sinks=s["sinks"])
    return dict(dq=dq, dk=dk, dv=dv)


_OWN = {"kv8": _own_kv8, "decode": _own_decode, "win_fwd": _own_win_fwd, "win_bwd": _own_win_bwd}


# ------------------------------------------------------------ plain forms
def _slots(pages, pos):
    """Rows of the pool that hold positions pos [..., n] of the sequences
    whose tables are pages [..., width]."""
    return pages.long().gather(-1, pos // PAGE) * PAGE + pos % PAGE


def _plain_codes(x):
    """Rows [..., 128] as whole steps: the step (bf16 of the largest magnitude
    over 127, kept from the ends of the exponents) and the codes."""
    x = x.float()
    step = (x.abs().amax(-1) / 127).to(BF).float().clamp_(2.0 ** -100, 2.0 ** 121)
    return torch.round(x / step[..., None]).clamp_(-127, 127).to(torch.int8), step


def _plain_write(s, slots, k, v):
    for name, x in (("k", k), ("v", v)):
        s[name + "_codes"][slots], s[name + "_step"][slots] = _plain_codes(x)


def _plain_rows(s, name, pages, width):
    """f32 [sequences, width, Hkv, 128]: the values of positions 0 .. width - 1."""
    pos = torch.arange(width, device=DEV).expand(pages.shape[0], width)
    slots = _slots(pages, pos)
    return s[name + "_codes"][slots].float().mul_(s[name + "_step"][slots][..., None])


def _plain_kv8(s):
    B, T = s["B"], s["T"]
    new = s["new"].long() if s["new"] is not None else torch.full((B,), T, dtype=I64, device=DEV)
    t = torch.arange(T, device=DEV).expand(B, T)
    live = t < new[:, None]
    # a padding token's position is its sequence's first new one: never written, and read as zeros
    pos = (s["lens"].long() - new)[:, None] + torch.where(live, t, torch.zeros_like(t))
    slots = _slots(s["pages"], pos.clamp_(0, s["pages"].shape[1] * PAGE - 1))
    _plain_write(s, slots[live], s["k"][live], s["v"][live])
    r = {}
    for name in ("k", "v"):
        x = s[name + "_codes"][slots].float() * s[name + "_step"][slots][..., None]
        r[name] = (x * live[:, :, None, None]).to(BF)
    return r


def _plain_decode(s):
    """Scores of the shared prefix by group, of the own tokens by sequence;
    one softmax over both."""
    B, T = s["B"], s["T"]
    Hq, Hkv = s["q"].shape[2], s["k_step"].shape[1]
    G = Hq // Hkv
    new = s["new"].long() if s["new"] is not None else torch.full((B,), T, dtype=I64, device=DEV)
    lens = s["lens"].long()
    head = lambda x: x.transpose(1, 2).contiguous()  # [sequences, Hkv, width, 128]
    q = s["q"].float().mul_(s["scale"]).view(B, T, Hkv, G, HD).transpose(1, 2).reshape(B, Hkv, T * G, HD)
    t = torch.arange(T, device=DEV)
    plen = torch.zeros(B, dtype=I64, device=DEV)
    parts, sight = [], []
    if s["prefix"] is not None:
        ppages, pl = s["prefix"]
        ng, W = ppages.shape[0], int(ppages.shape[1]) * PAGE
        g = B // ng
        plen = pl.long().repeat_interleave(g)
        by_group = lambda x: x.view(ng, g, Hkv, T * G, -1).transpose(1, 2).reshape(ng, Hkv, g * T * G, -1)
        by_seq = lambda x: x.view(ng, Hkv, g, T * G, -1).transpose(1, 2).reshape(B, Hkv, T * G, -1)
        pk, pv = (head(_plain_rows(s, n, ppages, W)) for n in ("k", "v"))
        parts.append((by_seq(torch.matmul(by_group(q), pk.transpose(2, 3).contiguous())),
                      lambda p: by_seq(torch.matmul(by_group(p), pv))))
        j = torch.arange(W, device=DEV)
        sight.append((j.expand(B, W), j[None] < plen[:, None]))
    L = int(s["pages"].shape[1]) * PAGE
    ok, ov = (head(_plain_rows(s, n, s["pages"], L)) for n in ("k", "v"))
    parts.append((torch.matmul(q, ok.transpose(2, 3).contiguous()), lambda p: torch.matmul(p, ov)))
    j = torch.arange(L, device=DEV)
    sight.append((plen[:, None] + j[None], j[None] < lens[:, None]))
    pos = (plen + lens - new)[:, None] + t[None]  # [B, T]
    z = []
    for (x, _), (kpos, live) in zip(parts, sight):
        see = live[:, None] & (kpos[:, None] <= pos[:, :, None]) & (t[None, :, None] < new[:, None, None])
        if s["window"]:
            see &= (kpos[:, None] > pos[:, :, None] - s["window"]) | (kpos[:, None] < s["sinks"])
        z.append(x.masked_fill_(~see.repeat_interleave(G, 1)[:, None], NEG))
    z = torch.cat(z, -1) if len(z) > 1 else z[0]
    m = z.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = z.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    some = l > 0
    p.div_(torch.where(some, l, torch.ones_like(l)))
    at, out = 0, 0
    for (_, times_v), (kpos, _) in zip(parts, sight):
        out = out + times_v(p[..., at:at + kpos.shape[-1]].contiguous())
        at += kpos.shape[-1]
    lse = torch.where(some, m + torch.log(l), torch.full_like(l, NEG))[..., 0]
    return dict(out=out.view(B, Hkv, T, G, HD).transpose(1, 2).reshape(B, T, Hq, HD).to(BF),
                lse=lse.view(B, Hkv, T, G).transpose(2, 3).reshape(B, Hq, T).contiguous())


def _heads(t, rep=1):
    """[B, T, H, 128] of any type -> f32 [B, H * rep, T, 128]."""
    t = t.float().transpose(1, 2)
    return (t.repeat_interleave(rep, 1) if rep > 1 else t).contiguous()


def _sight(s, T):
    """[B or 1, 1, T, T] truth values: may query row t read key column j."""
    t = torch.arange(T, device=DEV)
    back = t[:, None] - t[None, :]
    ok = ((back >= 0) & ((back < s["window"]) | (t[None, :] < s["sinks"])))[None]
    if s["seq_lens"] is not None:
        live = t[None, :] < s["seq_lens"][:, None]
        ok = ok & live[:, :, None] & live[:, None, :]
    return ok[:, None]


def _plain_probs(s):
    """q, k, v by head, and each row's exponentials, their sum and maximum."""
    rep = s["q"].shape[2] // s["k"].shape[2]
    q, k, v = _heads(s["q"]), _heads(s["k"], rep), _heads(s["v"], rep)
    z = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    z.masked_fill_(~_sight(s, q.shape[2]), NEG)
    m = z.amax(-1, keepdim=True).clamp_(min=-1e30)
    p = z.sub_(m).exp_()
    return q, k, v, p, p.sum(-1, keepdim=True), m


def _plain_win_fwd(s):
    _, _, v, p, l, m = _plain_probs(s)
    some = l > 0
    out = torch.matmul(p, v) / torch.where(some, l, torch.ones_like(l))
    lse = torch.where(some, m + torch.log(l), torch.full_like(l, NEG))[..., 0]
    return out.transpose(1, 2).to(BF).contiguous(), lse


def _plain_win_bwd(s):
    q, k, v, p, l, _ = _plain_probs(s)
    B, Hq, T, _ = q.shape
    Hkv = s["k"].shape[2]
    p.div_(torch.where(l > 0, l, torch.ones_like(l)))
    do = _heads(s["dout"])
    if s["seq_lens"] is not None:
        do = do * (torch.arange(T, device=DEV)[None, :] < s["seq_lens"][:, None])[:, None, :, None]
    group = lambda t: t.view(B, Hkv, Hq // Hkv, T, HD).sum(2).transpose(1, 2).to(BF).contiguous()
    dv = group(torch.matmul(p.transpose(2, 3), do))
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = dp.sub_((p * dp).sum(-1, keepdim=True)).mul_(p).mul_(s["scale"])
    del p
    dq = torch.matmul(ds, k).transpose(1, 2).to(BF).contiguous()
    return dict(dq=dq, dk=group(torch.matmul(ds.transpose(2, 3), q)), dv=dv)


_PLAIN = {"kv8": _plain_kv8, "decode": _plain_decode, "win_fwd": lambda s: dict(zip(("out", "lse"), _plain_win_fwd(s))),
          "win_bwd": _plain_win_bwd}


# ------------------------------------------------------------------- work
def _visible(p, window, sinks):
    """Keys that a query at position p reads, and the first one of its window."""
    first = max(0, p - window + 1) if window else 0
    return p + 1 - first + min(sinks, first), first


def work(case):
    kind, Hkv = case["kind"], case["Hkv"]
    row8 = 2 * (HD + 2)  # a token's key and value and their steps, one head
    if kind == "kv8":  # the new tokens in and out, their codes out and in
        tokens = sum(_own_lens(case)[1])
        return {"bytes": Hkv * (tokens * 2 * (row8 + 2 * HD) + case["B"] * case["T"] * 4 * HD), "flops": 8 * tokens * Hkv * HD}
    Hq, window, sinks = case["Hq"], case["window"], case["sinks"]
    if kind == "decode":
        lens, new = _own_lens(case)
        plens, g = _prefix_lens(case), case["group"] or 1
        pairs, own_keys, pre_keys = 0, 0, [0] * (case["B"] // g)
        for b, (n, m) in enumerate(zip(lens, new)):
            P = plens[b // g] if plens else 0
            pairs += sum(_visible(P + n - m + t, window, sinks)[0] for t in range(m))
            if m == 0:
                continue
            keys, first = _visible(P + n - m, window, sinks)  # what the first new token's sight reaches; the others add theirs
            sunk = min(sinks, first)
            pre = max(0, P - first) + min(sunk, P)
            pre_keys[b // g] = max(pre_keys[b // g], pre)
            own_keys += keys + m - 1 - pre
        b = Hkv * row8 * (own_keys + sum(pre_keys)) + case["B"] * case["T"] * Hq * (2 * 2 * HD + 4)
        return {"bytes": b, "flops": 4 * HD * Hq * pairs}
    lens = _lens(case)
    pairs = sum(_visible(t, window, sinks)[0] for n in lens for t in range(n))
    live, padded = sum(lens), case["B"] * case["T"]
    if kind == "win_fwd":
        return {"bytes": max(2 * HD * live * (Hq + 2 * Hkv) + padded * Hq * (2 * HD + 4), 1), "flops": 4 * HD * Hq * pairs}
    b = 2 * HD * (live * (3 * Hq + 2 * Hkv) + padded * (Hq + 2 * Hkv)) + 4 * live * Hq
    return {"bytes": max(b, 1), "flops": 10 * HD * Hq * pairs}


# ------------------------------------------------------------------ exact
def _held64(x):
    """What the cache holds of rows [..., 128]: the largest magnitude over 127,
    at 8 significant bits, is the step."""
    x = x.double()
    step = x.abs().amax(-1, keepdim=True) / 127
    up = step * (2.0 ** 45 + 1)
    step = (up - (up - step)).clamp(2.0 ** -100, 2.0 ** 121)  # the upper 8 of 53 bits, rounded to nearest
    return torch.round(x / step).clamp(-127, 127) * step


def _sees(pos, keys, window, sinks):
    """[queries, keys] truth values."""
    d = pos[:, None] - keys[None, :]
    return (d >= 0) & ((d < window) | (keys[None, :] < sinks)) if window else d >= 0


def _decode64(case, seed):
    x = _cache_inputs(case, seed)
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    G = Hq // Hkv
    out = torch.zeros((B, T, Hq, HD), dtype=F64, device=DEV)
    lse = torch.full((B, Hq, T), NEG, dtype=F64, device=DEV)
    at = [0]
    for n in x["lens"] + x["plens"]:
        at.append(at[-1] + n)
    for b, (n, m) in enumerate(zip(x["lens"], x["new"])):
        rows = [slice(at[b], at[b + 1])]
        P = 0
        if x["plens"]:
            i = b // case["group"]
            P = x["plens"][i]
            rows.insert(0, slice(at[B + i], at[B + i + 1]))
        if m == 0 or P + n == 0:
            continue
        k, v = (_held64(torch.cat([x[c][r] for r in rows])) for c in ("k", "v"))
        pos, keys = torch.arange(P + n - m, P + n, device=DEV), torch.arange(P + n, device=DEV)
        blind = ~_sees(pos, keys, case["window"], case["sinks"])
        for h in range(Hq):
            z = x["q"][b, :m, h].double() @ k[:, h // G].t() * HD ** -0.5
            z = z.masked_fill(blind, NEG)
            lse[b, h, :m] = torch.logsumexp(z, -1)
            out[b, :m, h] = torch.softmax(z, -1) @ v[:, h // G]
    return dict(out=out, lse=lse)


def _train64(case, seed):
    s = _train_inputs(case, seed)
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    rep, bwd = Hq // Hkv, case["kind"] == "win_bwd"
    new = lambda h: torch.zeros((B, T, h, HD), dtype=F64, device=DEV)
    out, lse = new(Hq), torch.full((B, Hq, T), NEG, dtype=F64, device=DEV)
    dq, dk, dv = (new(Hq), new(Hkv), new(Hkv)) if bwd else (None, None, None)
    for b, n in enumerate(_lens(case)):
        if n == 0:
            continue
        t = torch.arange(n, device=DEV)
        blind = ~_sees(t, t, case["window"], case["sinks"])
        for h in range(Hq):
            q, k, v = s["q"][b, :n, h].double(), s["k"][b, :n, h // rep].double(), s["v"][b, :n, h // rep].double()
            z = (q @ k.t() * s["scale"]).masked_fill(blind, NEG)
            if not bwd:
                lse[b, h, :n] = torch.logsumexp(z, -1)
                out[b, :n, h] = torch.softmax(z, -1) @ v
                continue
            p = torch.softmax(z, -1)
            do = s["dout"][b, :n, h].double()
            dp = do @ v.t()
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * s["scale"]
            dv[b, :n, h // rep] += p.t() @ do
            dk[b, :n, h // rep] += ds.t() @ q
            dq[b, :n, h] = ds @ k
    return dict(dq=dq, dk=dk, dv=dv) if bwd else dict(out=out, lse=lse)


def exact(case, seed):
    if case["kind"] == "decode":
        return _decode64(case, seed)
    if case["kind"] != "kv8":
        return _train64(case, seed)
    x = _cache_inputs(case, seed)
    live = torch.arange(case["T"], device=DEV)[None, :] < torch.tensor(x["new"], device=DEV)[:, None]
    return {c: _held64(x[c]) * live[:, :, None, None] for c in ("k", "v")}
