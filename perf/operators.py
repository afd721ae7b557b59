"""Operators of training and scoring on the decoder: what a call of each takes
and gives, its plain form in torch, and its 64-bit result.

* attn_fwd      attention for training: output and log-sum-exp of each row.
* attn_bwd      its backward from q, k, v, out, lse and dout.
* logprobs      log probabilities of given tokens, entropy, log-sum-exp and
                the top alternatives of each row of logits.
* logprobs_bwd  the gradient of log probabilities and entropy on the logits.
* ckpt8         an activation into its 8-bit checkpoint and back.
* swiglu8       gate and up pre-activations into 8-bit checkpoints, and from
                them what the MLP's backward reads: gate, up, silu(gate) * up.

listed() holds two sizes of each, draw() spreads over the ranges they stand
for. `own` selects the framework's entry points, otherwise run() computes the
plain form.
"""
import math

import torch

own = False

DEV = "cuda"
BF, F32, F64, I32, I64 = torch.bfloat16, torch.float32, torch.float64, torch.int32, torch.int64
HD = 128
BLOCK = 32  # columns that share an exponent in an 8-bit checkpoint
NEG = float("-inf")


# ------------------------------------------------------------------ cases
def listed():
    """Attention cases: B sequences padded to T tokens, `lens` their true
    lengths ("" = all T); fused = q, k, v are views of one projection output.
    Log-probability cases: rows of V logits, n given tokens and k
    alternatives a row; pad = columns at the row's end that are -inf."""
    return [
        # the decoder layer of this repository's benchmark: 2 x 4096 tokens, 32/8 heads
        dict(name="attn_fwd_2x4096", kind="attn_fwd", B=2, T=4096, Hq=32, Hkv=8, lens="", causal=True, fused=False),
        # a padded batch of documents out of a fused projection, one of them empty, one of a single token
        dict(name="attn_fwd_6x777_padded", kind="attn_fwd", B=6, T=777, Hq=32, Hkv=8, lens="777,700,1,513,0,64",
             causal=True, fused=True),
        # the same layer's backward
        dict(name="attn_bwd_2x4096", kind="attn_bwd", B=2, T=4096, Hq=32, Hkv=8, lens="", causal=True, fused=False),
        # a few short answers in one padded batch: latency
        dict(name="attn_bwd_4x61_padded", kind="attn_bwd", B=4, T=61, Hq=16, Hkv=4, lens="61,17,1,0", causal=True,
             fused=True),
        # a serving step of a small batch: the next token's alternatives from f32 logits
        dict(name="logprobs_7_f32_top20", kind="logprobs", rows=7, V=128256, dtype="f32", n=1, k=20, temp=0.7, pad=0),
        # scoring a batch of answers: one given token a row and a few alternatives, bf16 logits of a padded vocabulary
        dict(name="logprobs_4096_bf16_top5", kind="logprobs", rows=4096, V=128256, dtype="bf16", n=1, k=5, temp=1.0,
             pad=256),
        # the gradient of that batch's objective (a third of the rows are prompt, without gradient)
        dict(name="logprobs_bwd_4096_bf16", kind="logprobs_bwd", rows=4096, V=128256, dtype="bf16", n=1, temp=1.0,
             ent=True, pad=256),
        # several given tokens a row over an odd vocabulary, f32
        dict(name="logprobs_bwd_65_f32", kind="logprobs_bwd", rows=65, V=50257, dtype="f32", n=4, temp=0.7, ent=False,
             pad=0),
        # the residual stream of the benchmark's step (8 x 2048 tokens, hidden 4096) held for the backward
        dict(name="ckpt8_16384x4096", kind="ckpt8", rows=16384, cols=4096, dtype="bf16"),
        # ragged f32 activations: a width that no block divides
        dict(name="ckpt8_511x1409_f32", kind="ckpt8", rows=511, cols=1409, dtype="f32"),
        # the MLP's saved pre-activations: a packed batch, base 14336 and slice 1024
        dict(name="swiglu8_8192x15360", kind="swiglu8", rows=8192, cols=15360),
        # a short odd batch at the reference's default width
        dict(name="swiglu8_77x11008", kind="swiglu8", rows=77, cols=11008),
    ]


def _log_int(rng, lo, hi):
    """Log-uniform whole number in [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attn_fwd", "attn_bwd", "attn_bwd", "logprobs", "logprobs", "logprobs_bwd", "ckpt8", "swiglu8"])
    if kind in ("attn_fwd", "attn_bwd"):
        Hq, Hkv = rng.choice([(32, 8), (16, 4), (8, 8), (32, 4), (6, 2), (8, 1)])
        B = rng.randint(1, 8)
        T = _log_int(rng, 1, int((32 * 2 * 4096 ** 2 / (B * Hq)) ** 0.5) if B * Hq > 64 else 4096)
        lens = ""
        if rng.random() < 0.6:
            lens = ",".join(str(rng.randint(0, T) if rng.random() < 0.8 else T) for _ in range(B))
            if not any(int(v) for v in lens.split(",")):
                lens = ""
        return dict(kind=kind, B=B, T=T, Hq=Hq, Hkv=Hkv, lens=lens, causal=rng.random() < 0.8, fused=rng.random() < 0.5)
    if kind in ("logprobs", "logprobs_bwd"):
        dtype = rng.choice(["bf16", "bf16", "f32"])
        V = rng.choice([32000, 50257, 128256, _log_int(rng, 37, 160000)])
        rows = _log_int(rng, 1, max(1, min(8192, 4096 * 128256 * 2 // (V * (4 if dtype == "f32" else 2)))))
        pad = rng.choice([0, 0, min(256, V // 4)])
        c = dict(kind=kind, rows=rows, V=V, dtype=dtype, n=rng.choice([1, 1, 2, 8]), temp=rng.choice([1.0, 1.0, 0.7, 1.3]),
                 pad=pad)
        if kind == "logprobs":
            c["k"] = rng.choice([0, 1, 5, 20, 32])
        else:
            c["ent"] = rng.random() < 0.5
        return c
    if kind == "ckpt8":
        cols = rng.choice([2048, 4096, 14336, _log_int(rng, 5, 20000)])
        return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(16384, 16384 * 4096 // cols))), cols=cols,
                    dtype=rng.choice(["bf16", "f32"]))
    cols = rng.choice([15360, 11008, 16384, 8 * _log_int(rng, 4, 2000)])
    return dict(kind=kind, rows=_log_int(rng, 1, max(1, min(16384, 8192 * 15360 // cols))), cols=cols)


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

    def uniform(self, shape):
        return torch.rand(shape, generator=self.g, device=DEV, dtype=F32)

    def ints(self, shape, hi):
        return torch.randint(0, hi, shape, generator=self.g, device=DEV, dtype=I64)


def _attn_inputs(case, seed):
    """q of twice the keys' size: rows between flat and peaked. What lies past
    a sequence's end is finite and arbitrary."""
    d = _Draw(seed)
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    s = dict(scale=HD ** -0.5, causal=case["causal"])
    if case["fused"]:
        qkv = d.normal((B, T, Hq + 2 * Hkv, HD))
        qkv[:, :, :Hq] *= 2
        s["q"], s["k"], s["v"] = qkv[:, :, :Hq], qkv[:, :, Hq:Hq + Hkv], qkv[:, :, Hq + Hkv:]
    else:
        s["q"], s["k"], s["v"] = d.normal((B, T, Hq, HD), 2.0), d.normal((B, T, Hkv, HD)), d.normal((B, T, Hkv, HD))
    s["seq_lens"] = torch.tensor(_lens(case), dtype=I32, device=DEV) if case["lens"] else None
    if case["kind"] == "attn_bwd":
        s["dout"] = d.normal((B, T, Hq, HD))
    return s


def _logit_inputs(case, seed):
    """Logits as a language model gives them: a broad bulk and a few likely
    tokens, the given ones mostly among them; the columns of a padded
    vocabulary are -inf."""
    d = _Draw(seed)
    rows, V, n = case["rows"], case["V"], case["n"]
    real = V - case["pad"]
    x = d.normal((rows, V), 2.0, dtype=F32)
    likely = d.ints((rows, 8), real)
    x.scatter_add_(1, likely, 8.0 * d.uniform((rows, 8)))
    if case["pad"]:
        x[:, real:] = NEG
    ids = torch.where(d.uniform((rows, n)) < 0.7, likely.gather(1, d.ints((rows, n), 8)), d.ints((rows, n), real))
    s = dict(logits=x.to(BF) if case["dtype"] == "bf16" else x, ids=ids.to(I32), temp=case["temp"])
    if case["kind"] == "logprobs":
        s["k"] = case["k"]
    else:
        answer = (d.uniform((rows, 1)) > 1 / 3).float()
        answer[0] = 1.0
        s["g_logp"] = d.normal((rows, n), 1.0 / rows, dtype=F32) * answer
        s["g_ent"] = d.normal((rows,), 0.01 / rows, dtype=F32) * answer[:, 0] if case["ent"] else None
    return s


def _act_inputs(case, seed):
    """Activations with columns of very different size, as a residual stream
    has them, and rows that are zero (padding)."""
    d = _Draw(seed)
    rows, cols = case["rows"], case["cols"]

    def one(dtype):
        t = d.normal((rows, cols), dtype=F32)
        t *= torch.exp(d.normal((cols,), 1.0, dtype=F32))
        t[1:] *= (d.uniform((rows - 1, 1)) > 0.02).float()
        return t.to(dtype)

    if case["kind"] == "ckpt8":
        return dict(x=one(BF if case["dtype"] == "bf16" else F32))
    return dict(g=one(BF), u=one(BF))


def prepare(case, seed):
    kind = case["kind"]
    if kind in ("attn_fwd", "attn_bwd"):
        s = _attn_inputs(case, seed)
        if kind == "attn_bwd":
            s["out"], s["lse"] = _plain_attn_fwd(s)  # what the forward left
    elif kind in ("logprobs", "logprobs_bwd"):
        s = _logit_inputs(case, seed)
        if kind == "logprobs_bwd":
            s["lse"], s["entropy"] = _plain_row_stats(s["logits"].float() / s["temp"])[:2]
    else:
        s = _act_inputs(case, seed)
    s["kind"] = kind
    return s


# -------------------------------------------------------------------- run
def run(s):
    return (_OWN if own else _PLAIN)[s["kind"]](s)


def _own_attn_fwd(s):
    from glt_amd import ops
    out, lse = ops.attention_train(s["q"], s["k"], s["v"], causal=s["causal"], scale=s["scale"],
                                   seq_lens=s["seq_lens"])
    return dict(out=out, lse=lse)


def _own_attn_bwd(s):
    from glt_amd import ops
    dq, dk, dv = ops.attention_bwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], causal=s["causal"],
                                   scale=s["scale"], seq_lens=s["seq_lens"])
    return dict(dq=dq, dk=dk, dv=dv)


def _own_logprobs(s):
    from glt_amd import ops
    return ops.token_logprobs(s["logits"], s["ids"], top_k=s["k"], temperature=s["temp"])


def _own_logprobs_bwd(s):
    from glt_amd import ops
    return dict(grad=ops.token_logprobs_bwd(s["logits"], s["ids"], s["lse"], s["g_logp"], entropy=s["entropy"],
                                            grad_entropy=s["g_ent"], temperature=s["temp"]))


def _own_ckpt8(s):
    from glt_amd import ops
    return dict(x=ops.ckpt8_save(s["x"]).load())


def _own_swiglu8(s):
    from glt_amd import ops
    g, u, inter = ops.ckpt8_swiglu(ops.ckpt8_save(s["g"]), ops.ckpt8_save(s["u"]))
    return dict(g=g, u=u, inter=inter)


_OWN = {"attn_fwd": _own_attn_fwd, "attn_bwd": _own_attn_bwd, "logprobs": _own_logprobs,
        "logprobs_bwd": _own_logprobs_bwd, "ckpt8": _own_ckpt8, "swiglu8": _own_swiglu8}


# ------------------------------------------------------------ plain forms
def _allowed(T, seq_lens, causal):
    """[B or 1, 1, T, T] truth values: may query row t read key column s."""
    t = torch.arange(T, device=DEV)
    ok = (t[None, :] <= t[:, None]) if causal else torch.ones((T, T), dtype=torch.bool, device=DEV)
    ok = ok[None]
    if seq_lens is not None:
        live = t[None, :] < seq_lens[:, None]
        ok = ok & live[:, :, None] & live[:, None, :]
    return ok[:, None]


def _heads(t, rep=1):
    """[B, T, H, 128] of any type -> f32 [B, H * rep, T, 128]."""
    t = t.float().transpose(1, 2)
    return (t.repeat_interleave(rep, 1) if rep > 1 else t).contiguous()


def _plain_scores(s):
    rep = s["q"].shape[2] // s["k"].shape[2]
    q, k, v = _heads(s["q"]), _heads(s["k"], rep), _heads(s["v"], rep)
    z = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s["scale"])
    z.masked_fill_(~_allowed(q.shape[2], s["seq_lens"], s["causal"]), NEG)
    m = z.amax(-1, keepdim=True).clamp_(min=-1e30)  # a row without keys keeps a finite maximum
    p = z.sub_(m).exp_()
    l = p.sum(-1, keepdim=True)
    return q, k, v, p, l, m


def _plain_attn_fwd(s):
    q, k, v, p, l, m = _plain_scores(s)
    out = torch.matmul(p, v) / torch.where(l > 0, l, torch.ones_like(l))
    lse = torch.where(l > 0, m + torch.log(l), torch.full_like(l, NEG))[..., 0]
    return out.transpose(1, 2).to(BF).contiguous(), lse


def _plain_attn_bwd(s):
    q, k, v, p, l, _ = _plain_scores(s)
    B, Hq, T, _ = q.shape
    Hkv = s["k"].shape[2]
    p.div_(torch.where(l > 0, l, torch.ones_like(l)))
    do = _heads(s["dout"])
    if s["seq_lens"] is not None:
        live = torch.arange(T, device=DEV)[None, :] < s["seq_lens"][:, None]
        do = do * live[:, None, :, None]
    group = lambda t: t.view(B, Hkv, Hq // Hkv, T, HD).sum(2).transpose(1, 2).to(BF).contiguous()
    dv = group(torch.matmul(p.transpose(2, 3), do))
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    delta = (p * dp).sum(-1, keepdim=True)
    ds = dp.sub_(delta).mul_(p).mul_(s["scale"])
    del p
    dq = torch.matmul(ds, k).transpose(1, 2).to(BF).contiguous()
    return dq, group(torch.matmul(ds.transpose(2, 3), q)), dv


def _plain_row_stats(z):
    """lse, entropy, maximum and sum of each row of f32 logits; the sums in 64
    bits, where a peaked row would lose what is not its maximum."""
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    total = e.sum(-1, dtype=F64)
    t = torch.where(e > 0, e * (z - m), torch.zeros_like(e)).sum(-1, dtype=F64)
    lse = m[:, 0].double() + torch.log(total)
    return lse.float(), (torch.log(total) - t / total).float(), m, total


def _plain_logprobs(s):
    z = s["logits"].float() / s["temp"]
    lse, ent, m, total = _plain_row_stats(z)
    shift = torch.log(total)[:, None]
    r = dict(logprobs=((z.gather(1, s["ids"].long()) - m).double() - shift).float(), entropy=ent, lse=lse)
    if s["k"]:
        ids = torch.sort(s["logits"], dim=1, descending=True, stable=True)[1][:, :s["k"]]
        r["top_ids"] = ids.to(I32)
        r["top_logprobs"] = ((z.gather(1, ids) - m).double() - shift).float()
    return r


def _plain_logprobs_bwd(s):
    z = s["logits"].float() / s["temp"]
    logp = z - s["lse"][:, None]
    p = torch.exp(logp)
    g = p * -s["g_logp"].sum(-1, keepdim=True)
    if s["g_ent"] is not None:
        h = torch.where(p > 0, p * (logp + s["entropy"][:, None]), torch.zeros_like(p))
        g -= h * s["g_ent"][:, None]
    g.scatter_add_(1, s["ids"].long(), s["g_logp"])
    return dict(grad=(g / s["temp"]).to(s["logits"].dtype))


def _plain_block_step(x):
    """[rows, blocks, 32] f32 values (zero padded) and the power of two that
    is one code step of each block: the smallest for which the block's
    largest value rounds to a code of at most 127."""
    rows, cols = x.shape
    nb = -(-cols // BLOCK)
    t = torch.zeros((rows, nb * BLOCK), dtype=F32, device=x.device)
    t[:, :cols] = x
    t = t.view(rows, nb, BLOCK)
    top = t.abs().amax(-1, keepdim=True)
    e = (top.view(I32) + 0x10000) >> 23  # the exponent field once 127.5 / 64 and more have been carried up
    return t, e - 133


def _plain_codes(x):
    """The values that the 8-bit codes of x stand for, f32."""
    t, e = _plain_block_step(x)
    step = torch.exp2(e.double())  # 64 bits: a power of two that f32 may not hold
    codes = torch.round(t / step).clamp_(-127, 127)
    return (codes * step).float().reshape(x.shape[0], -1)[:, :x.shape[1]]


def _plain_ckpt8(s):
    return dict(x=_plain_codes(s["x"]).to(s["x"].dtype).contiguous())


def _plain_swiglu8(s):
    g, u = _plain_codes(s["g"]), _plain_codes(s["u"])
    return dict(g=g.to(BF), u=u.to(BF), inter=(g / (1 + torch.exp(-g)) * u).to(BF))


_PLAIN = {"attn_fwd": lambda s: dict(zip(("out", "lse"), _plain_attn_fwd(s))),
          "attn_bwd": lambda s: dict(zip(("dq", "dk", "dv"), _plain_attn_bwd(s))), "logprobs": _plain_logprobs,
          "logprobs_bwd": _plain_logprobs_bwd, "ckpt8": _plain_ckpt8, "swiglu8": _plain_swiglu8}


# ------------------------------------------------------------------- work
def work(case):
    kind = case["kind"]
    if kind in ("attn_fwd", "attn_bwd"):
        lens, Hq, Hkv = _lens(case), case["Hq"], case["Hkv"]
        pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
        live, padded = sum(lens), case["B"] * case["T"]
        if kind == "attn_fwd":
            b = 2 * HD * live * (Hq + 2 * Hkv) + padded * Hq * (2 * HD + 4)
            f = 4 * HD * Hq * pairs
        else:
            b = 2 * HD * (live * (3 * Hq + 2 * Hkv) + padded * (Hq + 2 * Hkv)) + 4 * live * Hq
            f = 10 * HD * Hq * pairs
        return {"bytes": max(b, 1), "flops": f}
    if kind in ("logprobs", "logprobs_bwd"):
        es = 4 if case["dtype"] == "f32" else 2
        rows, V = case["rows"], case["V"]
        if kind == "logprobs":
            return {"bytes": rows * (V * es + 8 * case["n"] + 8 + 8 * case["k"]), "flops": 4 * rows * V}
        return {"bytes": rows * (2 * V * es + 8 * case["n"] + 8), "flops": 4 * rows * V}
    values = case["rows"] * case["cols"]
    if kind == "ckpt8":  # the activation in and out, the codes and exponents out and in
        es = 4 if case["dtype"] == "f32" else 2
        return {"bytes": values * (2 * es + 2 + 2 / BLOCK), "flops": 4 * values}
    return {"bytes": values * (2 * 2 + 3 * 2 + 2 * (2 + 2 / BLOCK)), "flops": 12 * values}


# ------------------------------------------------------------------ exact
def _attn64(case, seed):
    s = _attn_inputs(case, seed)
    B, T, Hq, Hkv = case["B"], case["T"], case["Hq"], case["Hkv"]
    rep = Hq // Hkv
    lens = _lens(case)
    bwd = case["kind"] == "attn_bwd"
    new = lambda h, *tail: torch.zeros((B, T, h, *tail), dtype=F64, device=DEV)
    out, lse = new(Hq, HD), torch.full((B, Hq, T), NEG, dtype=F64, device=DEV)
    dq, dk, dv = (new(Hq, HD), new(Hkv, HD), new(Hkv, HD)) if bwd else (None, None, None)
    for b, n in enumerate(lens):
        future = torch.ones((n, n), dtype=torch.bool, device=DEV).triu(1) if case["causal"] else None
        for h in range(Hq if n else 0):
            q, k, v = s["q"][b, :n, h].double(), s["k"][b, :n, h // rep].double(), s["v"][b, :n, h // rep].double()
            z = q @ k.t() * s["scale"]
            if future is not None:
                z = z.masked_fill(future, NEG)
            lse[b, h, :n] = torch.logsumexp(z, -1)
            p = torch.softmax(z, -1)
            if not bwd:
                out[b, :n, h] = p @ v
                continue
            do = s["dout"][b, :n, h].double()
            dp = do @ v.t()
            ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * s["scale"]
            dv[b, :n, h // rep] += p.t() @ do
            dk[b, :n, h // rep] += ds.t() @ q
            dq[b, :n, h] = ds @ k
    return dict(dq=dq, dk=dk, dv=dv) if bwd else dict(out=out, lse=lse)


def _logprobs64(case, seed):
    s = _logit_inputs(case, seed)
    z = s["logits"].double() / case["temp"]
    ids = s["ids"].long()
    logp = torch.log_softmax(z, -1)
    if case["kind"] == "logprobs":
        p = logp.exp()
        r = dict(logprobs=logp.gather(1, ids), entropy=-torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(-1),
                 lse=torch.logsumexp(z, -1))
        if case["k"]:
            r["top_ids"] = None
            r["top_logprobs"] = logp.topk(case["k"], -1).values
        return r
    # the objective sum(g_logp * logp[ids]) + sum(g_ent * entropy), differentiated by hand
    p = logp.exp()
    d = torch.zeros_like(z).scatter_add_(1, ids, s["g_logp"].double())  # on the log probabilities
    if s["g_ent"] is not None:
        d -= s["g_ent"].double()[:, None] * torch.where(p > 0, p * (logp + 1), torch.zeros_like(p))
    return dict(grad=(d - p * d.sum(-1, keepdim=True)) / case["temp"])


def _codes64(x):
    """Values after 8 bits: one block of 32 columns a row of the table."""
    rows, cols = x.shape
    t = torch.nn.functional.pad(x.double(), (0, -cols % BLOCK)).reshape(-1, BLOCK)
    top = t.abs().amax(1)
    step = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -120))) - 6)
    step = torch.where(top / step >= 127.5, 2 * step, step)[:, None]
    return (torch.round(t / step) * step).reshape(rows, -1)[:, :cols]


def exact(case, seed):
    kind = case["kind"]
    if kind in ("attn_fwd", "attn_bwd"):
        return _attn64(case, seed)
    if kind in ("logprobs", "logprobs_bwd"):
        return _logprobs64(case, seed)
    s = _act_inputs(case, seed)
    if kind == "ckpt8":
        return dict(x=_codes64(s["x"]))
    g, u = _codes64(s["g"]), _codes64(s["u"])
    return dict(g=g, u=u, inter=g * torch.sigmoid(g) * u)
