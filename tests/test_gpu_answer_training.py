"""The operators together as a training step on answers runs them: attention
that keeps its log-sum-exp, the grafted MLP saved in 8 bits, the LM head, the
log probabilities of a padded batch's tokens with an entropy term, and the
gradients back through all of it, against the same chain differentiated in 64
bits.

Tolerance: some dozen roundings to bf16 on a path (each below 2^-9 in the
2-norm, 2.4 % if all add outright) and the 8-bit pre-activations (0.83 % each
in the 2-norm for normal values, through silu' and silu'' of size 1 at most):
5 % of a gradient's 2-norm."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

BF, F32, F64 = torch.bfloat16, torch.float32, torch.float64
EPS = 1e-5


def test_step_on_answers(dev):
    from glt_amd import ops
    B, T, Hq, Hkv, hd, I, S, V = 3, 72, 2, 1, 128, 320, 64, 1000
    D, N, M = Hq * hd, I + S, B * T
    lens = (72, 40, 5)
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    n = lambda *s, std=1.0, dt=BF: torch.empty(s, device="cuda").normal_(0, std, generator=g).to(dt)
    q, k, v = n(B, T, Hq, hd), n(B, T, Hkv, hd), n(B, T, Hkv, hd)
    wn, head = 1 + n(D, std=0.1), n(V, D, std=0.1)
    base = ops.BaseMLP(n(I, D, std=0.08), n(I, D, std=0.08), n(D, I, std=0.08))
    masters = [n(S, D, std=0.08, dt=F32) for _ in range(3)]
    sl = ops.GraftSlice(I, S, 0, D, *masters).pack()
    ids = torch.randint(0, V, (M, 1), generator=g, device="cuda").to(torch.int32)
    live = torch.arange(T, device="cuda")[None] < torch.tensor(lens, device="cuda")[:, None]
    ids[~live.reshape(-1)] = -1                                  # padding has no token
    seq_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    count = sum(lens)
    g_logp = torch.full((M, 1), -1.0 / count, device="cuda")     # the mean negative log likelihood
    g_ent = torch.where(live.reshape(-1), 0.1 / count, 0.0).float()

    # forward
    out, lse = ops.attention_train(q, k, v, seq_lens=seq_lens)
    x_mid = out.view(M, D)
    xn, var = ops.rms_norm(x_mid, wn, EPS)
    y, gate, up, _ = ops.mlp_forward(base, [sl], xn, N)
    g8, u8 = ops.ckpt8_save(gate), ops.ckpt8_save(up)
    del gate, up
    logits = ops.lm_head_fwd(y, head)
    r = ops.token_logprobs(logits, ids, top_k=4)
    # backward
    grad = ops.token_logprobs_bwd(logits, ids, r["lse"], g_logp, r["entropy"], g_ent, grad=logits)
    dy = ops.lm_head_bwd(grad, head)
    _, grads, d_mid = ops.mlp_backward(base, [sl], xn, dy, N, g8, u8, norm=(x_mid, wn, var, EPS))
    dq, dk, dv = ops.attention_bwd(q, k, v, out, lse, d_mid.to(BF).view(B, T, Hq, hd), seq_lens=seq_lens)
    torch.cuda.synchronize()

    # the same in 64 bits
    leaf = lambda t: t.detach().cpu().double().requires_grad_()
    Q, K, Vv, W = leaf(q), leaf(k), leaf(v), [leaf(m.to(BF)) for m in masters]
    okm = live.cpu()
    outs = []
    for b in range(B):
        s = torch.einsum("thd,sgd->hts", Q[b], K[b]) * hd ** -0.5
        t = torch.arange(T)
        s = s.masked_fill((t[None] > t[:, None])[None] | ~okm[b][None, None], -math.inf)
        p = torch.softmax(s, -1)
        o = torch.einsum("hts,sd->thd", p, Vv[b][:, 0])
        outs.append(torch.where(okm[b][:, None, None], o, torch.zeros_like(o)))
    x = torch.stack(outs).view(M, D)
    h = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * wn.cpu().double()
    G = torch.cat([base.gate.cpu().double(), W[0]])
    U = torch.cat([base.up.cpu().double(), W[1]])
    Dn = torch.cat([base.down.cpu().double().t(), W[2]])
    z = (torch.nn.functional.silu(h @ G.t()) * (h @ U.t())) @ Dn @ head.cpu().double().t()
    logp = torch.log_softmax(z, -1)
    rows = okm.reshape(-1)
    chosen = logp[rows].gather(1, ids.cpu().long()[rows])
    ent = -(logp[rows].exp() * logp[rows]).sum(-1)
    loss = (-chosen.sum() + 0.1 * ent.sum()) / count
    loss.backward()

    ours = (float(-r["logprobs"].double().sum()) + 0.1 * float(r["entropy"].double()[live.reshape(-1)].sum())) / count
    loss = float(loss.detach())
    assert abs(ours - loss) < 0.01 * abs(loss)
    for name, got, want in [("dq", dq, Q.grad), ("dk", dk, K.grad), ("dv", dv, Vv.grad)] + [
            (f"graft {p}", grads[0][p], W[p].grad) for p in range(3)]:
        a, b = got.cpu().double(), want
        assert float((a - b).norm()) <= 0.05 * float(b.norm()), (name, float((a - b).norm() / b.norm()))
    assert bool((r["top_logprobs"][:, 0] >= r["logprobs"][:, 0])[rows.cuda()].all())
    for b, m in enumerate(lens):
        assert not dq[b, m:].any() and not dk[b, m:].any() and not dv[b, m:].any()
