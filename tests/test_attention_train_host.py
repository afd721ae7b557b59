"""Refusals and sizes of the attention training entry points (CPU: every check
runs before any GPU call)."""
import ctypes

import pytest

from glt_amd import _ffi as F

P = 4096  # an aligned address that nothing reads


def desc(**kw):
    d = dict(B=2, T=40, n_q_heads=4, n_kv_heads=2, head_dim=128, scale=0.1, causal=1, q_ld=512, k_ld=256, v_ld=256,
             o_ld=512, seq_lens=None)
    d.update(kw)
    return F.AttnDesc(**d)


def fwd(d, q=P, k=P, v=P, out=P, lse=P):
    return F.load().glt_attention_train_fwd(ctypes.byref(d) if d else None, q, k, v, out, lse, None)


def bwd(d, ws=P, nbytes=1 << 40, **kw):
    a = dict(q=P, k=P, v=P, out=P, lse=P, dout=P, dq=P, dk=P, dv=P)
    a.update(kw)
    return F.load().glt_attention_bwd(ctypes.byref(d) if d else None, *a.values(), ws, nbytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(n_q_heads=5), 2),             # not a multiple of the kv heads
    (dict(n_kv_heads=0), 2),
    (dict(B=-1), 2),
    (dict(T=-1), 2),
    (dict(head_dim=64), 9),
    (dict(scale=0.0), 1),
    (dict(scale=-0.1), 1),
    (dict(scale=float("inf")), 1),
    (dict(scale=float("nan")), 1),
    (dict(q_ld=504), 2),                # fewer columns than the heads have
    (dict(k_ld=260), 2),                # no multiple of 8
    (dict(v_ld=0), 2),
    (dict(o_ld=-512), 2),
    (dict(k_ld=1 << 40), 2),
    (dict(T=1 << 22), 2),               # 4M rows of 512 columns pass 2 GiB
    (dict(B=1 << 30, n_q_heads=4), 2),  # more workgroups than a launch has
    (dict(B=1 << 22, T=1), 2),
    (dict(B=1 << 15, T=1 << 12), 2),    # more kv rows than the sum of parts can launch for
])
def test_descriptor_refusals(kw, code):
    assert fwd(desc(**kw)) == code
    assert bwd(desc(**kw)) == code


def test_pointer_and_workspace_refusals():
    assert fwd(None) == 1 and bwd(None) == 1
    for name in ("q", "k", "v", "out", "lse"):
        assert fwd(desc(), **{name: None}) == 1
    for name in ("q", "k", "v", "out"):
        assert fwd(desc(), **{name: P + 8}) == 4
    assert fwd(desc(), lse=P + 2) == 4
    assert fwd(desc(seq_lens=P + 1)) == 4
    for name in ("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv"):
        assert bwd(desc(), **{name: None}) == 1
        assert bwd(desc(), **{name: P + 2}) == 4
    need = F.load().glt_attention_bwd_workspace_size(ctypes.byref(desc()))
    assert bwd(desc(), ws=None) == 5
    assert bwd(desc(), nbytes=need - 1) == 5
    assert bwd(desc(), ws=P + 16) == 5


def test_empty_batches_need_nothing():
    for kw in (dict(B=0), dict(T=0)):
        assert fwd(desc(**kw), q=None, k=None, v=None, out=None, lse=None) == 0
        assert bwd(desc(**kw), ws=None, nbytes=0) == 0
    assert F.load().glt_attention_bwd_workspace_size(None) == 256


def test_workspace_holds_row_sums_and_partials():
    """lse and D of every row, and f32 dk and dv by query head where heads share a kv head."""
    lib = F.load()
    for B, T, Hq, Hkv in ((1, 1, 8, 1), (2, 61, 16, 4), (3, 777, 32, 8), (2, 4096, 32, 8), (1, 300, 6, 2)):
        d = desc(B=B, T=T, n_q_heads=Hq, n_kv_heads=Hkv, q_ld=Hq * 128, o_ld=Hq * 128, k_ld=Hkv * 128, v_ld=Hkv * 128)
        n = lib.glt_attention_bwd_workspace_size(ctypes.byref(d))
        assert n % 256 == 0 and n >= 8 * B * T * Hq
        assert n <= 8 * B * T * Hq + 256 + 8 * B * T * Hq * 128


def spread(**at):
    """Operands far apart, but for those given."""
    a = {n: (i + 1) << 32 for i, n in enumerate(("q", "k", "v", "out", "lse", "dout", "dq", "dk", "dv", "ws"))}
    a.update(at)
    return a


@pytest.mark.parametrize("at", [
    dict(dq=1 << 32), dict(dk=2 << 32), dict(dv=3 << 32),       # over what it is the gradient of
    dict(dv=1 << 32), dict(dq=6 << 32), dict(dk=4 << 32),
    dict(dq=(1 << 32) + 79 * 1024 + 512),                       # the last row's second half
    dict(dq=(1 << 32) - 79 * 1024 - 512),                       # the other way round
    dict(dk=(1 << 32) + 1024 * 30 + 512 - 16),                  # rows of another stride
    dict(dv=(5 << 32) + 16), dict(dk=7 << 32), dict(dv=8 << 32),
    dict(ws=(1 << 32) + 256), dict(ws=9 << 32), dict(ws=5 << 32),
])
def test_overlapping_gradients_are_refused(at):
    """The queries' gradient is written before the keys' kernel reads the
    queries: nothing that a call writes may lie over what it reads."""
    a = spread(**at)
    ws = a.pop("ws")
    assert bwd(desc(), ws=ws, **a) == 1
    assert b"overlap" in F.load().glt_last_error_string()


@pytest.mark.parametrize("at", [
    dict(out=2 << 32), dict(out=3 << 32), dict(out=(1 << 32) + 16), dict(out=(1 << 32) - 1024), dict(lse=1 << 32),
    dict(lse=2 << 32), dict(lse=3 << 32), dict(lse=(4 << 32) + 8),
])
def test_overlapping_outputs_are_refused(at):
    a = {n: v for n, v in spread(**at).items() if n in ("q", "k", "v", "out", "lse")}
    assert fwd(desc(), **a) == 1
    assert b"overlap" in F.load().glt_last_error_string()


def test_an_output_over_the_queries_has_their_stride():
    a = {n: v for n, v in spread(out=1 << 32).items() if n in ("q", "k", "v", "out", "lse")}
    assert fwd(desc(o_ld=520), **a) == 1
