"""Refusals and sizes of the 8-bit checkpoints, and of the MLP backward that
reads them (CPU: every check runs before any GPU call)."""
import ctypes

import pytest

from glt_amd import _ffi as F

P = 4096


def save(x=P, dtype=0, ld=64, rows=3, cols=64, ck=P):
    return F.load().glt_ckpt8_save(x, dtype, ld, rows, cols, ck, None)


def load(ck=P, rows=3, cols=64, x=P, dtype=0, ld=64):
    return F.load().glt_ckpt8_load(ck, rows, cols, x, dtype, ld, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), 3), (dict(rows=-1), 2), (dict(cols=0), 2), (dict(cols=-3), 2), (dict(ld=63), 2),
    (dict(rows=1 << 31), 2), (dict(rows=1 << 28, cols=256, ld=256), 2),  # parts of 8 columns past 32 bits
    (dict(x=None), 1), (dict(ck=None), 1),
    (dict(ck=P + 16), 4), (dict(x=P + 1), 4), (dict(x=P + 2, dtype=1), 4),
])
def test_refusals(kw, code):
    assert save(**kw) == code
    assert load(**kw) == code


def test_swiglu_refusals():
    f = F.load().glt_ckpt8_swiglu
    assert f(None, P, 3, 64, P, P, P, None) == 1
    assert f(P, P + 8, 3, 64, P, P, P, None) == 4
    assert f(P, P, 3, 64, P + 1, P, P, None) == 4
    assert f(P, P, -1, 64, P, P, P, None) == 2
    assert f(P, P, 3, 0, P, P, P, None) == 2
    assert f(P, P, 3, 64, None, None, None, None) == 0   # nothing wanted
    assert f(None, None, 0, 64, None, None, None, None) == 0


def test_no_rows_and_sizes():
    assert save(rows=0, x=None, ck=None) == 0 and load(rows=0, x=None, ck=None) == 0
    size = F.load().glt_ckpt8_size
    assert size(0, 64) == 256
    for rows, cols in ((1, 1), (3, 31), (3, 33), (511, 1409), (16384, 15360)):
        blocks = rows * -(-cols // 32)
        codes = -(-blocks * 32 // 256) * 256
        assert size(rows, cols) == codes + -(-blocks // 256) * 256


def test_mlp_backward_refusals():
    lib = F.load()

    def bwd(flags, dtype=F.DTYPE_BF16, gate=P, up=P):
        d = F.MlpDesc(16, 64, 64, 64, dtype, flags, 0, None, None)
        w = F.BaseWeights(P, P, P, P)
        return lib.glt_mlp_bwd(ctypes.byref(d), ctypes.byref(w), P, P, gate, up, None, None, None, None, 0, None)

    assert bwd(F.MLP_SAVED_CKPT8 | F.MLP_RECOMPUTE) == 1
    assert bwd(F.MLP_SAVED_CKPT8, dtype=F.DTYPE_F32) == 3
    assert bwd(F.MLP_SAVED_CKPT8, gate=P + 16) == 4
    assert bwd(F.MLP_SAVED_CKPT8, up=None) == 1
    assert bwd(F.MLP_SAVED_CKPT8) == 5                   # inter is not needed, the workspace is
    assert bwd(0) == 1                                   # without the flag inter is
    d = F.MlpDesc(16, 64, 64, 64, F.DTYPE_BF16, F.MLP_SAVED_CKPT8, 0, None, None)
    d0 = F.MlpDesc(16, 64, 64, 64, F.DTYPE_BF16, 0, 0, None, None)
    extra = lib.glt_mlp_bwd_workspace_size(ctypes.byref(d)) - lib.glt_mlp_bwd_workspace_size(ctypes.byref(d0))
    assert extra == 3 * 16 * 64 * 2                      # gate, up, inter restored
