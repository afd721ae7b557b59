"""Refusals and sizes of attention for training with a window (CPU)."""
import ctypes

import pytest

from glt_amd import _ffi as F
from test_attention_train_host import P, desc, spread


def fwd(d, window=8, sinks=2, **at):
    a = {n: v for n, v in spread(**at).items() if n in ("q", "k", "v", "out", "lse")}
    return F.load().glt_attention_window_fwd(ctypes.byref(d) if d else None, window, sinks, *a.values(), None)


def bwd(d, window=8, sinks=2, nbytes=1 << 31, **at):
    a = spread(**at)
    ws = a.pop("ws")
    return F.load().glt_attention_window_bwd(ctypes.byref(d) if d else None, window, sinks, *a.values(), ws, nbytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(window=0), 1), (dict(window=-5), 1), (dict(sinks=-1), 1), (dict(sinks=1025), 1),
    (dict(d=desc(causal=0)), 9), (dict(d=desc(head_dim=64)), 9), (dict(d=desc(n_q_heads=5)), 2),
    (dict(d=desc(q_ld=504)), 2), (dict(d=None), 1), (dict(q=None), 1), (dict(out=(1 << 32) + 8), 4),
])
def test_refusals(kw, code):
    kw = {"d": desc(), **kw}
    assert fwd(**kw) == code
    assert bwd(**kw) == code


def test_overlaps_are_refused():
    assert fwd(desc(), out=2 << 32) == 1 and fwd(desc(), lse=1 << 32) == 1
    assert bwd(desc(), dq=2 << 32) == 1 and bwd(desc(), ws=9 << 32) == 1


def test_workspace():
    lib = F.load()

    def size(d, window, sinks):
        return lib.glt_attention_window_bwd_workspace_size(ctypes.byref(d), window, sinks)
    d = desc(T=2000)
    plain = lib.glt_attention_bwd_workspace_size(ctypes.byref(d))
    assert size(d, 100, 0) == size(d, 2000, 9) == size(d, 0, 0) == plain
    # the parts of a block of 128 keys by head, its window and the queries after it 512 by 512
    one = 2 * 4 * 2 * 128 * 128 * 4
    assert size(d, 100, 1) == size(d, 100, 128) == plain + 5 * one
    assert size(d, 100, 129) == plain + 10 * one
    # 10 tiles by 10 with a window of 500, 16 by 16 with one of 950
    assert size(d, 500, 1) == plain + (1 + 3) * one and size(d, 950, 1) == plain + (1 + 1) * one
    # where key blocks fill the chip, a kv head's query heads need no parts
    big = desc(B=20, T=2000)
    assert size(big, 100, 0) < lib.glt_attention_bwd_workspace_size(ctypes.byref(big)) // 50
    assert bwd(d, 100, 1, nbytes=plain + 5 * one - 1) == 5
    assert bwd(d, 100, 1, ws=None) == 5
    assert lib.glt_attention_window_bwd_workspace_size(None, 1, 1) == 256


def test_empty_batches_need_nothing():
    for kw in (dict(B=0), dict(T=0)):
        assert fwd(desc(**kw), q=None, k=None, v=None, out=None, lse=None) == 0
        assert bwd(desc(**kw), ws=None, nbytes=0) == 0


def test_short_sequences_need_no_parts_for_sinks():
    """Where the first block's window reaches the end, its own workgroup reads every query."""
    lib = F.load()
    for T, window, more in ((128, 2, False), (192, 2, False), (193, 2, True), (192, 65, False), (400, 300, False)):
        d = desc(T=T)
        plain = lib.glt_attention_bwd_workspace_size(ctypes.byref(d))
        assert (lib.glt_attention_window_bwd_workspace_size(ctypes.byref(d), window, 4) > plain) == more, T


def test_results_over_the_lengths_are_refused():
    d = desc(seq_lens=20 << 32)
    for name in ("out", "lse"):
        assert fwd(d, **{name: 20 << 32}) == 1, name
        assert b"overlap" in F.load().glt_last_error_string()
    for name in ("dq", "dk", "dv", "ws"):
        assert bwd(d, **{name: 20 << 32}) == 1, name
        assert b"overlap" in F.load().glt_last_error_string()


@pytest.mark.parametrize("window,sinks,taken", [(40, 1025, True), (2 ** 31 - 1, 2 ** 31 - 1, True), (39, 1024, True),
                                                (39, 1025, False), (40, -1, False)])
def test_any_sinks_where_the_window_hides_nothing(window, sinks, taken):
    """40 tokens. (4: taken so far, and the operand's alignment refused.)"""
    assert fwd(desc(), window, sinks, out=(1 << 32) + 8) == (4 if taken else 1)
    assert bwd(desc(), window, sinks, out=(1 << 32) + 8) == (4 if taken else 1)
