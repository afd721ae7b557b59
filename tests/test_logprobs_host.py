"""Refusals and sizes of the log-probability entry points (CPU: every check
runs before any GPU call)."""
import pytest

from glt_amd import _ffi as F

P = 4096


def fwd(logits=P, dtype=0, ld=100, rows=3, V=100, temp=1.0, ids=P, n=1, k=2, lp=P, ent=P, lse=P, ti=P, tl=P, ws=P,
        nb=1 << 40):
    return F.load().glt_token_logprobs(logits, dtype, ld, rows, V, temp, ids, n, k, lp, ent, lse, ti, tl, ws, nb, None)


def bwd(logits=P, dtype=0, ld=100, rows=3, V=100, temp=1.0, ids=P, n=1, gl=P, lse=P, ent=P, ge=P, grad=2 * P, ldg=100):
    return F.load().glt_token_logprobs_bwd(logits, dtype, ld, rows, V, temp, ids, n, gl, lse, ent, ge, grad, ldg, None)


@pytest.mark.parametrize("kw,code", [
    (dict(dtype=2), 3), (dict(dtype=-1), 3),
    (dict(rows=-1), 2), (dict(V=0), 2), (dict(ld=99), 2),
    (dict(V=(1 << 20) + 1, ld=1 << 21), 9),
    (dict(n=-1), 9), (dict(n=65), 9),
    (dict(temp=0.0), 1), (dict(temp=-1.0), 1), (dict(temp=float("nan")), 1), (dict(temp=float("inf")), 1),
    (dict(rows=2 ** 31 - 1, V=20000, ld=20000, ldg=20000), 2),   # more workgroups than a launch has
    (dict(rows=1 << 24), 2),
    (dict(logits=None), 1), (dict(ids=None), 1),
    (dict(logits=P + 1), 4), (dict(logits=P + 2, dtype=1), 4), (dict(ids=P + 2), 4), (dict(lse=P + 1), 4),
])
def test_refusals_of_both(kw, code):
    assert bwd(**kw) == code
    kw.pop("ldg", None)
    assert fwd(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(k=-1), 9), (dict(k=65), 9), (dict(k=8, V=7, ld=7), 9),
    (dict(lp=None), 1), (dict(ti=None), 1), (dict(tl=None), 1),
    (dict(ti=P + 2), 4), (dict(ent=P + 2), 4),
    (dict(ws=None), 5), (dict(ws=P + 16), 5), (dict(nb=255), 5),
])
def test_refusals_of_the_forward(kw, code):
    assert fwd(**kw) == code


@pytest.mark.parametrize("kw,code", [
    (dict(ldg=99), 2), (dict(grad=P, ldg=101), 2),               # in place with another stride
    (dict(grad=None), 1), (dict(lse=None), 1), (dict(gl=None), 1), (dict(ent=None), 1),
    (dict(grad=2 * P + 1), 4), (dict(ge=P + 2), 4),
])
def test_refusals_of_the_backward(kw, code):
    assert bwd(**kw) == code


def test_no_rows_need_nothing():
    assert fwd(rows=0, logits=None, ids=None, lp=None, ti=None, tl=None, ws=None, nb=0) == 0
    assert bwd(rows=0, logits=None, ids=None, gl=None, lse=None, grad=None) == 0


def test_workspace_sizes():
    lib = F.load()
    assert lib.glt_token_logprobs_workspace_size(0, 100, 0, 5) == 256
    last = 0
    for rows in (1, 2, 7, 4096):
        n = lib.glt_token_logprobs_workspace_size(rows, 128256, 0, 20)
        # eight pieces of four 16-byte parts and 20 keys of 8 bytes
        assert n >= rows * 8 * (4 * 16 + 20 * 8) and n > last and n % 256 == 0
        last = n


@pytest.mark.parametrize("kw", [
    dict(grad=P + 2), dict(grad=P + 200), dict(grad=P - 200),            # a step or a row off, the same stride
    dict(grad=P + 600 - 2), dict(grad=P + 400, ldg=164),                 # the last logit; rows of another stride
    dict(ld=200, ldg=200, grad=P + 198), dict(ld=200, ldg=200, grad=P - 200 + 2),
    dict(lse=3 * P, grad=3 * P), dict(ent=3 * P, grad=3 * P + 8), dict(ge=3 * P, grad=3 * P - 598),
    dict(ids=3 * P, grad=3 * P + 10), dict(gl=3 * P, grad=3 * P - 200),
])
def test_a_gradient_partly_over_an_input_is_refused(kw):
    """Workgroups write their pieces while others read."""
    far = dict(logits=P, ids=16 * P, gl=17 * P, lse=18 * P, ent=19 * P, ge=20 * P)
    far.update(kw)
    assert bwd(**far) == 1
    assert b"overlap" in F.load().glt_last_error_string()
