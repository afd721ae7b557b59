"""Refusals and sizes of the 8-bit cache's entry points (CPU: every check runs
before any GPU call)."""
import ctypes

import pytest

from glt_amd import _ffi as F

P = 1 << 40  # an aligned address that nothing reads; operands lie 2^34 apart
CACHE = dict(data=P, n_pages=100, n_kv_heads=2, head_dim=128)
SEQS = dict(B=4, T=3, pages=P + 64, pages_ld=9, n_table=9, lens=P + 64, new_lens=None)
ATTN = dict(n_q_heads=8, scale=0.1, window=0, sinks=0, n_groups=0, prefix_pages=None, prefix_ld=0, n_prefix_table=0,
            prefix_lens=None)
PREFIX = dict(n_groups=2, prefix_pages=P + 64, prefix_ld=5, n_prefix_table=5, prefix_lens=P + 64)


def at(i):
    return P + (i << 34)


def make(cls, base, kw):
    d = dict(base)
    d.update({k: v for k, v in kw.items() if k in base})
    return cls(**d)


def descs(kw):
    c, s, d = make(F.Kv8Cache, CACHE, kw), make(F.Kv8Seqs, SEQS, kw), make(F.Kv8Attn, ATTN, kw)
    return ctypes.byref(c), ctypes.byref(s), ctypes.byref(d)


def tokens(fn, kw=(), k=at(1), v=at(2), k_ld=256, v_ld=256):
    c, s, _ = descs(dict(kw))
    return getattr(F.load(), fn)(c, s, k, k_ld, v, v_ld, None)


def attn(kw=(), q=at(1), out=at(2), lse=at(3), ws=at(4), nbytes=1 << 33, q_ld=1024, o_ld=1024):
    c, s, d = descs(dict(kw))
    return F.load().glt_kv8_attention(c, s, d, q, q_ld, out, o_ld, lse, ws, nbytes, None)


@pytest.mark.parametrize("kw,code", [
    (dict(head_dim=64), 9),
    (dict(n_pages=0), 2),
    (dict(n_pages=-1), 2),
    (dict(n_pages=1 << 31), 2),
    (dict(n_kv_heads=0), 2),
    (dict(n_kv_heads=5000), 2),
    (dict(B=-1), 2),
    (dict(B=8193), 2),
    (dict(T=-1), 2),
    (dict(T=(1 << 24) + 1), 2),
    (dict(n_table=-1), 2),
    (dict(n_table=(1 << 23) + 1, pages_ld=1 << 24), 2),  # more tokens than an int32 counts
    (dict(pages_ld=8), 2),
    (dict(data=None), 1),
    (dict(pages=None), 1),
    (dict(lens=None), 1),
    (dict(data=P + 8), 4),
    (dict(pages=P + 2), 4),
    (dict(lens=P + 1), 4),
    (dict(new_lens=P + 2), 4),
])
def test_cache_and_table_refusals(kw, code):
    assert tokens("glt_kv8_write", kw) == code
    assert tokens("glt_kv8_read", kw) == code
    assert attn(kw) == code


@pytest.mark.parametrize("fn", ["glt_kv8_write", "glt_kv8_read"])
def test_token_refusals(fn):
    for kw, code in ((dict(k=None), 1), (dict(v=None), 1), (dict(k=at(1) + 8), 4), (dict(v=at(2) + 2), 4),
                     (dict(k_ld=248), 2), (dict(v_ld=260), 2), (dict(k_ld=1 << 31), 2), (dict(v_ld=-256), 2),
                     (dict(k=P + 4096), 1), (dict(v=P - 16), 1)):  # over the cache
        assert tokens(fn, **kw) == code, kw
    assert F.load()[fn](None, None, None, 0, None, 0, None) == 1
    if fn == "glt_kv8_read":
        assert tokens(fn, v=at(1) + 512 * 3) == 1  # over each other


@pytest.mark.parametrize("kw,code", [
    (dict(n_q_heads=0), 2),
    (dict(n_q_heads=7), 2),
    (dict(scale=0.0), 1),
    (dict(scale=float("inf")), 1),
    (dict(scale=float("nan")), 1),
    (dict(window=-1), 1),
    (dict(sinks=-1), 1),
    (dict(n_groups=-1), 2),
    (dict(PREFIX, n_groups=3), 2),           # 4 sequences
    (dict(PREFIX, prefix_ld=4), 2),
    (dict(PREFIX, n_prefix_table=-1), 2),
    (dict(PREFIX, prefix_lens=None), 1),
    (dict(PREFIX, prefix_pages=None), 1),
    (dict(PREFIX, prefix_lens=P + 2), 4),
    (dict(B=8192, T=1 << 12), 2),            # more rows than a launch has
    (dict(n_q_heads=2 << 20), 2),
])
def test_attention_refusals(kw, code):
    assert attn(kw) == code


def test_attention_pointer_and_workspace_refusals():
    for n in ("q", "out", "lse"):
        assert attn(**{n: None}) == 1
    for n, v in (("q", at(1) + 8), ("out", at(2) + 8), ("lse", at(3) + 2)):
        assert attn(**{n: v}) == 4
    for kw in (dict(q_ld=1016), dict(o_ld=1028), dict(q_ld=1 << 31)):
        assert attn(**kw) == 2
    kw = dict(n_table=40, pages_ld=40)
    c, s, d = descs(kw)
    need = F.load().glt_kv8_attention_workspace_size(c, s, d)
    assert attn(kw, ws=None) == 5 and attn(kw, nbytes=need - 1) == 5 and attn(kw, ws=at(4) + 16) == 5
    lib = F.load()
    assert lib.glt_kv8_attention(None, s, d, P, 1024, P, 1024, P, P, 1 << 30, None) == 1
    assert lib.glt_kv8_attention(c, None, d, P, 1024, P, 1024, P, P, 1 << 30, None) == 1
    assert lib.glt_kv8_attention(c, s, None, P, 1024, P, 1024, P, P, 1 << 30, None) == 1


@pytest.mark.parametrize("kw", [
    dict(out=at(1)), dict(out=at(1) + 2048 * 11), dict(lse=at(1) + 4), dict(lse=at(2)), dict(ws=at(1) + 256),
    dict(ws=at(2)), dict(out=P), dict(lse=P + 1024), dict(ws=P + 256), dict(ws=at(3)),
])
def test_overlaps_are_refused(kw):
    assert attn(dict(n_table=40, pages_ld=40), **kw) == 1
    assert b"overlap" in F.load().glt_last_error_string()


def test_empty_calls_need_nothing():
    for kw in (dict(B=0, data=None, lens=None, pages=None), dict(T=0, data=None, lens=None, pages=None)):
        assert tokens("glt_kv8_write", kw, k=None, v=None) == 0
        assert tokens("glt_kv8_read", kw, k=None, v=None) == 0
        assert attn(kw, q=None, out=None, lse=None, ws=None, nbytes=0) == 0


def test_sizes():
    lib = F.load()
    assert lib.glt_kv8_size(10, 8, 128) == 10 * 8 * 64 * 260
    assert lib.glt_kv8_size(0, 8, 128) == 0 and lib.glt_kv8_size(10, 8, 64) == 0
    assert lib.glt_kv8_attention_workspace_size(None, None, None) == 0

    def ws(**kw):
        return lib.glt_kv8_attention_workspace_size(*descs(kw))
    # the pieces that a wavefront of the chip begins and goes on with, whatever the table's width (an output, a
    # maximum and a sum of each row), and the sequences' tiles
    wide = dict(n_table=100000, pages_ld=100000)
    assert ws(**wide) <= 2 * 256 * 12 * 12 * (512 + 8) + 4 * 5 + 1024
    assert ws(T=500, **wide) <= 2 * 256 * 256 * (512 + 8) + 4 * 5 + 1024
    # a few pages a sequence, in a table or a window: one launch, nothing between
    assert ws(n_table=24, pages_ld=24) == ws(window=1400, **wide) == 0
    assert ws(n_table=25, pages_ld=25) > 0 and ws(B=200, n_table=32, pages_ld=32) == 0
    assert ws(**PREFIX) > ws()


@pytest.mark.parametrize("fn", ["glt_kv8_write", "glt_kv8_read"])
@pytest.mark.parametrize("kw", [
    dict(B=8192, T=1, n_kv_heads=2048), dict(B=8192, T=66, n_kv_heads=1024), dict(B=64, T=1 << 24, n_kv_heads=2),
    dict(B=8192, T=1 << 24, n_kv_heads=4096),
])
def test_more_workgroups_than_a_launch_has_are_refused(fn, kw):
    """256 threads each, of less than 2^32 in all; pages of 64 tokens from any place of the first."""
    heads = 128 * kw["n_kv_heads"]
    assert tokens(fn, kw, k_ld=heads, v_ld=heads) == 2
    assert b"B=%d T=%d" % (kw["B"], kw["T"]) in F.load().glt_last_error_string()


# tables and lengths apart from the cache and each other
APART = dict(pages=at(5), lens=at(6), new_lens=at(7), n_table=40, pages_ld=50)
IN_TABLES = [at(5), at(5) + 4 * (3 * 50 + 38), at(6), at(7) - 368]


@pytest.mark.parametrize("where", IN_TABLES)
def test_results_in_tables_or_lengths_are_refused(where):
    """At their start, in the table's last two pages, and from before the new lengths on."""
    for n in ("out", "lse", "ws"):
        assert attn(APART, **{n: where & ~255 if n == "ws" else where}) == 1, n
        assert b"lengths" in F.load().glt_last_error_string()
    for n in ("k", "v"):
        assert tokens("glt_kv8_read", APART, **{n: where}) == 1, n
        assert b"lengths" in F.load().glt_last_error_string()
    assert tokens("glt_kv8_write", dict(APART, data=where)) == 1
    assert b"lengths" in F.load().glt_last_error_string()


def test_results_in_a_prefix_are_refused():
    kw = dict(APART, n_groups=2, prefix_pages=at(8), prefix_ld=64, n_prefix_table=60, prefix_lens=at(9))
    for where in (at(8), at(8) + 4 * 64, at(9)):
        for n in ("out", "lse", "ws"):
            assert attn(kw, **{n: where}) == 1, n
            assert b"prefix" in F.load().glt_last_error_string()


@pytest.mark.parametrize("T", [1, 6, 100])
def test_sequences_without_a_table_need_no_workspace(T):
    """They hold no tokens, so their prefix is read by no row."""
    kw = dict(PREFIX, T=T, pages=None, pages_ld=0, n_table=0)
    assert F.load().glt_kv8_attention_workspace_size(*descs(kw)) == 0
    kw["n_table"] = kw["pages_ld"] = 1
    assert F.load().glt_kv8_attention_workspace_size(*descs(kw)) > 0


@pytest.mark.parametrize("n_pages,heads", [(1 << 31, 1), ((1 << 52) + 1, 16), (1 << 62, 8), (-1, 8), (10, 4097), (10, -1)])
def test_no_size_for_caches_that_no_call_serves(n_pages, heads):
    """Their bytes may pass 64 bits: 2^52 + 1 pages of 16 heads came to 266240."""
    assert F.load().glt_kv8_size(n_pages, heads, 128) == 0
    assert F.load().glt_kv8_size((1 << 31) - 1, 4096, 128) == ((1 << 31) - 1) * 4096 * 64 * 260
