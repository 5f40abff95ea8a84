"""Calls on the paged cache and the sampler that are refused before anything is launched; the plain restatements
that the GPU tests compare with. No GPU needed."""
import ctypes as C

import numpy as np
import pytest

import kvref
import lancius_b200 as L

NULL, SHAPE, OP, DTYPE, OVERFLOW = -2, -3, -4, -5, -9
BUF = (C.c_uint8 * 4096)()
AT = (C.addressof(BUF) + 63) // 64 * 64   # never dereferenced: these calls fail their checks, or have no work


def pages(**kw):
    d = dict(k_codes=AT, v_codes=AT, k_scales=AT, v_scales=AT, n_pages=4, page_size=16, n_heads=2, head_dim=64,
             k_unit=1.0, v_unit=1.0)
    d.update(kw)
    return L.KvPages(*d.values())


def batch(**kw):
    d = dict(page_table=AT, table_width=2, seq_len=AT, token_start=None, n_seqs=3, n_tokens=3, max_seq_len=0, max_new=0)
    d.update(kw)
    return L.KvBatch(*d.values())


def append(p, b, q_out=AT, q=AT, q_ld=256, hq=4, k=AT, k_ld=128, v=AT, v_ld=128, base=1e4):
    return L.load().lcu_kv_append_paged(p, b, q_out, q, q_ld, hq, k, k_ld, v, v_ld, base, None)


BAD_PAGES = [(dict(k_codes=None), NULL), (dict(v_scales=None), NULL), (dict(k_codes=AT + 8), DTYPE),
             (dict(v_scales=AT + 4), DTYPE), (dict(head_dim=80), OP), (dict(head_dim=512), OP), (dict(page_size=0), SHAPE),
             (dict(page_size=24), SHAPE), (dict(page_size=8192), SHAPE), (dict(n_heads=0), SHAPE), (dict(n_heads=1 << 20), SHAPE),
             (dict(n_pages=1 << 40), SHAPE), (dict(k_unit=0.0), SHAPE), (dict(v_unit=float("nan")), SHAPE),
             (dict(v_unit=float("inf")), SHAPE)]
BAD_BATCH = [(dict(seq_len=None), NULL), (dict(page_table=None), NULL), (dict(n_seqs=70000), SHAPE),
             (dict(n_tokens=1 << 31), SHAPE), (dict(table_width=1 << 40), SHAPE), (dict(n_tokens=2), SHAPE)]


@pytest.mark.parametrize("kw,code", BAD_PAGES)
def test_pages_refused(kw, code):
    lib, p, b = L.load(), pages(**kw), batch()
    assert append(p, b) == code
    assert lib.lancius_get_error() == code
    assert lib.lcu_kv_read_paged(AT, AT, p, b, None) == code
    assert lib.lcu_attention_paged(AT, AT, 256, 4, p, b, AT, 1 << 30, None) == code
    assert lib.lcu_attention_paged_workspace(p, b, 4) == 0


@pytest.mark.parametrize("kw,code", BAD_BATCH)
def test_batch_refused(kw, code):
    lib, p, b = L.load(), pages(), batch(**kw)
    assert append(p, b) == code
    assert lib.lcu_kv_read_paged(AT, AT, p, b, None) == code
    assert lib.lcu_attention_paged(AT, AT, 256, 4, p, b, AT, 1 << 30, None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(k=None), NULL), (dict(q=None), NULL), (dict(q_out=None), NULL), (dict(q_ld=255), SHAPE), (dict(k_ld=127), SHAPE),
    (dict(v_ld=64), SHAPE), (dict(base=float("nan")), SHAPE), (dict(base=float("inf")), SHAPE),
    (dict(q_ld=512), SHAPE)])   # q_out = q with rows apart
def test_append_refused(kw, code):
    assert append(pages(), batch(), **kw) == code


def test_attention_refused():
    lib, p, b = L.load(), pages(), batch()
    assert lib.lcu_attention_paged(None, AT, 256, 4, p, b, AT, 1 << 30, None) == NULL
    assert lib.lcu_attention_paged(AT, None, 256, 4, p, b, AT, 1 << 30, None) == NULL
    assert lib.lcu_attention_paged(AT, AT, 128, 4, p, b, AT, 1 << 30, None) == SHAPE
    assert lib.lcu_attention_paged(AT, AT, 256, 3, p, b, AT, 1 << 30, None) == SHAPE
    assert lib.lcu_attention_paged(AT, AT, 256, 4, None, b, AT, 1 << 30, None) == NULL
    assert lib.lcu_attention_paged(AT, AT, 256, 4, p, None, AT, 1 << 30, None) == NULL
    many = batch(token_start=AT, n_tokens=70000)   # max_new 0: up to n_tokens per sequence
    assert lib.lcu_attention_paged(AT, AT, 256, 4, p, many, AT, 1 << 40, None) == SHAPE
    assert lib.lcu_attention_paged_workspace(p, many, 4) == 0
    assert lib.lcu_attention_paged(AT, AT, 256, 4, pages(n_pages=1 << 28), b, AT, 1 << 30, None) == SHAPE   # rows past 32 bits
    wide = batch(token_start=AT, n_tokens=65000, max_new=65000)   # rows of one KV head past 31 bits
    assert lib.lcu_attention_paged(AT, AT, 65000 * 64, 65000, pages(n_heads=1), wide, AT, 1 << 60, None) == SHAPE
    assert lib.lcu_attention_paged_workspace(pages(n_heads=1), wide, 65000) == 0


def test_nothing_to_do():
    """No sequence, no token, no row: success without a launch (and without a GPU)."""
    lib, p = L.load(), pages()
    for b in (batch(n_seqs=0, n_tokens=0, seq_len=None, page_table=None), batch(n_tokens=0, token_start=AT)):
        assert append(p, b) == 0
        assert lib.lcu_kv_read_paged(AT, AT, p, b, None) == 0
        assert lib.lcu_attention_paged(AT, AT, 256, 4, p, b, None, 0, None) == 0
    assert lib.lcu_sample(AT, AT, 5, 0, 5, None, None, None, None, AT, None) == 0


def test_sample_refused():
    f = L.load().lcu_sample
    assert f(None, AT, 5, 1, 5, None, None, None, None, AT, None) == NULL
    assert f(AT, None, 5, 1, 5, None, None, None, None, AT, None) == NULL
    assert f(AT, AT, 5, 1, 5, None, None, None, None, None, None) == NULL
    assert f(AT, AT, 4, 1, 5, None, None, None, None, AT, None) == SHAPE
    assert f(AT, AT, 5, 1, 0, None, None, None, None, AT, None) == SHAPE
    assert f(AT, AT, 1 << 20, 1, (1 << 18) + 1, None, None, None, None, AT, None) == SHAPE


def test_plain_quantise():
    """The restatement itself: grid points stay, halves go to the even code, non-finite groups are marked."""
    x = np.array([0, 1, 2, 3, 4, 5, 6, 7, -1, -7, 0.5, 1.5, 2.5, -0.5, -1.5, 6.5], np.float32)
    c, s = kvref.quantise(x)
    assert s.tolist() == [0x38]   # 1.0
    assert kvref.values(c, s).tolist() == [0, 1, 2, 3, 4, 5, 6, 7, -1, -7, 0, 2, 2, 0, -2, 6]
    for bad in (np.nan, np.inf, -np.inf):
        y = np.ones(32, np.float32)
        y[3] = bad
        c, s = kvref.quantise(y)
        assert s[0] == 0x7f and np.isnan(kvref.values(c, s)[:16]).all() and (c[:8] == 0x88).all()
        assert np.isfinite(kvref.values(c, s)[16:]).all()
    assert not kvref.values(*kvref.quantise(np.full(16, 2.0 ** -9, np.float32))).any()   # below half the smallest scale
    assert kvref.values(*kvref.quantise(np.full(16, 1e9, np.float32))).max() == 448 * 7


def test_plain_draw():
    x = np.array([1.0, 3.0, 3.0, -np.inf, np.nan, 2.0])
    assert kvref.draw(x, 0.3, temperature=0.0)[0] == 1
    assert kvref.draw(x, 0.99, top_k=1)[0] == 1
    assert kvref.draw(x, 0.51, top_k=2)[0] == 2
    assert kvref.draw(x, 0.99, min_p=0.5)[0] == 2
    assert kvref.draw(x, 1.0)[0] == 5
    assert kvref.draw(x, 0.0)[0] == 0
    # masses 1, 1, e^-1, e^-2: 0.4 of 2.503 is 1.001, more than the first rank has, so two stay
    assert kvref.draw(x, 0.9, top_p=0.4)[0] == 2
    assert kvref.draw(x, 0.9, top_p=0.0)[0] == 1
    assert kvref.draw(np.full(3, -np.inf), 0.5)[0] == -1
