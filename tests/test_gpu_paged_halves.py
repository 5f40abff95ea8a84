"""The attention over the paged cache holds q and the weights as two 16-bit halves. Rows made so that the low halves alone
decide the answer: without those of q, or those of the weights, each case is many tolerances off."""
import numpy as np
import pytest

import kvref
from test_gpu_paged import Cache, attend, lib, tolerance  # noqa: F401

GROUPS = (3, 8, 16, 20)   # rows to a key head: one kernel shape each, where the head size has it


def small_q(dim, rows):
    """Two keys, all +a and all -a, values +1 and -1. q is -1 on half of its channels and 1 + d, d = 2^-12 .. 1.98 2^-12, on the
    others: the high halves cancel and give equal weights, the exact scores are +-a d sqrt(dim) / 2, 1/2 to 1."""
    rng = np.random.default_rng(dim + rows)
    q = -np.ones((rows, dim), np.float32)
    for r in range(rows):
        more = 1 + np.float32(2.0 ** -12 * rng.uniform(1.0, 1.98))
        q[r, rng.permutation(dim)[:dim // 2]] = more
    k = np.full((2, dim), 2.0 ** 12 / np.sqrt(dim))
    k[1] *= -1
    v = np.ones((2, dim))
    v[1] *= -1
    return q, k, v


def small_p(dim, rows):
    """Eight keys next to zero: weights between 1 and 1/2, whose high halves are up to 2^-12 off."""
    rng = np.random.default_rng(dim * rows)
    q = rng.uniform(-1, 1, (rows, dim)).astype(np.float32)
    k = rng.integers(-7, 8, (8, dim)) * 2.0 ** -9
    v = rng.integers(-7, 8, (8, dim)) * 1.0
    return q, k, v


def halves(x, low=True):
    """x as an f16 number plus, if wanted, the f16 number nearest to what is missing."""
    hi = x.astype(np.float16).astype(np.float64)
    return hi + (x - hi).astype(np.float16).astype(np.float64) if low else hi


def restated(q, k, v, q_low=True, p_low=True):
    """The kernel's arithmetic in 64 bits but for the halves: q scaled by a power of two to 1 .. 2, weights up to 2^7."""
    q = q.astype(np.float64)
    top = 2.0 ** np.floor(np.log2(np.abs(q).max(1, keepdims=True)))
    s = halves(q / top, q_low) * top @ k.T / np.sqrt(q.shape[1])
    p = 2.0 ** 7 * np.exp(s - s.max(1, keepdims=True))
    return halves(p, p_low) @ v / p.sum(1, keepdims=True)


def cases():
    return [(f, dim, rows) for f in (small_q, small_p) for dim in (64, 128, 256) for rows in GROUPS]


def bound(q, k, v):
    ref, size = kvref.attention(q[None], k[:, None], v[:, None], [len(k)])
    return ref[0], tolerance(size, q.shape[1], np.abs(v).max(), len(k))


@pytest.mark.parametrize("make,dim,rows", cases())
def test_oracle_without_a_low_half(make, dim, rows):
    """The cases tell: both halves stay within the tolerance, a missing one does not, by a factor of 4 or more."""
    q, k, v = make(dim, rows)
    ref, tol = bound(q, k, v)
    assert np.max(np.abs(restated(q, k, v) - ref)) <= tol
    lost = restated(q, k, v, q_low=make is not small_q, p_low=make is not small_p)
    assert np.max(np.abs(lost - ref), 1).max() >= 4 * tol
    if make is small_q:
        assert np.max(np.abs(lost - ref), 1).min() >= 4 * tol   # every row


@pytest.mark.gpu
@pytest.mark.parametrize("make,dim,rows", cases())
def test_both_halves_count(lib, make, dim, rows):
    import torch
    q, k, v = make(dim, rows)
    unit = np.float32(np.abs(k).max() / 7)   # codes -7 .. 7 with a scale of 1
    c = Cache([len(k)], 1, dim, 16, (float(unit), 1.0))
    for codes, scales, x in ((c.kc, c.ks, k / np.float64(unit)), (c.vc, c.vs, v)):
        n = np.rint(x).astype(np.int64) + 8
        assert np.allclose(n - 8, x, atol=1e-6, rtol=0) and n.min() >= 1 and n.max() <= 15
        page = int(c.table_np[0, 0])
        codes[page, 0, :len(k)] = torch.from_numpy((n[:, 0::2] + 16 * n[:, 1::2]).astype(np.uint8)).cuda()
        scales[page, 0, :len(k)] = 0x38
    ref, tol = bound(q, c.kv(0, len(k))[0][:, 0], v)
    out = attend(lib, c, c.batch([len(k)]), q[None], rows).reshape(rows, dim)
    assert np.max(np.abs(out - ref)) <= tol
