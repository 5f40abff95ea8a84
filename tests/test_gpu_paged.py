"""The paged 4-bit cache on the GPU: appending, reading back, attention over it, sampling, and a decode loop of
them, against the 64-bit restatements in kvref.py."""
import numpy as np
import pytest

import kvref
import lancius_b200 as L

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")
SHAPE = -3
BASE = 10000.0


@pytest.fixture(scope="module")
def lib():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    lib = L.load()
    lib.lcu_check_stream(None)
    return lib


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def ptr(t):
    return None if t is None else t.data_ptr()


class Cache:
    """A cache with room for `lens`, pages handed out in shuffled order, filled with `fill` bytes."""

    def __init__(self, lens, heads, dim, page, unit=(1.0, 1.0), seed=0, fill=0, spare=2):
        rng = np.random.default_rng(seed)
        need = [-(-n // page) for n in lens]
        total = sum(need) + spare
        ids = rng.permutation(total)
        self.table_np = np.full((len(lens), max(max(need), 1)), -1, np.int32)   # unused entries are no pages
        at = 0
        for b, n in enumerate(need):
            self.table_np[b, :n] = ids[at:at + n]
            at += n
        self.unused = torch.from_numpy(ids[at:].copy()).cuda()
        self.heads, self.dim, self.page, self.unit = heads, dim, page, unit
        mk = lambda w: torch.full((total, heads, page, w), fill, dtype=torch.uint8, device="cuda")
        self.kc, self.vc, self.ks, self.vs = mk(dim // 2), mk(dim // 2), mk(dim // 16), mk(dim // 16)
        self.table = i32(self.table_np)
        self.pages = L.KvPages(ptr(self.kc), ptr(self.vc), ptr(self.ks), ptr(self.vs), total, page, heads, dim, *unit)

    def batch(self, seq_len, start=None, tokens=None, max_len=0, max_new=0):
        self.hold = (i32(seq_len), None if start is None else i32(start))
        n = tokens if tokens is not None else len(seq_len) if start is None else start[-1]
        return L.KvBatch(ptr(self.table), self.table.shape[1], ptr(self.hold[0]), ptr(self.hold[1]), len(seq_len), n,
                         max_len, max_new)

    def rows(self, s, n):
        """Bytes of sequence s's first n rows: codes and scales of k and v, [n, heads, ...]."""
        out = []
        for t in (self.kc, self.ks, self.vc, self.vs):
            a = t.cpu().numpy()
            j = np.arange(n)
            out.append(a[self.table_np[s, j // self.page], :, j % self.page])
        return out

    def kv(self, s, n):
        kc, ks, vc, vs = self.rows(s, n)
        return kvref.values(kc, ks, self.unit[0]), kvref.values(vc, vs, self.unit[1])


def fill_random(c, seed, spread=1.0):
    rng = np.random.default_rng(seed)
    for codes, scales in ((c.kc, c.ks), (c.vc, c.vs)):
        x = rng.standard_normal((*codes.shape[:3], c.dim)).astype(np.float32) * spread
        a, b = kvref.quantise(x)
        codes.copy_(torch.from_numpy(a))
        scales.copy_(torch.from_numpy(b))


def starts(new):
    return [0] + [int(n) for n in np.cumsum(new)]


def append(lib, c, b, x, hq, base=BASE, ld=None, stream=None):
    """x [T, (hq + 2 heads) dim] as one projection's output (row stride ld); returns the rotated q."""
    w = (hq + 2 * c.heads) * c.dim
    ld = ld or w
    buf = torch.zeros((max(len(x), 1), ld), device="cuda")
    buf[:len(x), :w] = torch.from_numpy(x)
    q = torch.full((len(x), hq * c.dim), 7.0, device="cuda")
    at = buf.data_ptr()
    k = at + 4 * hq * c.dim
    rc = lib.lcu_kv_append_paged(c.pages, b, ptr(q) if hq else None, at if hq else None, ld, hq, k, ld,
                                 k + 4 * c.heads * c.dim, ld, base, stream)
    assert rc == 0
    torch.cuda.synchronize()
    return q.cpu().numpy()


def attend(lib, c, b, q, hq, ld=None, stream=None, out=None):
    n = c.heads * c.dim
    t = torch.zeros((len(q), ld or hq * c.dim), device="cuda")
    t[:, :hq * c.dim] = torch.from_numpy(np.asarray(q, np.float32).reshape(len(q), -1))
    out = torch.full((len(q), hq * c.dim), 7.0, device="cuda") if out is None else out
    need = lib.lcu_attention_paged_workspace(c.pages, b, hq)
    space = torch.full((max(need, 16),), 0xff, dtype=torch.uint8, device="cuda")
    assert n and lib.lcu_attention_paged(ptr(out), ptr(t), t.shape[1], hq, c.pages, b, ptr(space), need, stream) == 0
    torch.cuda.synchronize()
    return out.cpu().numpy()


def tolerance(size, dim, vmax, limit):
    """Bound of an output's error. A score is a sum of q k held in at least 22 bits and added in FP32 (each of the
    dim / 16 partial sums truncated, 2^-23): with Σ|q||k| / sqrt(dim) <= size it is off by size (2^-22 + (dim / 16 + 2)
    2^-23). A weight is off by that, relatively, plus 2^-22 for exp2 and 2^-22 for its own bits; the weights' sum as
    much. Sums over keys: each of up to `limit` / 16 partial sums truncated, but no warp adds more than 1024 keys."""
    w = size * (2.0 ** -22 + (dim / 16 + 2) * 2.0 ** -23) + 2.0 ** -21
    return vmax * (2 * w + (min(limit, 1024) / 16 + 4) * 2.0 ** -23)


# ---- append and read -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim,page,heads,hq,new,past,unit,ld", [
    (128, 16, 2, 2, [1], [0], (1.0, 1.0), None),               # the very first token
    (128, 16, 2, 4, [3, 0, 1, 17, 33], [0, 5, 15, 14, 1000], (1.0, 1.0), None),   # an empty sequence, page borders
    (64, 8, 3, 6, [7, 9], [1, 120000], (0.25, 3.0), 64 * 12 + 4),
    (64, 1, 1, 1, [2, 1, 1], [3, 0, 7], (1.0, 1.0), 64 * 3 + 1),   # unaligned rows
    (256, 4096, 1, 8, [5], [4090], (1.0, 0.01), None),
    (256, 32, 2, 2, [130], [0], (1.0, 1.0), None)])
def test_append_and_read(lib, dim, page, heads, hq, new, past, unit, ld):
    rng = np.random.default_rng(dim + page)
    lens = [a + b for a, b in zip(past, new)]
    c = Cache(lens, heads, dim, page, unit, seed=3, fill=0x5a)
    b = c.batch(lens, starts(new))
    t = sum(new)
    x = (rng.standard_normal((t, hq + 2 * heads, dim)) * np.exp(rng.standard_normal((1, hq + 2 * heads, dim)))).astype(np.float32)
    if hq >= heads:
        x[:, :heads] = x[:, hq:hq + heads]   # the first q heads hold the keys' numbers: their rotated form is seen in q_out
    before = [a.clone() for a in (c.kc, c.ks, c.vc, c.vs)]
    q = append(lib, c, b, x.reshape(t, -1), hq, ld=ld).reshape(t, hq, dim)
    pos = np.concatenate([np.arange(n - k, n) for n, k in zip(lens, new)])
    want = kvref.rotate(x[:, :hq], pos, BASE)
    # rounded to FP32 once, half a step; sines of angles up to 120000 known to 2^-53 of the angle and a few steps
    pair = np.hypot(want[..., 0::2], want[..., 1::2]).repeat(2, -1)
    assert np.all(np.abs(q - want) <= 2.0 ** -24 * np.abs(want) + 1e-10 * pair)
    at = 0
    touched = np.zeros(c.kc.shape[:1] + (page,), bool)
    for s, (n, k) in enumerate(zip(lens, new)):
        kc, ks, vc, vs = c.rows(s, n)
        for got, ref in zip((kc[n - k:], ks[n - k:]), kvref.quantise(q[at:at + k, :heads], unit[0])):
            assert np.array_equal(got, ref)
        for got, ref in zip((vc[n - k:], vs[n - k:]), kvref.quantise(x[at:at + k, hq + heads:], unit[1])):
            assert np.array_equal(got, ref)
        for j in range(n - k, n):
            touched[c.table_np[s, j // page], j % page] = True
        at += k
    for a, o in zip((c.kc, c.ks, c.vc, c.vs), before):   # every other slot as it was
        same = (a == o).all(-1).all(1).cpu().numpy()
        assert same[~touched].all()
    ko = torch.full((t, heads, dim), 7.0, device="cuda")
    vo = torch.full((t, heads, dim), 7.0, device="cuda")
    assert lib.lcu_kv_read_paged(ptr(ko), ptr(vo), c.pages, b, None) == 0
    assert lib.lcu_check_stream(None) == 0
    want_k = np.concatenate([c.kv(s, n)[0][n - k:] for s, (n, k) in enumerate(zip(lens, new))])
    want_v = np.concatenate([c.kv(s, n)[1][n - k:] for s, (n, k) in enumerate(zip(lens, new))])
    for got, ref in ((ko, want_k), (vo, want_v)):   # code * scale is exact in FP32, the unit rounds once
        assert np.all(np.abs(got.cpu().numpy() - ref) <= 2.0 ** -24 * np.abs(ref))


def test_append_in_place_and_without_q(lib):
    c, d = Cache([9, 4], 2, 64, 16, seed=1), Cache([9, 4], 2, 64, 16, seed=1)
    x = np.random.default_rng(0).standard_normal((2, 8 * 64)).astype(np.float32)
    b = c.batch([9, 4])
    want = append(lib, c, b, x, 4)
    q = torch.from_numpy(x[:, :256].copy()).cuda()
    kv = torch.from_numpy(x[:, 256:].copy()).cuda()
    bd = d.batch([9, 4])
    assert lib.lcu_kv_append_paged(d.pages, bd, ptr(q), ptr(q), 256, 4, ptr(kv), 256, ptr(kv) + 512, 256, BASE, None) == 0
    torch.cuda.synchronize()
    assert np.array_equal(q.cpu().numpy(), want)
    for a, o in ((c.kc, d.kc), (c.ks, d.ks), (c.vc, d.vc), (c.vs, d.vs)):
        assert torch.equal(a, o)
    d.kc.zero_()
    assert lib.lcu_kv_append_paged(d.pages, bd, None, None, 0, 0, ptr(kv), 256, ptr(kv) + 512, 256, BASE, None) == 0
    torch.cuda.synchronize()
    assert torch.equal(c.kc, d.kc)


def test_append_no_rotation_and_odd_values(lib):
    """rope_base 0 keeps the numbers; zeros, subnormals, infinities, NaN, rounding borders and values over the largest."""
    x = np.zeros((1, 3, 128), np.float32)
    x[0, 0] = np.tile(np.array([0, -0.0, 1e-40, 0.5, 1.5, 2.5, 3.5, 4.5, 5.5, 6.5, 7, -0.5, -1.5, -2.5, -6.5, -7], np.float32), 8)
    x[0, 1, :16] = 1e30
    x[0, 1, 16] = np.nan
    x[0, 1, 40] = np.inf
    x[0, 1, 50] = -np.inf
    x[0, 1, 64:80] = 2.0 ** -10 * 3      # scale 2^-11: below half of the smallest
    x[0, 1, 80:96] = np.linspace(-7 * 2.0 ** -9, 7 * 2.0 ** -9, 16)   # the smallest scale
    x[0, 2] = x[0, 1, ::-1]
    c = Cache([1], 1, 128, 16)
    q = append(lib, c, c.batch([1]), x.reshape(1, -1), 1, base=0.0)
    assert np.array_equal(q.reshape(-1).view(np.uint32), x[0, 0].view(np.uint32))
    got = c.rows(0, 1)
    for a, ref in zip(got, (*kvref.quantise(x[:, 1]), *kvref.quantise(x[:, 2]))):
        assert np.array_equal(a[:, 0], ref)


def test_rows_of_no_sequence_stay(lib):
    """Padded rows behind the last sequence, and idle slots (seq_len 0), are neither appended nor rotated."""
    c = Cache([20, 20], 1, 64, 16, fill=3)
    x = np.random.default_rng(1).standard_normal((8, 3 * 64)).astype(np.float32)
    b = c.batch([20, 20], [0, 2, 3], tokens=8)
    q = append(lib, c, b, x, 1)
    assert (q[3:] == 7.0).all() and not (q[:3] == 7.0).any()
    out = attend(lib, c, b, x[:, :64], 1)
    assert (out[3:] == 7.0).all() and not (out[:3] == 7.0).any()
    c = Cache([20, 20], 1, 64, 16, fill=3)
    kc = c.kc.clone()
    b = c.batch([0, 0])
    assert (append(lib, c, b, x[:2], 1) == 7.0).all() and torch.equal(kc, c.kc)
    assert (attend(lib, c, b, x[:2, :64], 1) == 0.0).all()
    # two new tokens but one key: the first has position -1
    b = c.batch([1], [0, 2])
    q = append(lib, c, b, x[:2], 1)
    assert (q[0] == 7.0).all() and not (q[1] == 7.0).any()
    out = attend(lib, c, b, x[:2, :64], 1)
    assert (out[0] == 0.0).all() and not (out[1] == 0.0).all()
    assert lib.lcu_check_stream(None) == 0


def test_bad_pages_and_lengths_are_reported(lib):
    c = Cache([40, 40], 1, 64, 16, fill=3)
    fill_random(c, 1)
    x = np.random.default_rng(1).standard_normal((2, 3 * 64)).astype(np.float32)
    for page in (-1, c.kc.shape[0], 2 ** 31 - 1):
        keep = c.kc.clone()
        c.table[1, 2] = page
        b = c.batch([40, 40])
        append(lib, c, b, x, 1)
        assert lib.lcu_check_stream(None) == SHAPE and lib.lcu_check_stream(None) == 0
        changed = (keep != c.kc).any(-1).any(1).sum().item()
        assert changed <= 1   # the first sequence's row
        ko, vo = torch.full((2, 1, 64), 7.0, device="cuda"), torch.full((2, 1, 64), 7.0, device="cuda")
        assert lib.lcu_kv_read_paged(ptr(ko), ptr(vo), c.pages, b, None) == 0
        assert lib.lcu_check_stream(None) == SHAPE
        assert (ko[1] == 0).all() and (ko[0] != 0).any()
        out = attend(lib, c, b, x[:, :64], 1)
        assert lib.lcu_check_stream(None) == SHAPE and lib.lcu_check_stream(None) == 0
        # the page's keys count as zeros
        k, v = c.kv(1, 40)
        k[32:], v[32:] = 0, 0
        ref, size = kvref.attention(x[1:, :64].reshape(1, 1, 64), k, v, [40])
        assert np.max(np.abs(out[1] - ref.reshape(-1))) <= tolerance(size, 64, np.abs(v).max(), 40)
    c.table[1, 2] = int(c.table_np[1, 2])
    b = c.batch([40, 49])   # one position past the table
    append(lib, c, b, x, 1)
    assert lib.lcu_check_stream(None) == SHAPE
    attend(lib, c, b, x[:, :64], 1)
    assert lib.lcu_check_stream(None) == SHAPE
    b = c.batch([40, 30], max_len=33)   # over the host's bound: the keys up to it
    out = attend(lib, c, b, x[:, :64], 1)
    assert lib.lcu_check_stream(None) == SHAPE
    k, v = c.kv(0, 33)
    ref, size = kvref.attention(x[:1, :64].reshape(1, 1, 64), k, v, [33])
    assert np.max(np.abs(out[0] - ref.reshape(-1))) <= tolerance(size, 64, np.abs(v).max(), 33)


# ---- attention -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dim,page,heads,group,lens,new,unit", [
    (128, 16, 2, 1, [1], [1], (1.0, 1.0)),
    (128, 16, 2, 4, [31, 32, 33, 1, 64, 0, 127, 129], None, (1.0, 1.0)),
    (128, 32, 1, 8, [700, 3, 1500], None, (0.5, 2.0)),
    (128, 1, 2, 3, [5, 70], None, (1.0, 1.0)),                  # group of three, pages of one token
    (128, 16, 1, 16, [300], None, (1.0, 1.0)),                  # more than eight rows to a key head
    (128, 64, 2, 2, [100, 40, 260], [5, 0, 9], (1.0, 1.0)),     # several new tokens, one sequence without
    (128, 16, 1, 2, [40], [40], (1.0, 1.0)),                    # the whole sequence is new
    (64, 8, 3, 4, [200, 65, 2], [1, 3, 2], (1.0, 1.0)),
    (64, 16, 1, 12, [1000, 17], [2, 7], (3.0, 0.125)),
    (256, 16, 1, 8, [500, 90, 33], None, (1.0, 1.0)),
    (256, 4096, 2, 2, [130], [3], (1.0, 1.0)),
    (64, 16, 1, 1, [9000], None, (1.0, 1.0)),                   # one row, a long cache: split and joined
    (128, 16, 1, 4, [20000, 5], None, (1.0, 1.0)),
    (256, 32, 1, 2, [12000], [6], (1.0, 1.0))])
def test_attention(lib, dim, page, heads, group, lens, new, unit):
    rng = np.random.default_rng(sum(lens) + dim)
    c = Cache([max(n, 1) for n in lens], heads, dim, page, unit, seed=4)
    fill_random(c, 5)
    c.ks[c.unused], c.vs[c.unused] = 0x7f, 0x7f
    hq, one = heads * group, new is None
    new = [1] * len(lens) if one else new
    # slots behind the last key hold NaN: they must not be seen
    for s, n in enumerate(lens):
        last = c.table_np[s, max(n - 1, 0) // page]
        c.ks[last, :, (n - 1) % page + 1 if n else 0:] = 0x7f
        c.vs[last, :, (n - 1) % page + 1 if n else 0:] = 0x7f
    q = rng.standard_normal((sum(new), hq, dim)).astype(np.float32) * 1.2
    b = c.batch(lens, None if one else starts(new), max_new=0 if one else max(new))
    out = attend(lib, c, b, q, hq, ld=hq * dim + (0 if dim == 64 else 3)).reshape(-1, hq, dim)
    assert lib.lcu_check_stream(None) == 0
    at = 0
    for s, (n, k) in enumerate(zip(lens, new)):
        kk, vv = c.kv(s, n)
        ref, size = kvref.attention(q[at:at + k], kk, vv, [n - k + 1 + i for i in range(k)])
        if k:
            tol = tolerance(size, dim, np.abs(vv).max() if n else 1.0, n)
            assert np.max(np.abs(out[at:at + k] - ref)) <= tol
        at += k


@pytest.mark.parametrize("dim,page,heads,group,lens,new", [
    (64, 16, 2, 4, [700, 20, 5], [5, 5, 5]),         # 20 rows to a key head
    (64, 32, 1, 8, [100, 2500], [3, 6]),             # 24 rows, and 48 in two blocks
    (128, 16, 2, 4, [333, 64], [5, 2]),
    (128, 32, 1, 8, [200, 90, 1900], [3, 1, 6]),
    (128, 64, 3, 3, [130], [9]),                     # 27 rows: blocks of 16 whose second is not full
    (256, 16, 1, 4, [300, 44], [5, 1]),
    (256, 32, 2, 8, [1000, 257, 1], None),
    (128, 16, 8, 4, [777], None),                    # up to eight chunks: joined within one launch
    (128, 16, 1, 1, [1024, 1, 128, 129, 0, 900], None),
    (64, 8, 2, 8, [513, 1000], None),
    (256, 16, 1, 2, [640], [2])])
def test_attention_aligned_rows(lib, dim, page, heads, group, lens, new):
    """Rows of q without gaps, more rows to a key head, few chunks; the second sequence starts with the first one's pages."""
    c = Cache([max(n, 1) for n in lens], heads, dim, page, seed=8)
    fill_random(c, 9)
    c.ks[c.unused], c.vs[c.unused] = 0x7f, 0x7f
    if len(lens) > 1:
        same = min(lens[0], lens[1]) // page
        c.table_np[1, :same] = c.table_np[0, :same]
        c.table.copy_(i32(c.table_np))
    hq, one = heads * group, new is None
    new = [1] * len(lens) if one else new
    q = np.random.default_rng(sum(lens)).standard_normal((sum(new), hq, dim)).astype(np.float32)
    b = c.batch(lens, None if one else starts(new), max_new=0 if one else max(new))
    out = attend(lib, c, b, q, hq).reshape(-1, hq, dim)
    assert lib.lcu_check_stream(None) == 0
    at = 0
    for s, (n, k) in enumerate(zip(lens, new)):
        kk, vv = c.kv(s, n)
        ref, size = kvref.attention(q[at:at + k], kk, vv, [n - k + 1 + i for i in range(k)])
        assert np.max(np.abs(out[at:at + k] - ref)) <= tolerance(size, dim, np.abs(vv).max() if n else 1.0, n)
        at += k


def test_attention_extreme_scores(lib):
    """Rows whose scores lie far apart, large and tiny queries, a zero query, equal keys."""
    c = Cache([300], 1, 128, 16)
    fill_random(c, 8)
    rng = np.random.default_rng(2)
    q = rng.standard_normal((5, 1, 128)).astype(np.float32)
    for i, f in enumerate((1e-30, 0.0, 1.0, 60.0, 1e5)):
        k, v = c.kv(0, 300)
        row = (q[i:i + 1] * np.float32(f)).astype(np.float32)
        out = attend(lib, c, c.batch([300]), row, 1).reshape(1, 1, 128)
        ref, size = kvref.attention(row, k, v, [300])
        tol = tolerance(size, 128, np.abs(v).max(), 300)
        if f <= 60:
            assert np.max(np.abs(out - ref)) <= tol
        else:   # one key takes all the weight
            s = (k[:, 0] @ row[0, 0].astype(np.float64))
            assert np.max(np.abs(out[0, 0] - v[np.argmax(s), 0])) <= 2.0 ** -20 * np.abs(v).max()


def test_nan_shows_only_where_seen(lib):
    """A NaN key or value makes the rows that see it NaN, in all channels, and no others."""
    for which in ("ks", "vs"):
        for dim in (64, 128, 256):
            c = Cache([50, 50], 2, dim, 16, seed=dim)
            fill_random(c, 9)
            page, slot = int(c.table_np[0, 47 // 16]), 47 % 16
            getattr(c, which)[page, 1, slot, 2] = 0x7f
            q = np.random.default_rng(3).standard_normal((8, 4, dim)).astype(np.float32)
            b = c.batch([50, 50], [0, 4, 8])
            out = attend(lib, c, b, q, 4).reshape(8, 4, dim)
            bad = np.isnan(out)
            want = np.zeros((8, 4), bool)
            want[1:4, 2:] = True        # rows at positions 47, 48, 49 of the first sequence, the second key head
            assert np.array_equal(bad.all(-1), want) and np.array_equal(bad.any(-1), want)
    c = Cache([50, 50], 1, 128, 16)
    fill_random(c, 9)
    q = np.random.default_rng(3).standard_normal((2, 2, 128)).astype(np.float32)
    q[0, 1, 5] = np.nan
    q[1, 0, 7] = np.inf
    out = attend(lib, c, c.batch([50, 50]), q, 2).reshape(2, 2, 128)
    assert np.array_equal(np.isnan(out).all(-1), [[False, True], [True, False]])
    assert np.isfinite(out[0, 0]).all() and np.isfinite(out[1, 1]).all()


def test_attention_workspace_too_small(lib):
    c = Cache([9000], 1, 64, 16)
    b = c.batch([9000])
    q = torch.zeros((1, 64), device="cuda")
    need = lib.lcu_attention_paged_workspace(c.pages, b, 1)
    if need:
        space = torch.empty(need, dtype=torch.uint8, device="cuda")
        assert lib.lcu_attention_paged(ptr(q), ptr(q), 64, 1, c.pages, b, ptr(space), need - 1, None) == -9
        assert lib.lcu_attention_paged(ptr(q), ptr(q), 64, 1, c.pages, b, None, need, None) == -2
        assert lib.lcu_attention_paged(ptr(q), ptr(q), 64, 1, c.pages, b, ptr(space) + 8, need, None) == -5


def test_repeated_calls_give_the_same_bits(lib):
    c = Cache([5000, 33, 800], 2, 128, 16)
    fill_random(c, 12)
    q = np.random.default_rng(3).standard_normal((3, 8, 128)).astype(np.float32)
    b = c.batch([5000, 33, 800])
    first = attend(lib, c, b, q, 8)
    for _ in range(3):
        assert np.array_equal(first, attend(lib, c, b, q, 8))


# ---- sampling --------------------------------------------------------------------------------------------------

def sample(lib, x, u, temperature=None, top_k=None, top_p=None, min_p=None, ld=None, stream=None):
    rows, v = x.shape
    buf = torch.full((rows, ld or v), 99.0, device="cuda")
    buf[:, :v] = torch.from_numpy(x)
    f32 = lambda a: None if a is None else torch.tensor(np.broadcast_to(a, rows).copy(), dtype=torch.float32, device="cuda")
    t, k, p, m = f32(temperature), None if top_k is None else i32(np.broadcast_to(top_k, rows)), f32(top_p), f32(min_p)
    uu = f32(u)
    out = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    assert lib.lcu_sample(ptr(out), ptr(buf), buf.shape[1], rows, v, ptr(t), ptr(k), ptr(p), ptr(m), ptr(uu), stream) == 0
    torch.cuda.synchronize()
    return out.cpu().numpy()


def check_sample(got, x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    rows = len(got)
    f = lambda a: np.broadcast_to(np.asarray(a, np.float32), rows).astype(np.float64)
    k = np.broadcast_to(top_k, rows)
    t, p, m, uu = f(temperature), f(top_p), f(min_p), f(u)
    for i in range(rows):
        want, gap = kvref.draw(x[i], uu[i], t[i], int(k[i]), p[i], m[i])
        # sums in 64 bits: only a u within 1e-11 of a border may go either way
        assert got[i] == want or gap < 1e-11, (i, got[i], want, gap)


@pytest.mark.parametrize("rows,vocab,ld", [(1, 1, None), (3, 2, 5), (5, 31, None), (4, 33, 40), (7, 1000, 1001), (3, 4097, None),
                                           (2, 32768, None), (3, 50021, 50024), (2, 131072, None), (1, 262144, None)])
@pytest.mark.parametrize("bits", [32, 16])
def test_sample(lib, rows, vocab, ld, bits):
    rng = np.random.default_rng(vocab + bits)
    x = (rng.standard_normal((rows, vocab)) * 2.5).astype(np.float32)
    if bits == 16:   # many ties
        x = torch.from_numpy(x).bfloat16().float().numpy()
    u = rng.random(rows).astype(np.float32)
    for kw in (dict(), dict(temperature=0.0), dict(temperature=0.7), dict(top_k=1), dict(top_k=50), dict(top_k=vocab),
               dict(top_k=max(1, vocab // 2)), dict(top_p=0.9), dict(top_p=0.999), dict(top_p=0.0), dict(min_p=0.05),
               dict(min_p=1.0), dict(temperature=1.3, top_k=40, top_p=0.8, min_p=0.02), dict(top_k=3000, top_p=0.95)):
        check_sample(sample(lib, x, u, ld=ld, **kw), x, u, **kw)


def test_sample_rows_differ(lib):
    rng = np.random.default_rng(5)
    x = (rng.standard_normal((64, 5003)) * 3).astype(np.float32)
    kw = dict(temperature=np.where(rng.random(64) < 0.3, 0, rng.random(64) + 0.3), top_k=rng.integers(-1, 300, 64),
              top_p=rng.random(64) * 1.2, min_p=rng.random(64) * 0.2 - 0.1)
    u = rng.random(64)
    check_sample(sample(lib, x, u, **kw), x, u, **kw)


@pytest.mark.parametrize("rows,vocab", [(400, 1500), (170, 20001)])
def test_sample_many_rows(lib, rows, vocab):
    """More CTAs than two per SM."""
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((rows, vocab)) * rng.uniform(0.5, 4, (rows, 1))).astype(np.float32)
    x[::3] = torch.from_numpy(x[::3]).bfloat16().float().numpy()
    kw = dict(temperature=np.where(rng.random(rows) < 0.1, 0, rng.random(rows) + 0.3), top_k=rng.integers(-200, 700, rows),
              top_p=rng.random(rows) * 1.5, min_p=rng.random(rows) * 0.1 - 0.06)
    u = rng.random(rows)
    check_sample(sample(lib, x, u, **kw), x, u, **kw)
    check_sample(sample(lib, x, u), x, u)


def test_sample_odd_logits(lib):
    inf, nan = np.inf, np.nan
    v = 300
    x = np.full((10, v), -inf, np.float32)
    x[1, 5] = -3e38
    x[2, [7, 200]] = inf
    x[2, 8] = 3e38
    x[3] = nan
    x[4] = 0.0
    x[4, ::2] = -0.0                     # equal to zero
    x[5] = np.linspace(-1e-38, 1e-38, v)
    x[6, 10:20] = -3.4e38                # masked with the lowest value ...
    x[6, 100] = 1.0
    x[7] = 3.0
    x[7, 3] = nan
    x[8] = np.float32(-3.4028235e38)     # ... in every place
    x[9, v - 1] = 2.0
    x[9, 0] = 2.0
    for u in (0.0, 0.25, 0.5, 0.9999999, 1.0):
        for kw in (dict(), dict(top_k=2), dict(top_p=0.5), dict(min_p=0.3), dict(top_k=101, top_p=0.7), dict(temperature=0.0),
                   dict(temperature=np.nan)):
            got = sample(lib, x, np.full(10, u, np.float32), **kw)
            if "temperature" in kw:
                kw = dict(temperature=0.0)
            check_sample(got, x, np.full(10, u, np.float32), **kw)
    assert sample(lib, x, 0.1)[[0, 3]].tolist() == [-1, -1]


def test_sample_min_p_over_one(lib):
    """Counts as 1: all that equal the largest stay."""
    x = np.zeros((3, 40), np.float32)
    x[1, 5:30] = 2.0
    x[2, [3, 39]] = np.inf
    for u in (0.0, 0.3, 0.6, 0.999):
        uu = np.full(3, u, np.float32)
        got = sample(lib, x, uu, min_p=1.3)
        check_sample(got, x, uu, min_p=1.0)
        assert got.tolist() == [int(40 * u), 5 + int(25 * u), 39 if u >= 0.5 else 3]


def test_sample_extreme_temperatures(lib):
    """Temperatures at which every other logit weighs nothing, or all weigh the same; logits far from zero."""
    rng = np.random.default_rng(11)
    x = (rng.standard_normal((6, 9000)) * 3).astype(np.float32)
    x[2] += 3e4
    x[3] *= 1e30
    x[4] = np.where(rng.random(9000) < 0.5, np.float32(1.0), np.nextafter(np.float32(1.0), np.float32(2.0)))
    x[5, :40] = -np.inf
    u = np.array([0.2, 0.4, 0.6, 0.8, 0.3, 0.999], np.float32)
    for t in (1e-30, 1e-12, 1e-7, 1e-3, 50.0, 1e6, 1e30, np.inf):
        for kw in (dict(), dict(top_k=30), dict(top_k=2000), dict(top_p=0.7), dict(min_p=0.2)):
            got = sample(lib, x, u, temperature=t, **kw)
            check_sample(got, x, u, temperature=t, **kw)


def test_sample_logits_far_from_zero(lib):
    """Neighbouring FP32 values lie further apart than the weights reach, or the range passes FP32's largest number."""
    rng = np.random.default_rng(12)
    v = 5003
    x = np.zeros((6, v), np.float32)
    steps = rng.integers(0, 6, (6, v))
    for i, top in enumerate((1e10, 1e12, 3e38, -1e12)):
        x[i] = top
        for s in range(1, 6):
            lower = np.nextafter(x[i], np.float32(-np.inf))
            x[i] = np.where(steps[i] >= s, lower, x[i])
    x[4] = rng.choice(np.array([3.4e38, 1e38, -3.4e38, 0], np.float32), v)
    x[5] = -1e30
    x[5, [17, 4000]] = np.float32(-1e12)
    u = np.array([0.2, 0.4, 0.6, 0.8, 0.3, 0.7], np.float32)
    for t in (1e-3, 0.7, 1.0, 2.0, 50.0, 100.0, 1000.0, 1e5, 1e37):
        for kw in (dict(), dict(top_k=3), dict(top_k=200), dict(top_k=2000), dict(top_p=0.7), dict(min_p=0.2), dict(min_p=1e-6)):
            check_sample(sample(lib, x, u, temperature=t, **kw), x, u, temperature=t, **kw)


def test_sample_last_kept(lib):
    """u = 1 and NaN take the last kept index that weighs anything, also where its weight is far below the others'."""
    x = np.full((4, 700), -np.inf, np.float32)
    x[:, 5] = 0.0
    x[0, 600] = -600.0           # 2^-866
    x[1, 600] = -800.0           # nothing
    x[2, [300, 650]] = -60.0
    x[3] = np.linspace(0, -650, 700)
    for u in (1.0, 7.0, np.nan):
        for kw in (dict(), dict(top_k=4), dict(top_k=600), dict(min_p=0.0)):
            got = sample(lib, x, np.full(4, u, np.float32), **kw)
            want = [600, 5, 650, min(kw.get("top_k", 700), 700) - 1]
            assert got.tolist() == want, (u, kw)


def test_sample_follows_the_distribution(lib):
    """Evenly spaced u hit each token in proportion to its mass, to one hit either way."""
    x = np.random.default_rng(6).standard_normal(50).astype(np.float32)
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    got = np.bincount(sample(lib, np.tile(x, (n, 1)), u, top_k=20, temperature=0.8), minlength=50)
    w, _ = kvref.kept(x, float(np.float32(0.8)), 20, 1.0, 0.0)
    assert np.all(np.abs(got - n * w / w.sum()) <= 1.0)


@pytest.mark.parametrize("vocab", [5000, 40000, 262144])
def test_sample_many_equal_logits(lib, vocab):
    """More equal logits at the cut than a list holds; rows that are mostly masked with the type's lowest value."""
    rng = np.random.default_rng(vocab)
    x = np.zeros((5, vocab), np.float32)
    x[1, ::3] = 2.5
    x[2] = np.round(rng.standard_normal(vocab))
    x[3] = np.float32(-3.4028235e38)
    some = rng.choice(vocab, 2000, replace=False)
    x[3, some] = rng.standard_normal(2000)
    x[4] = -np.inf
    x[4, some] = np.round(rng.standard_normal(2000) * 4) / 4
    for u in (0.0, 0.31, 0.77, 0.999):
        uu = np.full(5, u, np.float32)
        for kw in (dict(top_k=1500), dict(top_k=700, top_p=0.37), dict(top_p=0.37), dict(top_p=0.9999), dict(top_k=300, min_p=0.5),
                   dict(min_p=0.01, top_p=0.63, temperature=0.4)):
            check_sample(sample(lib, x, uu, **kw), x, uu, **kw)


# ---- together ----------------------------------------------------------------------------------------------------

def model(lib, seed, hq, heads, dim, vocab):
    rng = np.random.default_rng(seed)
    w = (hq + 2 * heads) * dim
    emb = torch.from_numpy(rng.standard_normal((vocab, 64)).astype(np.float32)).cuda()
    proj = torch.from_numpy((rng.standard_normal((64, w)) / 8).astype(np.float32)).cuda()
    head = torch.from_numpy((rng.standard_normal((hq * dim, vocab)) / 8).astype(np.float32)).cuda()
    return emb, proj, head


def step(lib, m, c, b, ids, hq, u, space, stream, bufs):
    """One step of a one-layer decoder through the library's calls: projection, append, attention, logits, token."""
    emb, proj, head = m
    qkv, q, o, logits, token, x = bufs
    heads, dim, t = c.heads, c.dim, x.shape[0]
    torch.index_select(emb, 0, ids, out=x)
    ld = qkv.shape[1]
    assert lib.lcu_matmul(ptr(qkv), ptr(x), ptr(proj), t, 64, ld, None, 0, 0, stream) == 0
    k = ptr(qkv) + 4 * hq * dim
    assert lib.lcu_kv_append_paged(c.pages, b, ptr(q), ptr(qkv), ld, hq, k, ld, k + 4 * heads * dim, ld, BASE, stream) == 0
    assert lib.lcu_attention_paged(ptr(o), ptr(q), hq * dim, hq, c.pages, b, ptr(space), space.numel(), stream) == 0
    assert lib.lcu_matmul(ptr(logits), ptr(o), ptr(head), t, hq * dim, head.shape[1], None, 0, 0, stream) == 0
    assert lib.lcu_sample(ptr(token), ptr(logits), head.shape[1], t, head.shape[1], None, None, None, None, ptr(u), stream) == 0


def buffers(t, hq, heads, dim, vocab):
    e = lambda *s: torch.empty(s, device="cuda")
    return (e(t, (hq + 2 * heads) * dim), e(t, hq * dim), e(t, hq * dim), e(t, vocab),
            torch.zeros(t, dtype=torch.int32, device="cuda"), e(t, 64))


@pytest.mark.parametrize("dim,page", [(64, 16), (128, 8)])
def test_decode_loop_matches_prompt_pass(lib, dim, page):
    """Tokens fed one at a time (a side stream, then a captured graph replayed) leave the same cache and give the
    same answers as the whole sequences appended and attended in one call."""
    hq, heads, vocab, n, seqs = 4, 2, 500, 37, 3
    m = model(lib, 1, hq, heads, dim, vocab)
    rng = np.random.default_rng(2)
    fed = torch.from_numpy(rng.integers(0, vocab, (seqs, n))).cuda()
    u = torch.from_numpy(rng.random((n, seqs)).astype(np.float32)).cuda()
    c = Cache([n] * seqs, heads, dim, page, seed=7)
    lens = torch.zeros(seqs, dtype=torch.int32, device="cuda")
    b = L.KvBatch(ptr(c.table), c.table.shape[1], ptr(lens), None, seqs, seqs, n, 1)
    space = torch.empty(max(16, lib.lcu_attention_paged_workspace(c.pages, b, hq)), dtype=torch.uint8, device="cuda")
    bufs = buffers(seqs, hq, heads, dim, vocab)
    ids, uu = fed[:, 0].clone(), u[0].clone()
    outs, tokens = [], []
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        for i in range(5):
            ids.copy_(fed[:, i])
            uu.copy_(u[i])
            lens.fill_(i + 1)
            step(lib, m, c, b, ids, hq, uu, space, side.cuda_stream, bufs)
            outs.append(bufs[2].clone())
            tokens.append(bufs[4].clone())
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            step(lib, m, c, b, ids, hq, uu, space, side.cuda_stream, bufs)
        for i in range(5, n):
            ids.copy_(fed[:, i])
            uu.copy_(u[i])
            lens.fill_(i + 1)
            g.replay()
            outs.append(bufs[2].clone())
            tokens.append(bufs[4].clone())
    side.synchronize()
    assert lib.lcu_check_stream(side.cuda_stream) == 0
    c2 = Cache([n] * seqs, heads, dim, page, seed=7)
    b2 = c2.batch([n] * seqs, [n * i for i in range(seqs + 1)], max_new=n)
    space = torch.empty(max(16, lib.lcu_attention_paged_workspace(c2.pages, b2, hq)), dtype=torch.uint8, device="cuda")
    bufs = buffers(seqs * n, hq, heads, dim, vocab)
    step(lib, m, c2, b2, fed.reshape(-1), hq, u.t().contiguous().reshape(-1), space, None, bufs)
    torch.cuda.synchronize()
    for s in range(seqs):   # the projections are the same sums whatever the row count: small GEMMs run row by row
        for a, o in zip(c.rows(s, n), c2.rows(s, n)):
            assert np.array_equal(a, o)
    one, two = torch.stack(outs, 1).cpu().numpy(), bufs[2].view(seqs, n, -1).cpu().numpy()
    for s in range(seqs):
        k, v = c.kv(s, n)
        ref, size = kvref.attention(bufs[1].view(seqs, n, hq, dim)[s].cpu().numpy(), k, v, list(range(1, n + 1)))
        tol = tolerance(size, dim, np.abs(v).max(), n)
        assert np.max(np.abs(one[s] - ref.reshape(n, -1))) <= tol and np.max(np.abs(two[s] - ref.reshape(n, -1))) <= tol
    logits = bufs[3].view(seqs, n, vocab).cpu().numpy()
    for s in range(seqs):
        got = bufs[4].view(seqs, n)[s].cpu().numpy()
        check_sample(got, logits[s], u[:, s].cpu().numpy())


def test_cache_past_32_bit_offsets(lib):
    """Rows that start more than 2^32 bytes into the cache."""
    dim, page, heads = 256, 4096, 1
    total = 2 ** 32 // (page * dim // 2) + 40   # pages; a page holds 512 KB of codes
    mk = lambda w: torch.empty((total, heads, page, w), dtype=torch.uint8, device="cuda")
    c = Cache([5000, 300], heads, dim, page, seed=1)   # its table only
    c.kc, c.vc, c.ks, c.vs = mk(dim // 2), mk(dim // 2), mk(dim // 16), mk(dim // 16)
    c.table_np = np.array([[total - 1, total - 3], [total - 2, 0]], np.int32)
    c.table = i32(c.table_np)
    c.pages = L.KvPages(ptr(c.kc), ptr(c.vc), ptr(c.ks), ptr(c.vs), total, page, heads, dim, 1.0, 1.0)
    rng = np.random.default_rng(5)
    x = rng.standard_normal((5300, 3, dim)).astype(np.float32)
    b = c.batch([5000, 300], [0, 5000, 5300])
    q = append(lib, c, b, x.reshape(5300, -1), 1)
    ko, vo = torch.zeros((5300, 1, dim), device="cuda"), torch.zeros((5300, 1, dim), device="cuda")
    assert lib.lcu_kv_read_paged(ptr(ko), ptr(vo), c.pages, b, None) == 0
    b = c.batch([5000, 300])
    out = attend(lib, c, b, q[[4999, 5299]], 1)
    assert lib.lcu_check_stream(None) == 0
    at = 0
    for s, n in enumerate((5000, 300)):
        k, v = ko[at:at + n].double().cpu().numpy(), vo[at:at + n].double().cpu().numpy()
        assert np.array_equal(v[:, 0], kvref.values(*kvref.quantise(x[at:at + n, 2])))
        row = q[[4999, 5299]][s].reshape(1, 1, dim)
        ref, size = kvref.attention(row, k, v, [n])
        assert np.max(np.abs(out[s] - ref.reshape(-1))) <= tolerance(size, dim, np.abs(v).max(), n)
        at += n


def test_captured_split_attention_follows_lengths(lib):
    """One captured call, replayed with other lengths (chunks come and go) and other page tables."""
    c = Cache([9000, 3000], 2, 128, 16, seed=2)
    fill_random(c, 21)
    q = np.random.default_rng(3).standard_normal((2, 4, 128)).astype(np.float32)
    t = torch.from_numpy(q.reshape(2, -1)).cuda()
    out = torch.zeros((2, 4 * 128), device="cuda")
    lens = i32([9000, 3000])
    b = L.KvBatch(ptr(c.table), c.table.shape[1], ptr(lens), None, 2, 2, 9000, 1)
    need = lib.lcu_attention_paged_workspace(c.pages, b, 4)
    assert need > 0
    space = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        assert lib.lcu_attention_paged(ptr(out), ptr(t), 512, 4, c.pages, b, ptr(space), need, side.cuda_stream) == 0
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            assert lib.lcu_attention_paged(ptr(out), ptr(t), 512, 4, c.pages, b, ptr(space), need, side.cuda_stream) == 0
        for n in ([9000, 3000], [1, 2999], [0, 17], [8999, 128]):
            lens.copy_(i32(n))
            out.fill_(7.0)
            g.replay()
            side.synchronize()
            got = out.view(2, 4, 128).cpu().numpy()
            for s in range(2):
                k, v = c.kv(s, n[s])
                ref, size = kvref.attention(q[s:s + 1], k, v, [n[s]])
                tol = tolerance(size, 128, np.abs(v).max() if n[s] else 1.0, n[s])
                assert np.max(np.abs(got[s] - ref[0])) <= tol
    assert lib.lcu_check_stream(side.cuda_stream) == 0


def test_captured_cluster_attention_follows_lengths(lib):
    """As above with few keys, whose chunks join within the one launch and need no workspace."""
    c = Cache([1000, 1000, 1000], 2, 64, 16, seed=4)
    fill_random(c, 22)
    q = np.random.default_rng(5).standard_normal((3, 12, 64)).astype(np.float32)
    t = torch.from_numpy(q.reshape(3, -1)).cuda()
    out = torch.zeros((3, 12 * 64), device="cuda")
    lens = i32([1000, 1000, 1000])
    b = L.KvBatch(ptr(c.table), c.table.shape[1], ptr(lens), None, 3, 3, 1000, 1)
    assert lib.lcu_attention_paged_workspace(c.pages, b, 12) == 0
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        call = lambda: lib.lcu_attention_paged(ptr(out), ptr(t), 768, 12, c.pages, b, None, 0, side.cuda_stream)
        assert call() == 0
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            assert call() == 0
        for n in ([1000, 300, 129], [1, 1000, 128], [0, 17, 999], [640, 641, 0]):
            lens.copy_(i32(n))
            out.fill_(7.0)
            g.replay()
            side.synchronize()
            got = out.view(3, 12, 64).cpu().numpy()
            for s in range(3):
                k, v = c.kv(s, n[s])
                ref, size = kvref.attention(q[s:s + 1], k, v, [n[s]])
                assert np.max(np.abs(got[s] - ref[0])) <= tolerance(size, 64, np.abs(v).max() if n[s] else 1.0, n[s])
    assert lib.lcu_check_stream(side.cuda_stream) == 0


def test_two_streams_at_once(lib):
    """Two calls in flight on two streams, each with its own workspace."""
    c = Cache([6000, 4000], 2, 128, 16)
    fill_random(c, 13)
    q = np.random.default_rng(3).standard_normal((2, 8, 128)).astype(np.float32)
    b = c.batch([6000, 4000])
    want = attend(lib, c, b, q, 8)
    need = max(16, lib.lcu_attention_paged_workspace(c.pages, b, 8))
    t = torch.from_numpy(q.reshape(2, -1)).cuda()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [torch.zeros((2, 8 * 128), device="cuda") for _ in streams]
    spaces = [torch.empty(need, dtype=torch.uint8, device="cuda") for _ in streams]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, o, w in zip(streams, outs, spaces):
            assert lib.lcu_attention_paged(ptr(o), ptr(t), 8 * 128, 8, c.pages, b, ptr(w), need, s.cuda_stream) == 0
    torch.cuda.synchronize()
    for o in outs:
        assert np.array_equal(o.cpu().numpy(), want)
