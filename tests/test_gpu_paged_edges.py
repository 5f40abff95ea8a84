"""The paged cache, its attention and the sampler where numbers, lengths and bounds end: units and queries whose product
leaves FP32's range, token ranges that do not fit, weights far below the largest, the longest sequences, prompts."""
import os
import subprocess
import sys

import numpy as np
import pytest

import kvref
import lancius_b200 as L
from test_gpu_paged import (BASE, SHAPE, Cache, append, attend, check_sample, fill_random, i32, lib, ptr, sample, starts,  # noqa: F401
                            tolerance)

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# ---- attention: units ------------------------------------------------------------------------------------------

def check_scores(lib, dim, group, unit, top):
    """Keys in multiples of `unit`, queries of up to `top`, lengths that leave masked keys in the last tile."""
    lens = [777, 33]
    c = Cache(lens, 1, dim, 16, (unit, 1.0), seed=1)
    fill_random(c, dim)
    rng = np.random.default_rng(dim + group)
    q = rng.standard_normal((2, group, dim)).astype(np.float32)
    q = (q / np.abs(q).max() * top).astype(np.float32)
    out = attend(lib, c, c.batch(lens), q, group).reshape(2, group, dim)
    for s, n in enumerate(lens):
        k, v = c.kv(s, n)
        ref, size = kvref.attention(q[s:s + 1], k, v, [n])
        if size < 1e6:
            tol = tolerance(size, dim, np.abs(v).max(), n)
        else:   # scores next to each other differ by far more than their rounding: one weight, held in 22 bits, a
            # truncated sum of its halves and two roundings: 2^-22 + 2^-23 + 2^-23
            x = np.sort(np.einsum("gd,kd->gk", q[s].astype(np.float64), k[:, 0]) / np.sqrt(dim), 1)
            assert np.all(x[:, -1] - x[:, -2] > max(30, 2.0 ** -17 * size))   # the oracle's
            tol = 2.0 ** -21 * np.abs(v).max()
        assert np.max(np.abs(out[s] - ref[0])) <= tol


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 5, 12])
@pytest.mark.parametrize("top", [1e6, 1e7, 1e8, 1e9, 1e15, 1e30])
def test_attention_far_scores(lib, dim, group, top):
    """Scores whose neighbouring FP32 numbers are further apart than the weights reach: one key takes all the weight."""
    check_scores(lib, dim, group, 1.0, top)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 5, 12])
@pytest.mark.parametrize("unit,top", [
    (1e-20, 1e-27), (1e-30, 1e-38),      # scores next to nothing: the mean of the values
    (3e37, 2e-38), (1e-38, 1e37),        # large and small numbers with ordinary products
    (2.0, 1.6e38), (3e37, 1e30)])        # scores past FP32's largest: one key takes all the weight
def test_attention_scores_scale(lib, dim, group, unit, top):
    """Keys of any positive unit, queries of any size."""
    check_scores(lib, dim, group, unit, top)


@pytest.mark.parametrize("lens", [[40], [777], [9000]])   # one chunk, a cluster of them, two launches
@pytest.mark.parametrize("unit", [3e37, 2e-38])
def test_attention_value_unit(lib, lens, unit):
    """Values next to FP32's largest and smallest normal numbers."""
    c = Cache(lens, 1, 128, 16, (1.0, unit), seed=1)
    fill_random(c, 3)
    q = np.random.default_rng(4).standard_normal((1, 2, 128)).astype(np.float32)
    out = attend(lib, c, c.batch(lens), q, 2).reshape(1, 2, 128)
    k, v = c.kv(0, lens[0])
    ref, size = kvref.attention(q, k, v, lens)
    # the last product may fall among the subnormal numbers, which are 2^-149 apart
    assert np.max(np.abs(out - ref)) <= tolerance(size, 128, np.abs(v).max(), lens[0]) + 2.0 ** -150


# ---- token ranges ----------------------------------------------------------------------------------------------

@pytest.mark.parametrize("start,tokens,reported", [
    ([0, 3, 8], 6, True),        # the second sequence's last two rows are not in the arrays
    ([0, 3, 8], 3, True),        # nor any of its rows
    ([-2, 3, 6], 6, True),       # the first one's first two
    ([1, 3, 6], 8, False)])      # rows of no sequence before and behind
def test_token_ranges_past_the_arrays(lib, start, tokens, reported):
    """Rows that the arrays hold have the positions that token_start gives them, in all three calls; the others are reported."""
    hq, heads, dim, lens = 2, 1, 64, [40, 50]
    want = SHAPE if reported else 0
    rows = [(s, t, lens[s] - start[s + 1] + t) for s in range(2) for t in range(max(start[s], 0), min(start[s + 1], tokens))]
    rng = np.random.default_rng(1)
    x = rng.standard_normal((tokens, hq + 2 * heads, dim)).astype(np.float32)
    c = Cache(lens, heads, dim, 16, seed=2)
    fill_random(c, 3)
    b = c.batch(lens, start, tokens=tokens, max_new=5)
    q = append(lib, c, b, x.reshape(tokens, -1), hq).reshape(tokens, hq, dim)
    assert lib.lcu_check_stream(None) == want and lib.lcu_check_stream(None) == 0
    ko, vo = torch.full((tokens, heads, dim), 7.0, device="cuda"), torch.full((tokens, heads, dim), 7.0, device="cuda")
    assert lib.lcu_kv_read_paged(ptr(ko), ptr(vo), c.pages, b, None) == 0
    assert lib.lcu_check_stream(None) == want
    out = attend(lib, c, b, x[:, :hq], hq).reshape(tokens, hq, dim)
    assert lib.lcu_check_stream(None) == want and lib.lcu_check_stream(None) == 0
    held = set()
    for s, t, pos in rows:
        held.add(t)
        k, v = c.kv(s, lens[s])
        ref = kvref.rotate(x[t:t + 1, :hq], [pos], BASE)[0]
        assert np.all(np.abs(q[t] - ref) <= 2.0 ** -23 * np.abs(x[t, :hq]).max())
        assert np.array_equal(v[pos], kvref.values(*kvref.quantise(x[t, hq + heads:])))
        assert np.array_equal(vo[t].cpu().numpy(), v[pos].astype(np.float32))
        ref, size = kvref.attention(x[t:t + 1, :hq], k, v, [pos + 1])
        assert np.max(np.abs(out[t] - ref[0])) <= tolerance(size, dim, np.abs(v).max(), pos + 1)
    for t in set(range(tokens)) - held:
        assert (q[t] == 7.0).all() and (out[t] == 7.0).all() and (ko[t] == 7.0).all()


def test_bad_pages_are_not_other_calls_faults(lib):
    """A bad page is reported by lcu_check_stream, and neither fails nor vanishes in calls that check their own work."""
    c = Cache([40], 1, 64, 16)
    c.table[0, 2] = -1
    x = np.random.default_rng(1).standard_normal((1, 3 * 64)).astype(np.float32)
    append(lib, c, c.batch([40]), x, 1)
    n = 256
    a = torch.randn((n, n), device="cuda")
    y = torch.empty((n, n), device="cuda")
    ctx = lib.lcu_create(0)
    assert ctx
    assert lib.lcu_synchronize(ctx) == 0
    lib.lcu_destroy(ctx)
    assert lib.lcu_matmul(ptr(y), ptr(a), ptr(a), n, n, n, None, 0, 0, None) == 0
    assert lib.lcu_check_stream(None) == SHAPE and lib.lcu_check_stream(None) == 0


def test_words_are_read_only_after_a_launch(lib):
    """A program that never calls the paged cache does not load its kernels for lcu_check_stream, nor wait for its words."""
    code = """
import ctypes as C, torch, lancius_b200 as L
lib = L.load()
for name in ("lcu_kv_fault_addr", "lcu_attn_paged_fault_addr"):
    f = getattr(lib, name)
    f.restype, f.argtypes = C.c_void_p, []
    assert lib.lcu_check_stream(None) == 0 and f() is None, name
from test_gpu_paged import Cache, append, attend
import numpy as np
c = Cache([40], 1, 64, 16)
append(lib, c, c.batch([40]), np.ones((1, 192), np.float32), 1)
assert lib.lcu_kv_fault_addr() and lib.lcu_attn_paged_fault_addr() is None
attend(lib, c, c.batch([40]), np.ones((1, 64), np.float32), 1)
assert lib.lcu_attn_paged_fault_addr()
"""
    here = os.path.dirname(os.path.abspath(__file__))
    env = dict(os.environ, PYTHONPATH=os.pathsep.join((os.path.dirname(here), here)))
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300, env=env)


# ---- the longest sequences, prompts ----------------------------------------------------------------------------

def test_attention_next_to_31_bits(lib):
    """The longest sequence that a table can describe: all of its entries name one of two pages."""
    page, width = 16, (2 ** 31 - 1) // 16
    c = Cache([32], 1, 64, page, spare=0)
    n = page * width - 3
    c.kc.fill_(0x88)                 # keys of zero: equal weights
    c.ks.fill_(0x38)
    c.vs.fill_(0x38)
    c.vc[0].fill_(0x99)              # 1
    c.vc[1].fill_(0x77)              # -1
    table = torch.ones(width, dtype=torch.int32, device="cuda")
    table[:width // 4] = 0
    lens = i32([n])
    b = L.KvBatch(ptr(table), width, ptr(lens), None, 1, 1, 0, 0)
    out = attend(lib, c, b, np.ones((1, 64), np.float32), 1)
    assert lib.lcu_check_stream(None) == 0
    first = page * (width // 4)
    # sums of up to 2^21 chunks of equal weight: every one but the last chunk's is a whole number below 2^24 times 2^15
    assert np.max(np.abs(out - (first - (n - first)) / n)) <= 2.0 ** -20


@pytest.mark.parametrize("dim,heads,group,lens,new", [
    (64, 2, 4, [2500, 100], [2500, 1]),
    (128, 2, 4, [2000, 333, 700, 1], [1500, 1, 1, 1]),          # a prompt beside single tokens
    (256, 1, 2, [1300, 1900], [1, 1200])])
def test_attention_prompts(lib, dim, heads, group, lens, new):
    """More than a thousand new tokens in a call, over several chunks of keys."""
    hq = heads * group
    c = Cache(lens, heads, dim, 32, seed=6)
    fill_random(c, 7)
    q = np.random.default_rng(8).standard_normal((sum(new), hq, dim)).astype(np.float32)
    out = torch.from_numpy(attend(lib, c, c.batch(lens, starts(new), max_new=max(new)), q, hq).reshape(-1, hq, dim)).cuda().double()
    assert lib.lcu_check_stream(None) == 0
    at = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        k, v = (torch.from_numpy(a).cuda().repeat_interleave(group, 1) for a in c.kv(s, n))
        x = torch.from_numpy(q[at:at + m]).cuda().double()
        size = torch.einsum("nhd,khd->nhk", x.abs(), k.abs()).max().item() / dim ** 0.5
        z = torch.einsum("nhd,khd->nhk", x, k) / dim ** 0.5
        limit = torch.arange(n - m, n, device="cuda")
        z = z.masked_fill(torch.arange(n, device="cuda") > limit[:, None, None], -np.inf)
        ref = torch.einsum("nhk,khd->nhd", z.softmax(2), v)
        assert (out[at:at + m] - ref).abs().max().item() <= tolerance(size, dim, v.abs().max().item(), n)
        at += m


def test_attention_workspace_refusals(lib):
    """A call that needs a workspace refuses none, a short one and an unaligned one."""
    c = Cache([9000], 1, 64, 16)
    b = c.batch([9000])
    q = torch.zeros((1, 64), device="cuda")
    need = lib.lcu_attention_paged_workspace(c.pages, b, 1)
    assert need > 0
    space = torch.empty(need + 16, dtype=torch.uint8, device="cuda")
    assert lib.lcu_attention_paged(ptr(q), ptr(q), 64, 1, c.pages, b, ptr(space), need - 1, None) == -9
    assert lib.lcu_attention_paged(ptr(q), ptr(q), 64, 1, c.pages, b, None, need, None) == -2
    assert lib.lcu_attention_paged(ptr(q), ptr(q), 64, 1, c.pages, b, ptr(space) + 8, need, None) == -5


# ---- sampling ----------------------------------------------------------------------------------------------------

def test_sample_small_weights_of_few_candidates(lib):
    """Weights far below the largest count in the draw as the others do: u = 0 takes the first kept index that weighs anything."""
    x = np.full((5, 700), -np.inf, np.float32)
    x[0, [100, 200]] = -40.0, 0.0
    x[1, [3, 4, 600]] = -35.0, -36.0, 0.0
    x[2, [3, 4, 600]] = -35.0, -36.0, 0.0
    x[3] = np.random.default_rng(1).permutation(np.linspace(0, -650, 700))
    x[4, 50:60] = np.linspace(-300, 0, 10)
    u = np.array([0.0, 5e-16, 7e-16, 0.0, 1e-38], np.float32)
    for kw in (dict(top_k=5), dict(top_k=100), dict(top_k=200, min_p=1e-38), dict(top_k=150, top_p=1.0)):
        want = [kvref.draw(x[i], float(u[i]), 1.0, kw["top_k"], 1.0, float(np.float32(kw.get("min_p", 0.0))))[0] for i in range(5)]
        assert want[:3] == [100, 3, 4]
        assert sample(lib, x, u, **kw).tolist() == want


def test_sample_cut_at_2_to_the_minus_1000(lib):
    """Without filters and with one: a logit above 2^-1000 of the largest has a weight, one below has none."""
    t = np.array([0.5, 1.0, 3.0, 0.5, 1.0, 3.0], np.float32)
    x = np.full((6, 700), -np.inf, np.float32)
    x[:, 5] = 0.0
    x[:, 600] = np.where(np.arange(6) < 3, -693.1, -693.2) * t
    for kw in (dict(), dict(min_p=0.0)):
        assert sample(lib, x, np.ones(6, np.float32), temperature=t, **kw).tolist() == [600] * 3 + [5] * 3


@pytest.mark.parametrize("t", [4e35, 5e35, 7e35, 9e35, 2e36, 3e38])
def test_sample_hot_rows_of_far_logits(lib, t):
    """Temperatures at which 693 t is at, or past, FP32's largest number, with logits over all of its range."""
    rng = np.random.default_rng(13)
    x = rng.uniform(-3.4e38, 3.4e38, (6, 5003)).astype(np.float32)
    x[1] = rng.choice(np.array([3.4e38, -3.4e38], np.float32), 5003)
    x[2] = -3.4e38
    x[2, [17, 4000]] = 3.4e38
    x[3, ::2] = -np.inf
    u = np.array([0.2, 0.4, 0.6, 0.8, 0.3, 0.999], np.float32)
    for kw in (dict(), dict(top_k=3), dict(top_p=0.7), dict(min_p=0.2)):
        check_sample(sample(lib, x, u, temperature=t, **kw), x, u, temperature=t, **kw)
