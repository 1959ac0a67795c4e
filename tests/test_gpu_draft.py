"""Steps with drafted tokens on the GPU, against plain 64-bit forms of the same
definitions.

Tolerances, from the arithmetic:
  * a turned key is quantised exactly (but for one value in some 10^12): the
    stored values are equal bit for bit;
  * a turned query is two products and a sum in fp32, of cosines and sines
    rounded once: three roundings of at most 2^-24 of |a| + |b| (times the
    factor), then half a step of its type;
  * the attention as in test_gpu_kv4.py, whose scores, weights and sums it
    shares; 16-bit queries of many columns have K and V themselves rounded to
    fp16 (half a step, 2^-11, of each value): a score is off by |scale| A 2^-11
    more, and V adds once more sum p |v|;
  * verification and kept rows are whole numbers, or bits that move: equal.
"""
import math

import numpy as np
import pytest
import torch

from distcomp_b200 import draft, engine, kv4
from test_gpu_kv4 import H16, check, filled, rows, stored

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
PAGE = 64


@pytest.fixture(autouse=True)
def _quiet():
    yield
    torch.cuda.synchronize()


# -------------------------------------------------------------- rotation ---

def turned(x, pos, freq, factor, interleaved):
    """Rows [n, heads, hd] (numpy, 64 bits) turned by their positions; and |a| + |b| of each value's pair."""
    rot = 2 * len(freq)
    angle = np.fmod(pos.astype(np.longdouble)[:, None] * np.asarray(freq, dtype=np.longdouble), 2 * np.longdouble("3.14159265358979323846264338327950288"))
    c, s = (f(angle.astype(np.float64))[:, None] * factor for f in (np.cos, np.sin))
    a, b = (np.arange(0, rot, 2), np.arange(1, rot, 2)) if interleaved else (np.arange(rot // 2), np.arange(rot // 2, rot))
    y, size = x.copy(), np.abs(x)
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    size[..., a] = size[..., b] = (np.abs(x[..., a]) + np.abs(x[..., b])) * abs(factor)
    return y, size


def half_of(x):
    """fp16 of 64-bit values, rounded once."""
    return np.asarray(x, dtype=np.float64).astype(np.float16)


def held(x):
    """What the cache holds of rows [..., hd] of 64-bit values."""
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        m = np.take_along_axis(b, np.argmax(np.where(np.isnan(b), -1, np.abs(b)), -1)[..., None], -1)
        d = half_of(np.clip(m / -8.0, -65504, 65504)).astype(np.float64)
        fine = np.isfinite(b).all(-1, keepdims=True)
        code = np.where(d != 0, np.clip(np.floor(b / np.where(d != 0, d, 1) + 8.5), 0, 15), 8)
        return np.where(fine, (code - 8) * d, np.nan).reshape(x.shape)


def same(got, want):
    got = got.double().cpu().numpy() if torch.is_tensor(got) else got
    assert np.array_equal(got, want, equal_nan=True), f"{(got != want).sum()} of {want.size} values differ"


def q_check(got, q, pos, freq, factor, interleaved):
    want, size = turned(q.double().cpu().numpy(), pos, freq, factor, interleaved)
    h = torch.finfo(q.dtype).eps / 2
    err = np.abs(got.double().cpu().numpy() - want)
    assert (err <= 3 * 2.0 ** -24 * size + h * np.abs(want) + 1e-40 + (2.0 ** -25 if q.dtype == torch.float16 else 0)).all(), err.max()


def freq_of(rot, base=10000.0):
    return [base ** (-2.0 * i / rot) for i in range(rot // 2)]


@pytest.mark.parametrize("hd,rot", [(32, 32), (64, 64), (96, 96), (128, 128), (128, 64), (96, 20), (64, 2), (32, 0), (128, 90)])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
def test_rows_are_turned_and_stored(hd, rot, interleaved, dtype):
    n_kv, rep, lens, new = 3, 2, [130, 5, 64, 1], [66, 5, 1, 0]
    pool = kv4.KvPool(2, n_kv, hd, 9, 4, 3)
    pool.extend([2, 0, 3, 1], [lens[s] for s in (2, 0, 3, 1)])
    seq, total = [0, 1, 2, 3], sum(new)
    w = rows(hd + rot, total, (rep + 2) * n_kv * hd + 24).to(dtype)       # side by side, an odd distance apart
    q, k, v = (w[:, a * n_kv * hd:b * n_kv * hd].unflatten(1, (-1, hd)) for a, b in ((0, rep), (rep, rep + 1), (rep + 1, rep + 2)))
    before = w.clone()
    rope = draft.Rope(hd, rot=rot, interleaved=interleaved, freq=freq_of(rot), factor=1.25)
    ko, vo = (torch.empty(total, n_kv, hd, device="cuda") for _ in range(2))
    depth = torch.tensor(np.random.default_rng(1).integers(0, 70, total), dtype=torch.int32, device="cuda")
    pos = np.concatenate([np.full(m, lens[s] - m) for s, m in zip(seq, new)]) + depth.cpu().numpy()
    out = pool.append_rope(1, rope, q, k, v, seq, new, depth=depth, k_out=ko, v_out=vo)
    assert torch.equal(w, before)
    q_check(out, q, pos, freq_of(rot), 1.25, interleaved)
    wk, wv = held(turned(k.double().cpu().numpy(), pos, freq_of(rot), 1.25, interleaved)[0]), held(v.double().cpu().numpy())
    same(ko, wk)
    same(vo, wv)
    r = 0
    for s, m in zip(seq, new):
        gk, gv = pool.read(1, s, lens[s] - m, m)
        same(gk.astype(np.float64), wk[r:r + m])
        same(gv.astype(np.float64), wv[r:r + m])
        r += m
    for s in range(4):                                # the other layer, and what lay before
        assert not np.any(pool.read(0, s)[0]) and not np.any(pool.read(1, s, 0, lens[s] - new[s])[1])


def test_rows_like_an_append_when_nothing_turns():
    """Position 0, or no turning dimensions: the bytes of append()."""
    hd, n_kv, n = 128, 8, 300
    k, v = rows(1, n, n_kv, hd), rows(2, n, n_kv, hd)
    a, b = kv4.KvPool(1, n_kv, hd, 10, 2, 5), kv4.KvPool(1, n_kv, hd, 10, 2, 5)
    for p in (a, b):
        p.extend([0, 1], [n, n])
    a.append(0, torch.cat((k, k)), torch.cat((v, v)), [0, 1], [n, n])
    b.append_rope(0, draft.Rope(hd, rot=0, freq=[]), None, k, v, [0], [n])
    b.append_rope(0, draft.Rope(hd), None, k, v, [1], [n], depth=torch.zeros(n, dtype=torch.int32, device="cuda"))
    ka, kb = a.read(0, 0)[0], b.read(0, 0)[0]
    assert np.array_equal(ka, kb) and np.array_equal(a.read(0, 1)[1], b.read(0, 1)[1])


def test_rows_at_far_positions():
    """Angles of positions past 10^5, and past 2^31 by their depth."""
    hd, n_kv, n = 64, 2, 40
    pool = kv4.KvPool(1, n_kv, hd, 3200, 1, 3200)
    pool.extend([0], [200000])
    rope = draft.Rope(hd, base=500000.0)
    f = freq_of(hd, 500000.0)
    q, k, v = rows(1, n, 4, hd), rows(2, n, n_kv, hd), rows(3, n, n_kv, hd)
    depth = torch.arange(n, dtype=torch.int32, device="cuda")
    depth[20:] += 2147483000
    depth[30:] *= -1
    pos = 200000 - n + depth.cpu().numpy().astype(np.int64)
    out = pool.append_rope(0, rope, q, k, v, [0], [n], depth=depth)
    # the frequencies are those of 64 bits: past 2^31 their own rounding, 2^-53 of the angle, shows in the last digits
    q_check(out, q, pos, f, 1.0, False)
    same(pool.read(0, 0, 200000 - n, 20)[0].astype(np.float64), held(turned(k.double().cpu().numpy(), pos, f, 1.0, False)[0])[:20])


def test_rows_in_place_without_queries_and_misaligned():
    hd, n_kv, n = 64, 3, 9
    rope, f = draft.Rope(hd, interleaved=True), freq_of(hd)
    for dtype in TYPES:
        pool = kv4.KvPool(1, n_kv, hd, 3, 1, 3)
        pool.extend([0], [n])
        flat = rows(4, n * 12 * hd + 1).to(dtype)[1:].view(n, 12, hd)    # one element off
        q, k, v = flat[:, :6], flat[:, 6:9], flat[:, 9:]
        old = flat.clone()
        assert pool.append_rope(0, rope, q, k, v, [0], [n], q_out=q) is q
        q_check(q, old[:, :6], np.arange(n), f, 1.0, True)
        assert torch.equal(flat[:, 6:], old[:, 6:])
        want = held(turned(old[:, 6:9].double().cpu().numpy(), np.arange(n), f, 1.0, True)[0])
        same(pool.read(0, 0)[0].astype(np.float64), want)
        assert pool.append_rope(0, rope, None, k, v, [0], [n]) is None
        same(pool.read(0, 0)[0].astype(np.float64), want)


def test_rows_of_unusual_values():
    """Zeros, tiny and huge rows, infinities and NaN: each block by itself; ties between a value and its negative."""
    hd, n_kv = 64, 1
    k = rows(1, 8, n_kv, hd)
    k[0] = 0.0
    k[1] = 1e-9
    k[2, 0, 40] = 1e30
    k[3, 0, 3] = math.inf                             # its partner is dimension 35: both blocks
    k[4, 0, 50] = math.nan
    k[5] = 0.0
    k[5, 0, 7], k[5, 0, 9] = -3.0, 3.0
    k[6, 0, :32] = 2.0
    k[6, 0, 32:] = -2.0
    v = k.clone()
    pool = kv4.KvPool(1, n_kv, hd, 2, 1, 2)
    pool.extend([0], [8])
    depth = torch.tensor([0, 0, 5, 9, 9, 0, 0, 3], dtype=torch.int32, device="cuda")
    pool.append_rope(0, draft.Rope(hd), None, k, v, [0], [8], depth=depth)
    with np.errstate(invalid="ignore"):
        want = held(turned(k.double().cpu().numpy(), depth.cpu().numpy(), freq_of(hd), 1.0, False)[0])
    gk, gv = pool.read(0, 0)
    same(gk.astype(np.float64), want)
    same(gv.astype(np.float64), held(v.double().cpu().numpy()))


def test_rows_of_more_sequences_than_one_launch_lists():
    hd, n_kv, n = 32, 1, 1500
    new = [(i * 7) % 3 for i in range(n)]
    pool = kv4.KvPool(1, n_kv, hd, n, n, 1)
    pool.extend(np.arange(n), [3] * n)
    total = sum(new)
    q, k, v = rows(1, total, 2, hd), rows(2, total, n_kv, hd), rows(3, total, n_kv, hd)
    order = np.random.default_rng(5).permutation(n).astype(np.int32)
    out = pool.append_rope(0, draft.Rope(hd), q, k, v, order, new)
    pos = np.concatenate([3 - m + np.arange(m) for m in new])
    q_check(out, q, pos, freq_of(hd), 1.0, False)
    want = held(turned(k.double().cpu().numpy(), pos, freq_of(hd), 1.0, False)[0])
    r0 = np.cumsum([0] + new)
    for i in (0, 1, 2, 500, 1023, 1024, 1025, 1498, 1499):
        if new[i]:
            same(pool.read(0, int(order[i]), 3 - new[i], new[i])[0].astype(np.float64), want[r0[i]:r0[i + 1]])


# ------------------------------------------------------------------ tree ---

def random_tree(r, n):
    return [-1 if j == 0 or r.random() < 0.1 else int(r.integers(max(0, j - 6), j)) for j in range(n)]


def tree_check(pool, vals, q, seq, new, masks, out, scale=None, every=1):
    """masks: per sequence a list of Python ints.  every: one in so many heads is looked at."""
    H, hd = q.shape[1], q.shape[2]
    half, wide = torch.finfo(q.dtype).eps / 2, q.dtype == torch.float32
    scale = hd ** -0.5 if scale is None else scale
    hw, extra, hk = (0.0, 0.0, 0.0) if wide else (2 * H16, 2.0 ** -24, H16)
    qn, r0 = q.double().cpu().numpy(), 0
    for s, m, mk in zip(seq, new, masks):
        k, v = vals[s]
        n, base = len(k), len(k) - m
        seen = np.ones((m, n), bool)
        for j in range(m):
            seen[j, base:] = [mk[j] >> t & 1 for t in range(m)]
        want, tol = np.zeros((m, H, hd)), np.zeros((m, H, hd))
        for h in range(0, H, every):
            kh, vh = k[:, h // (H // k.shape[1])], v[:, h // (H // k.shape[1])]
            for j in range(m):
                see = seen[j]
                if not see.any():
                    continue
                qj, kk, vv = qn[r0 + j, h], kh[see], vh[see]
                with np.errstate(invalid="ignore"):
                    sc = kk @ qj * scale
                    A = np.max(np.abs(kk) @ np.abs(qj))
                    if np.isnan(sc).any():
                        want[j, h] = np.nan
                        continue
                    ds = abs(scale) * A * (2.0 ** -23 * (hd / 2 + 16) + hk) + 2.0 ** -20
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    want[j, h] = p @ vv
                    fin = np.nan_to_num(np.abs(vv))
                    vmax = fin.max()
                    tol[j, h] = vmax * (2 * ds + 2.0 ** -23 * (n / 16 + 64) + extra) + hw * (p @ fin) + half * np.nan_to_num(np.abs(want[j, h]))
        check(out[r0:r0 + m, ::every], want[:, ::every], tol[:, ::every])
        r0 += m
    assert r0 == q.shape[0]


def make(seed, new, chain=False):
    r = np.random.default_rng(seed)
    masks = []
    for n in new:
        m = []
        for j, p in enumerate(list(range(-1, n - 1)) if chain else random_tree(r, n)):
            m.append((m[p] if p >= 0 else 0) | 1 << j)
        masks.append(m)
    flat = np.array([x for m in masks for x in m], dtype=np.uint64).view(np.int64)
    return masks, torch.from_numpy(flat).cuda()


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rep", [1, 3, 4, 8])
def test_tree_shapes(hd, dtype, rep):
    """Lengths and trees around the borders of units, pages and tiles; sequences without rows among them."""
    n_kv, lens, new = 2, [1, 40, 64, 65, 130, 200, 97, 3], [1, 9, 2, 17, 5, 33, 0, 3]
    pool, vals = filled(n_kv, hd, lens, hd + rep)
    masks, mask = make(hd * rep, new)
    q = rows(7, sum(new), n_kv * rep, hd, spread=1.5).to(dtype)
    out = torch.full((sum(new) + 1, n_kv * rep, hd), 77.0, dtype=dtype, device="cuda")
    got = pool.attend_tree(0, q, list(range(8)), new, mask, out=out[:-1])
    tree_check(pool, vals, q, range(8), new, masks, got)
    assert (out[-1] == 77).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_kv,rep,lens,new", [(1, 1, [5000], [64]), (8, 4, [4097], [6]), (2, 8, [3000, 64, 2222], [64, 64, 1]), (4, 1, [30000], [3]),
                                               (1, 16, [10001, 9], [40, 9]), (8, 5, [1000] * 3, [7, 7, 7])])
def test_tree_long(dtype, n_kv, rep, lens, new):
    """Rows that several CTAs share, every width of a group of tiles."""
    hd = 128
    pool, vals = filled(n_kv, hd, lens, 11)
    masks, mask = make(5, new)
    q = rows(9, sum(new), n_kv * rep, hd, spread=1.5).to(dtype)
    got = pool.attend_tree(0, q, list(range(len(new))), new, mask)
    tree_check(pool, vals, q, range(len(new)), new, masks, got)
    # the same bits again, from another stream's workspace, and from a given one
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        again = pool.attend_tree(0, q, list(range(len(new))), new, mask)
    s.synchronize()
    ws = pool.tree_workspace()
    ws.fill_(255)                                     # whatever it held
    third = pool.attend_tree(0, q, list(range(len(new))), new, mask, ws=ws)
    assert torch.equal(got, again) and torch.equal(got, third)


@pytest.mark.parametrize("hd,rep", [(128, 4), (128, 7), (64, 8), (64, 4)])
@pytest.mark.parametrize("dtype", TYPES[1:])
def test_tree_of_many_columns(hd, rep, dtype):
    """16-bit queries of up to 512 columns a KV head (the tensor-memory kernel): lengths around the borders of its units."""
    n_kv, lens, new = 5, [1, 63, 64, 65, 127, 128, 129, 200, 256, 257, 383, 700], [1, 40, 64, 33, 17, 64, 2, 20, 64, 64, 0, 31]
    pool, vals = filled(n_kv, hd, lens, hd + rep)
    masks, mask = make(hd * rep, new)
    q = rows(7, sum(new), n_kv * rep, hd, spread=1.5).to(dtype)
    out = torch.full((sum(new) + 1, n_kv * rep, hd), 77.0, dtype=dtype, device="cuda")
    got = pool.attend_tree(0, q, list(range(len(lens))), new, mask, out=out[:-1])
    tree_check(pool, vals, q, range(len(lens)), new, masks, got)
    assert (out[-1] == 77).all()


@pytest.mark.parametrize("n_kv,rep,lens,new,dtype", [(8, 5, [1000] * 3, [7] * 3, torch.float16), (8, 8, [2000] * 8, [16] * 8, torch.bfloat16),
                                                     (8, 4, [300] * 40, [24] * 40, torch.float16), (2, 4, [5000] * 5, [6] * 5, torch.float32)])
def test_tree_gives_the_same_bits_again(n_kv, rep, lens, new, dtype):
    """Many rows a CTA, rows shared by CTAs: no order of the warps shows."""
    pool, _ = filled(n_kv, 128, lens, 11)
    _, mask = make(5, new)
    q = rows(9, sum(new), n_kv * rep, 128, spread=1.5).to(dtype)
    seq = list(range(len(new)))
    want = pool.attend_tree(0, q, seq, new, mask)
    for _ in range(60):
        assert torch.equal(pool.attend_tree(0, q, seq, new, mask), want)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("big", [2.0 ** 14, 60000.0, 500000.0])
def test_tree_of_large_values(dtype, big):
    """Keys and values past fp16's range (the cache holds up to 8 * 65504), from some unit on."""
    hd, n_kv, rep, lens, new = 128, 6, 8, [700, 900, 130, 400], [20, 16, 9, 24]
    pool, vals = filled(n_kv, hd, lens, 3)
    masks, mask = make(8, new)
    k, v = rows(1, 160, n_kv, hd), rows(2, 160, n_kv, hd)
    v[3, 1, 40] = v[90, :, 7] = -big
    k[30, 2, 5] = big
    v[110, 3] = big
    pool.append(0, k[:100], v[:100], [1], [100])
    pool.append(0, k[100:], v[100:], [2], [60])
    vals = [tuple(x.astype(np.float64) for x in pool.read(0, s)) for s in range(4)]
    q = (rows(5, sum(new), n_kv * rep, hd) * 1e-3).to(dtype)
    tree_check(pool, vals, q, range(4), new, masks, pool.attend_tree(0, q, [0, 1, 2, 3], new, mask))


@pytest.mark.parametrize("dtype", TYPES)
def test_tree_without_masks_is_causal(dtype):
    hd, n_kv, rep, lens, new = 64, 2, 4, [500, 20, 64], [20, 20, 1]
    pool, vals = filled(n_kv, hd, lens, 3)
    masks, mask = make(0, new, chain=True)
    q = rows(2, sum(new), n_kv * rep, hd).to(dtype)
    a, b = pool.attend_tree(0, q, [0, 1, 2], new), pool.attend_tree(0, q, [0, 1, 2], new, mask)
    assert torch.equal(a, b)
    tree_check(pool, vals, q, range(3), new, masks, a)
    # one row a sequence: what attend gives, within both tolerances
    q = rows(3, 3, n_kv * rep, hd).to(dtype)
    tree_check(pool, vals, q, range(3), [1, 1, 1], [[1]] * 3, pool.attend(0, q, [0, 1, 2]))
    tree_check(pool, vals, q, range(3), [1, 1, 1], [[1]] * 3, pool.attend_tree(0, q, [0, 1, 2], [1, 1, 1]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_kv,rep", [(2, 2), (40, 3)])
def test_tree_masks_of_any_bits(dtype, n_kv, rep):
    """Rows that see nothing, only others, every bit of the word; sequences of drafts alone."""
    hd, lens, new = 128, [64, 64, 7, 100], [64, 64, 7, 4]
    pool, vals = filled(n_kv, hd, lens, 3)
    r = np.random.default_rng(4)
    masks = [[int(x) for x in r.integers(0, 2 ** 64, m, dtype=np.uint64)] for m in new]
    masks[0][0] = masks[0][9] = masks[2][6] = 0
    masks[0][63] = 1 << 63
    masks[1][1] = 2 ** 64 - 1
    masks[3] = [0, 1 << 63, 0xF0, 8]                  # bits behind the last row have no effect
    mask = torch.from_numpy(np.array([x for m in masks for x in m], dtype=np.uint64).view(np.int64)).cuda()
    q = rows(2, sum(new), n_kv * rep, hd).to(dtype)
    out = pool.attend_tree(0, q, [0, 1, 2, 3], new, mask)
    tree_check(pool, vals, q, range(4), new, masks, out)
    assert not out[0].any() and not out[9].any() and not out[64 + 64 + 6].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,n_kv,rep", [(64, 2, 2), (128, 2, 8), (128, 9, 8), (64, 9, 8)])
def test_tree_values_that_are_not_finite(dtype, hd, n_kv, rep):
    """NaN keys and values: without effect where they are not seen, NaN where they are, however little they weigh."""
    lens, new = [150, 2000], [12, 20]
    pool, vals = filled(n_kv, hd, lens, 3)
    masks, mask = make(8, new)
    vals = [list(v) for v in vals]
    k, v = (torch.from_numpy(np.concatenate([vals[0][j][-12:], vals[1][j][-20:]])).float().cuda() for j in (0, 1))
    # draft 3 of sequence 0: a NaN key of head 0; draft 5: a NaN value of head 1, block 1; draft 7 of sequence 1: both of head 1
    k[3, 0, 1] = v[5, 1, 40] = k[12 + 7, 1, 0] = v[12 + 7, 1, hd - 1] = math.nan
    v[12 + 9, 0, 33] = math.inf
    v[4, 1] = 60000.0                                 # large where it is not seen: no other row's digits
    pool.append(0, k, v, [0, 1], new)
    a = [pool.read(0, s) for s in (0, 1)]
    vals = [(x.astype(np.float64), y.astype(np.float64)) for x, y in a]
    assert np.isnan(vals[0][0]).any() and np.isnan(vals[1][1]).any()
    q = rows(5, sum(new), n_kv * rep, hd, spread=1.5).to(dtype)
    out = pool.attend_tree(0, q, [0, 1], new, mask)
    tree_check(pool, vals, q, range(2), new, masks, out)
    assert torch.isnan(out).any() and torch.isfinite(out[:3]).all()
    # a NaN or infinite query: its own rows alone
    q[2, 1, 5] = math.nan
    q[20, 0, 3] = math.inf
    two = pool.attend_tree(0, q, [0, 1], new, mask)
    assert torch.isnan(two[2, 1]).all() and torch.isnan(two[20, 0]).all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[2, 1] = keep[20, 0] = False
    assert torch.equal(torch.nan_to_num(out[keep]), torch.nan_to_num(two[keep]))


def test_tree_of_a_cached_nan():
    """Seen by every row of its head, and of no other sequence's."""
    hd, n_kv = 128, 2
    pool, vals = filled(n_kv, hd, [300, 300], 3)
    k, v = rows(1, 300, n_kv, hd), rows(2, 300, n_kv, hd)
    k[17, 1, 9] = math.nan
    v[250, 0, 70] = math.nan
    pool.append(0, k, v, [0], [300])
    masks, mask = make(3, [5, 5])
    q = rows(3, 10, 8, hd)
    out = pool.attend_tree(0, q, [0, 1], [5, 5], mask)
    vals[0] = tuple(x.astype(np.float64) for x in pool.read(0, 0))
    tree_check(pool, vals, q, range(2), [5, 5], masks, out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n_kv,rep", [(1, 4), (12, 6)])
def test_tree_peaked_flat_and_scaled(dtype, n_kv, rep):
    hd, lens, new = 128, [900, 700], [9, 8]
    pool, vals = filled(n_kv, hd, lens, 3)
    masks, mask = make(3, new)
    q = rows(3, 17, n_kv * rep, hd)
    q[0] *= 40.0
    q[1] *= 1e-6
    q[2] = 0.0
    q[3] *= 1e-20 if dtype == torch.float32 else 1e-4
    q[4] *= 300.0
    q = q.to(dtype)
    for scale in (None, 0.0, -0.3, 1e-3):
        out = pool.attend_tree(0, q, [0, 1], new, mask, scale=scale)
        tree_check(pool, vals, q, range(2), new, masks, out, scale=scale)


# Calls of many columns, whose 16-bit queries the kernel on tensor memory takes.
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_values_that_are_not_finite_among_many(dtype, hd):
    n_kv, rep, lens, new = 8, 8, [150, 2000, 1500, 700, 900], [12, 20, 64, 33, 16]
    pool, vals = filled(n_kv, hd, lens, 3)
    masks, mask = make(8, new)
    k, v = (torch.from_numpy(np.concatenate([x[j][-m:] for x, m in zip(vals, new)])).float().cuda() for j in (0, 1))
    k[3, 0, 1] = v[5, 7, 40] = k[12 + 7, 1, 0] = v[12 + 7, 1, hd - 1] = v[32 + 50, 6, 3] = math.nan
    v[12 + 9, 0, 33] = math.inf
    v[4, 1] = v[32 + 9, 3] = 60000.0
    pool.append(0, k, v, range(5), new)
    vals = [tuple(x.astype(np.float64) for x in pool.read(0, s)) for s in range(5)]
    q = rows(5, sum(new), n_kv * rep, hd, spread=1.5).to(dtype)
    out = pool.attend_tree(0, q, range(5), new, mask)
    tree_check(pool, vals, q, range(5), new, masks, out, every=13)
    q[2, 1, 5] = math.nan
    q[100, 0, 3] = math.inf
    two = pool.attend_tree(0, q, range(5), new, mask)
    assert torch.isnan(two[2, 1]).all() and torch.isnan(two[100, 0]).all()
    keep = torch.ones_like(out, dtype=torch.bool)
    keep[2, 1] = keep[100, 0] = False
    assert torch.equal(torch.nan_to_num(out[keep]), torch.nan_to_num(two[keep]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_masks_of_any_bits_among_many(dtype, hd):
    n_kv, rep, lens, new = 8, 8, [64, 64, 7, 100, 1500, 2000], [64, 64, 7, 4, 64, 33]
    pool, vals = filled(n_kv, hd, lens, 3)
    r = np.random.default_rng(4)
    masks = [[int(x) for x in r.integers(0, 2 ** 64, m, dtype=np.uint64)] for m in new]
    masks[0][0] = masks[0][9] = masks[2][6] = masks[4][63] = 0
    masks[0][63] = 1 << 63
    masks[1][1] = 2 ** 64 - 1
    masks[3] = [0, 1 << 63, 0xF0, 8]                  # bits behind the last row have no effect
    mask = torch.from_numpy(np.array([x for m in masks for x in m], dtype=np.uint64).view(np.int64)).cuda()
    q = rows(2, sum(new), n_kv * rep, hd).to(dtype)
    out = pool.attend_tree(0, q, range(6), new, mask)
    tree_check(pool, vals, q, range(6), new, masks, out, every=13)
    assert not out[0].any() and not out[9].any() and not out[64 + 64 + 6].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_tree_peaked_flat_and_scaled_among_many(dtype, hd):
    n_kv, rep, lens, new = 9, 8, [900, 2100, 1300], [64, 40, 33]
    pool, vals = filled(n_kv, hd, lens, 3)
    masks, mask = make(3, new)
    q = rows(3, sum(new), n_kv * rep, hd)
    q[0] *= 40.0
    q[1] *= 1e-6
    q[2] = 0.0
    q[3] *= 1e-20 if dtype == torch.float32 else 1e-4
    q[70] *= 300.0
    q = q.to(dtype)
    for scale in (None, 0.0, -0.3, 1e-3):
        out = pool.attend_tree(0, q, range(3), new, mask, scale=scale)
        tree_check(pool, vals, q, range(3), new, masks, out, scale=scale, every=23)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n_kv,rep,n,len_,new", [(8, 4, 17, 300, 64), (8, 8, 17, 100, 16), (8, 8, 1, 4000, 16), (8, 4, 8, 100, 64), (8, 4, 1, 900, 6), (7, 3, 11, 500, 20)])
def test_tree_rows_of_one_length(dtype, hd, n_kv, rep, n, len_, new):
    """Whole rows, as many a CTA, and few rows in many parts, joined in blocks of fewer columns."""
    pool, vals = filled(n_kv, hd, [len_] * n, 7)
    masks, mask = make(9, [new] * n)
    q = rows(6, new * n, n_kv * rep, hd, spread=1.5).to(dtype)
    out = torch.full((new * n + 1, n_kv * rep, hd), 77.0, dtype=dtype, device="cuda")
    tree_check(pool, vals, q, range(n), [new] * n, masks, pool.attend_tree(0, q, range(n), [new] * n, mask, out=out[:-1]), every=11)
    assert (out[-1] == 77).all()


def test_tree_strided_misaligned_and_many():
    hd, n_kv, rep, n = 64, 2, 3, 130
    r = np.random.default_rng(2)
    lens = [int(x) for x in r.integers(1, 150, n)]
    new = [int(min(l, x)) for l, x in zip(lens, r.integers(0, 12, n))]
    pool, vals = filled(n_kv, hd, lens, 3)
    order = [int(x) for x in r.permutation(n)]
    new = [new[s] for s in order]
    masks, mask = make(3, new)
    total = sum(new)
    for dtype in TYPES:
        w = rows(4, total * 9 * hd + 1).to(dtype)[1:].view(total, 9, hd)
        out = torch.full((total * 8 * hd + 1,), 5.0, dtype=dtype, device="cuda")[1:].view(total, 8, hd)
        pool.attend_tree(0, w[:, 1:7], order, new, mask, out=out[:, 2:])
        tree_check(pool, vals, w[:, 1:7], order, new, masks, out[:, 2:])
        assert (out[:, :2] == 5).all()


def test_tree_of_more_sequences_than_one_launch_lists():
    hd, n_kv, n = 32, 1, 1300
    new = [i % 4 for i in range(n)]
    pool, vals = filled(n_kv, hd, [4 + i % 5 for i in range(n)], 3)
    masks, mask = make(3, new)
    q = rows(4, sum(new), 2, hd)
    out = pool.attend_tree(0, q, None, new, mask)
    tree_check(pool, vals, q, range(n), new, masks, out)


def test_tree_beyond_32_bits():
    """Pages further than 4 GB into the layer."""
    hd, n_kv = 128, 8
    far = (5 << 30) // kv4.page_bytes(n_kv, hd)
    pool = kv4.KvPool(1, n_kv, hd, far + 4, 2, far)
    pool.extend([0, 1], [far * PAGE, 100])
    k, v, q = rows(1, 100, n_kv, hd), rows(2, 100, n_kv, hd), rows(3, 6, 16, hd)
    f = freq_of(hd)
    ko = torch.empty_like(k)
    pool.append_rope(0, draft.Rope(hd), None, k, v, [1], [100], k_out=ko, v_out=torch.empty_like(v))
    assert pool.pages(1) == [far, far + 1]
    vals = {1: (held(turned(k.double().cpu().numpy(), np.arange(100), f, 1.0, False)[0]), stored(v))}
    same(ko, vals[1][0])
    masks, mask = make(3, [6])
    tree_check(pool, vals, q, [1], [6], masks, pool.attend_tree(0, q, [1], [6], mask))
    pool.keep([1], [40], [[0, 5, 39]])
    a = pool.read(0, 1, 60, 3)
    same(a[0].astype(np.float64), vals[1][0][[60, 65, 99]])


def test_tree_captured_follows_the_lengths():
    """append_rope and attend_tree in a graph, replayed as the sequences grow; two graphs with workspaces of their own."""
    hd, n_kv, rep, new = 128, 2, 4, [5, 1, 12]
    lens, total = [60, 1, 500], 18
    pool = kv4.KvPool(1, n_kv, hd, 60, 3, 30)
    pool.extend([0, 1, 2], lens)
    kd, vd = rows(1, sum(lens), n_kv, hd), rows(2, sum(lens), n_kv, hd)
    pool.append(0, kd, vd, [0, 1, 2], lens)
    parents = [[-1, 0, 0, 1, 1], [-1], list(range(-1, 11))]
    depth, mask = draft.tree(parents)
    masks = [[int(x) & (2 ** 64 - 1) for x in draft.tree(p, device=None)[1]] for p in parents]
    rope, f = draft.Rope(hd), freq_of(hd)
    q, k, v = (torch.zeros(total, h, hd, device="cuda") for h in (rep * n_kv, n_kv, n_kv))
    outs, graphs = [torch.zeros_like(q) for _ in range(2)], []
    pool.extend([0, 1, 2], new)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    wss = [pool.tree_workspace() for _ in range(2)]
    with torch.cuda.stream(s):
        with pytest.raises(engine.EngineError, match="workspace of its own"):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=s):
                pool.attend_tree(0, q, [0, 1, 2], new, mask)
    torch.cuda.synchronize()
    for out, ws in zip(outs, wss):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            turned_q = pool.append_rope(0, rope, q, k, v, [0, 1, 2], new, depth=depth)
            pool.attend_tree(0, turned_q, [0, 1, 2], new, mask, out=out, ws=ws)
        graphs.append((g, turned_q))
    for step in range(4):
        q.copy_(rows(10 + step, *q.shape)), k.copy_(rows(20 + step, *k.shape)), v.copy_(rows(30 + step, *v.shape))
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        vals = [tuple(x.astype(np.float64) for x in pool.read(0, i)) for i in range(3)]
        held_now = [pool.length(i) for i in range(3)]
        pos = np.concatenate([h - m + np.array(draft.tree(p, device=None)[0]) for h, m, p in zip(held_now, new, parents)])
        wk = held(turned(k.double().cpu().numpy(), pos, f, 1.0, False)[0])
        r = np.cumsum([0] + new)
        for i in range(3):
            same(vals[i][0][-new[i]:], wk[r[i]:r[i + 1]])
        for (g, tq), out in zip(graphs, outs):
            tree_check(pool, vals, tq, range(3), new, masks, out)
        pool.keep([0, 1, 2], new, [[0, 2], [0], list(range(step, 12))])
        pool.extend([0, 1, 2], [n + (200 if step == 1 and i == 0 else 0) for i, n in enumerate(new)])
        if step == 1:
            pool.append(0, rows(50, 205, n_kv, hd), rows(51, 205, n_kv, hd), [0], [205])


def test_tree_on_two_streams():
    hd, n_kv, rep = 128, 2, 4
    pool, vals = filled(n_kv, hd, [3000, 2500], 3)
    masks, mask = make(3, [16, 16])
    q = rows(4, 32, n_kv * rep, hd)
    want = pool.attend_tree(0, q, [0, 1], [16, 16], mask)
    streams = [torch.cuda.Stream() for _ in range(20)]
    before = pool.info().device_bytes
    outs = []
    for s in streams:                                 # more than the pool keeps workspaces for
        s.wait_stream(torch.cuda.current_stream())
        outs.append(torch.zeros_like(q))
        pool.attend_tree(0, q, [0, 1], [16, 16], mask, out=outs[-1], stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    assert pool.info().device_bytes <= before + 16 * pool.tree_ws_bytes()
    pool.close()


def clear_check(q, kn, vn, seen, scale, out, hk):
    """Rows whose largest score is clear of all rounding show its value: weights are off by 2^-11, values by as much
    where they are rounded to fp16, and the output is rounded once.  All rows are finite.  seen [rows, positions]."""
    R, H, hd = q.shape
    rep = H // kn.shape[1]
    k, v = (torch.from_numpy(np.ascontiguousarray(x)).cuda().repeat_interleave(rep, 1) for x in (kn, vn))
    assert torch.isfinite(out).all()
    sc = torch.einsum("rhd,thd->rht", q.double(), k) * scale
    size = (torch.einsum("rhd,thd->rht", q.double().abs(), k.abs()) * abs(scale)).masked_fill(~seen[:, None], 0.0).amax(-1)
    two = sc.masked_fill(~seen[:, None], -math.inf).topk(2, -1)
    clear = two.values[..., 0] - two.values[..., 1] > 2 * size * (2.0 ** -23 * (hd / 2 + 16) + hk) + 64
    want = v[two.indices[..., 0], torch.arange(H, device="cuda")[None]]
    half, wide = torch.finfo(q.dtype).eps / 2, q.dtype == torch.float32
    tol = (half + (2.0 ** -20 if wide else 2 * H16)) * want.abs() + 2.0 ** -20
    err = ((out.double() - want).abs() / tol).amax(-1)[clear]
    assert clear.sum() > 0.2 * clear.numel() and err.max() <= 1.0, (clear.sum(), err.max())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,count", [(64, 8), (128, 8), (32, 2), (96, 2), (128, 1)])
@pytest.mark.parametrize("top", [18, 20, 24, 27, 30])
def test_tree_of_large_scores(dtype, hd, count, top):
    """Scores around 2^top and beyond, past which a float has no room for anything beside them."""
    n, m, n_kv, rep = 150 if count > 1 else 6000, 64, 8, 8
    pool = kv4.KvPool(1, n_kv, hd, (n // PAGE + 1) * count, count, n // PAGE + 1)
    pool.extend(range(count), [n] * count)
    k, v, q = rows(1, n, n_kv, hd), rows(2, n, n_kv, hd), rows(5, m * count, n_kv * rep, hd).to(dtype)
    k[70] *= 2.0 ** 12
    k[-30] *= 2.0 ** 12                               # of the drafts too
    for s in range(count):
        pool.append(0, k, v, [s], [n])
    kn, vn = stored(k), stored(v)
    masks, mask = make(3, [m] * count)
    seen = torch.ones(m * count, n, dtype=torch.bool)
    for i, x in enumerate(np.array(masks, dtype=np.uint64).reshape(-1)):
        seen[i, n - m:] = torch.tensor([bool(int(x) >> t & 1) for t in range(m)])
    size = torch.einsum("rhd,hd->rh", q.double(), torch.from_numpy(kn[70]).cuda().repeat_interleave(rep, 0)).abs().median()
    scale = 2.0 ** top / float(size)
    got = pool.attend_tree(0, q, range(count), [m] * count, mask, scale=scale)
    clear_check(q, kn, vn, seen.cuda(), scale, got, 0.0 if dtype == torch.float32 else H16)
    if dtype != torch.float32 and count == 8:         # the other kernel, on the codes themselves
        engine.inject_tree_registers()
        other = pool.attend_tree(0, q, range(count), [m] * count, mask, scale=scale)
        assert not torch.equal(got, other)
        clear_check(q, kn, vn, seen.cuda(), scale, other, 0.0)


# ---------------------------------------------------------------- verify ---

def verify_plain(logits, tokens, parents, n_row, u, u_next, temp, q):
    """The definition, in 64 bits."""
    kept, n_kept, nxt, r0 = [], [], [], 0
    for i, n in enumerate(n_row):
        if n == 0:
            n_kept.append(0), nxt.append(-1)
            continue

        def target(j):
            x = logits[r0 + j]
            if np.isnan(x).any() or (x == np.inf).any() or not (x > -np.inf).any():
                return None
            if not temp[i] > 0:
                f = np.zeros(len(x))
                f[np.argmax(x)] = 1.0
                return f
            e = np.exp(np.where(x > -np.inf, x - x.max(), -np.inf) / temp[i])
            return e / e.sum()

        cur, path, f = 0, [0], target(0)
        for j in range(1, n):
            if f is None or parents[r0 + j] != cur or not 0 <= tokens[r0 + j] < len(logits[0]):
                continue
            x, F = tokens[r0 + j], f.sum()
            greedy = not temp[i] > 0
            if f[x] > 0 if greedy else u[r0 + j] * (q[r0 + cur][x] if q is not None else 1.0) * F < f[x]:
                cur = j
                path.append(j)
                f = target(j)
            elif not greedy:
                f = np.maximum(f / F - q[r0 + cur], 0) if q is not None else np.where(np.arange(len(f)) == x, 0.0, f)
        n_kept.append(len(path))
        kept += path + [-1] * (n - len(path))
        if f is None:
            nxt.append(-1)
        else:
            if not f.sum() > 0:
                f = target(cur)
            c = np.cumsum(f)
            nxt.append(int(min(np.searchsorted(c, u_next[i] * c[-1], side="right"), np.nonzero(f > 0)[0][-1])))
        r0 += n
    return kept, n_kept, nxt


def verify_case(seed, n_row, vocab, dtype, dense, greedy, spread=3.0):
    g = np.random.default_rng(seed)
    total = sum(n_row)
    logits = torch.from_numpy(g.standard_normal((total, vocab)).astype(np.float32) * spread).to(dtype)
    about = torch.softmax(logits.float() + torch.from_numpy(g.standard_normal((total, vocab)).astype(np.float32)) * 0.7, -1)
    parents, tokens, r0 = [], [], 0
    for n in n_row:
        p = random_tree(g, n)
        for j in range(n):
            up = r0 + max(p[j], 0)
            if dense:
                w = about[up].double().numpy()
                tokens.append(int(g.choice(vocab, p=w / w.sum())))
            else:
                tokens.append(int(torch.argsort(about[up], descending=True)[min(int(g.integers(0, 3)), vocab - 1)]))
        parents += p
        r0 += n
    temp = g.uniform(0.3, 1.5, len(n_row)).astype(np.float32)
    if greedy == "some":
        temp[::2] = 0.0
    elif greedy:
        temp[:] = [0.0, -1.0, np.nan][seed % 3]
    u, un = g.random(total, dtype=np.float32), g.random(len(n_row), dtype=np.float32)
    return logits, about if dense else None, np.array(tokens, np.int32), np.array(parents, np.int32), u, un, temp


def verify_check(case, n_row, got=None):
    logits, q, tokens, parents, u, un, temp = case
    dev = [None if x is None else torch.as_tensor(x).cuda() for x in case]
    if got is None:
        got = draft.verify(dev[0], dev[2], dev[3], n_row, dev[4], dev[5], temperature=dev[6], draft=dev[1])
    want = verify_plain(logits.double().numpy(), tokens, parents, n_row, u.astype(np.float64), un.astype(np.float64), temp.astype(np.float64),
                        None if q is None else q.double().numpy())
    for g, w in zip(got, want):
        assert g.tolist() == list(w)
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("dense", [False, True])
@pytest.mark.parametrize("greedy", [False, True, "some"])
@pytest.mark.parametrize("vocab", [1, 7, 300, 4099, 32000])
def test_verify(dtype, dense, greedy, vocab):
    n_row = [5, 1, 0, 12, 3, 64, 2, 7]
    for seed in range(2):
        verify_check(verify_case(seed, n_row, vocab, dtype, dense, greedy), n_row)


@pytest.mark.parametrize("n", [1, 3, 17, 70, 1100])
def test_verify_counts_of_sequences(n):
    """Clusters of every size; more sequences than one launch lists."""
    n_row = [1 + i % 4 for i in range(n)]
    verify_check(verify_case(n, n_row, 2500, torch.float32, n % 2 == 0, False), n_row)


def test_verify_large_vocabulary():
    for n, dense in ((1, False), (2, True), (9, False)):
        n_row = [6] * n
        verify_check(verify_case(n, n_row, 128256, torch.bfloat16, dense, False), n_row)


def test_verify_rows_without_a_distribution():
    n_row = [3, 2, 2, 4, 1, 2]
    logits, q, tokens, parents, u, un, temp = verify_case(1, n_row, 500, torch.float32, False, "some")
    parents[:] = [-1, 0, 1, -1, 0, -1, 0, -1, 0, 1, 2, -1, -1, 0]
    u[:] = 0.0                                        # whatever has weight is accepted
    tokens[:] = np.argmax(logits.numpy(), 1)[[0, 0, 1, 3, 3, 5, 5, 7, 7, 8, 9, 11, 12, 12]]
    logits[1, 3] = math.nan                           # row 1 of sequence 0, after which nothing is tried
    logits[3, 499] = math.inf
    logits[6] = -math.inf
    logits[9, :250] = -math.inf                       # (a distribution all the same)
    logits[11, 5] = math.nan
    kept, n_kept, nxt = verify_check((logits, None, tokens, parents, u, un, temp), n_row)
    assert nxt.tolist()[:3] == [-1, -1, -1] and nxt.tolist()[4] == -1 and n_kept.tolist() == [2, 1, 2, 4, 1, 2]


def test_verify_borders():
    """Numbers of 0 and just below 1, tokens outside the vocabulary, parents outside the tree, tokens drafted twice,
    draws that leave nothing, logits of -infinity and of equal size, very low and high temperatures."""
    vocab, n_row = 64, [6] * 12
    logits, q, tokens, parents, u, un, temp = verify_case(5, n_row, vocab, torch.float32, True, False)
    u[::5] = 0.0
    u[1::7] = np.float32(1 - 2.0 ** -24)
    un[::3] = 0.0
    un[1::3] = np.float32(1 - 2.0 ** -24)
    tokens[3], tokens[8], tokens[15] = -1, vocab, 2 ** 31 - 1
    parents[4], parents[10], parents[16], parents[23] = 99, 5, -7, 2 ** 31 - 1
    tokens[25] = tokens[26] = tokens[27]
    parents[24:30] = [-1, 0, 0, 0, 1, 2]
    logits[30:36] = 0.0
    logits[36:42, 10:] = -math.inf
    temp[7], temp[8], temp[9] = 1e-30, 1e30, math.inf
    q[54:60] = 0.0                                    # tokens that the drafter could not have drawn
    q[60:66] = torch.softmax(logits[60:66] / float(temp[10]), -1)        # the target's own distribution
    verify_check((logits, q, tokens, parents, u, un, temp), n_row)
    verify_check((logits, None, tokens, parents, u, un, temp), n_row)
    # everything rejected: drafts that have all of the weight, and numbers that are not below 1
    one = torch.full((4, vocab), -math.inf)
    one[:, 9] = 1.0
    case = (one, None, np.array([0, 9, 9, 3], np.int32), np.array([-1, 0, 0, 0], np.int32), np.array([0, 1.5, 2, 0.5], np.float32),
            np.array([0.5], np.float32), np.array([1.0], np.float32))
    kept, n_kept, nxt = verify_check(case, [4])
    assert n_kept.tolist() == [1] and nxt.tolist() == [9]
    # a number that is none accepts nothing, and draws the last
    case[4][:], case[5][:] = math.nan, math.nan
    dev = [None if x is None else torch.as_tensor(x).cuda() for x in case]
    kept, n_kept, nxt = draft.verify(dev[0], dev[2], dev[3], [4], dev[4], dev[5], temperature=dev[6])
    assert kept.tolist() == [0, -1, -1, -1] and nxt.tolist() == [9]


def test_verify_strided_given_and_captured():
    vocab, n_row = 1001, [4, 9, 2]
    case = verify_case(7, n_row, vocab, torch.float16, True, False)
    logits, q, tokens, parents, u, un, temp = case
    lw, qw = torch.zeros(15, vocab + 6, dtype=torch.float16, device="cuda"), torch.zeros(15, vocab + 3, device="cuda")
    lw[:, 5:vocab + 5], qw[:, 1:vocab + 1] = logits.cuda(), q.cuda()
    dev = [torch.as_tensor(x).cuda() for x in (tokens, parents, u, un, temp)]
    out = [torch.full((n,), 9, dtype=torch.int32, device="cuda") for n in (15, 3, 3)]

    def call():
        return draft.verify(lw[:, 5:vocab + 5], dev[0], dev[1], n_row, dev[2], dev[3], temperature=dev[4], draft=qw[:, 1:vocab + 1], kept=out[0], n_kept=out[1],
                            next=out[2])
    assert call()[0] is out[0]
    verify_check(case, n_row, out)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        call()
    for seed in (8, 9):
        r = np.random.default_rng(seed)
        u[:], un[:] = r.random(15, dtype=np.float32), r.random(3, dtype=np.float32)
        dev[2].copy_(torch.from_numpy(u)), dev[3].copy_(torch.from_numpy(un))
        g.replay()
        torch.cuda.synchronize()
        verify_check(case, n_row, out)
    # no temperature: 1
    temp[:] = 1.0
    got = draft.verify(logits.cuda(), dev[0], dev[1], n_row, dev[2], dev[3], draft=q.cuda())
    verify_check(case, n_row, got)


@pytest.mark.parametrize("vocab", [128, 1024, 2048])
@pytest.mark.parametrize("n", [1, 300, 700])
def test_verify_short_rows_at_once(n, vocab):
    """Rows so short that a warp reads them in one step, soon after its block began: the exponential's table is whole by
    then, in every block and in launches one behind the other."""
    g = np.random.default_rng(n + vocab)
    n_row = [int(x) for x in g.integers(1, 4, n)]
    case = verify_case(n, n_row, vocab, torch.float32, False, False)
    want = verify_check(case, n_row)
    dev = [None if x is None else torch.as_tensor(x).cuda() for x in case]
    outs = [draft.verify(dev[0], dev[2], dev[3], n_row, dev[4], dev[5], temperature=dev[6]) for _ in range(50)]
    assert all(torch.equal(a, b) for got in outs for a, b in zip(got, want))


# ------------------------------------------------------------------ keep ---

@pytest.mark.parametrize("hd,n_kv,layers", [(128, 8, 3), (64, 1, 2), (32, 5, 1), (96, 3, 2), (64, 300, 1)])
def test_keep_moves_rows(hd, n_kv, layers):
    r = np.random.default_rng(hd)
    n = 6
    lens = [int(x) for x in r.integers(70, 200, n)]
    pool = kv4.KvPool(layers, n_kv, hd, sum(-(-v // PAGE) for v in lens) + 2, n, 4)
    pool.extend(np.arange(n), lens)
    for l in range(layers):
        pool.append(l, rows(l, sum(lens), n_kv, hd), rows(9 + l, sum(lens), n_kv, hd), list(range(n)), lens)
    before = [[pool.read(l, s) for l in range(layers)] for s in range(n)]
    new = [64, 1, 70, 0, 33, 60]
    kept = [sorted(int(x) for x in r.choice(m, int(r.integers(0, m + 1)), replace=False)) if m else [] for m in new]
    kept[0] = list(range(1, 64, 2))                   # places that are sources too
    kept[2] = list(range(3, 70))
    order = [4, 0, 2, 5, 1, 3]
    pool.keep(order, [new[s] for s in order], [kept[s] for s in order])
    for s in range(n):
        base = lens[s] - new[s]
        assert pool.length(s) == base + len(kept[s])
        at = list(range(base)) + [base + j for j in kept[s]]
        for l in range(layers):
            for a, b in zip(pool.read(l, s), before[s][l]):
                assert np.array_equal(a, b[at])
    assert pool.lengths.tolist() == [pool.length(s) for s in range(n)]
    for s in range(n):
        assert pool.table[s].tolist() == pool.pages(s) + [-1] * (4 - len(pool.pages(s)))


def test_keep_more_than_one_launch_lists():
    """Many sequences, and one whose moves go on in another launch."""
    hd, n_kv, n = 32, 1, 400
    pool = kv4.KvPool(1, n_kv, hd, 900, n, 20)
    lens = [40] * (n - 1) + [1200]
    pool.extend(np.arange(n), lens)
    pool.append(0, rows(1, sum(lens), n_kv, hd), rows(2, sum(lens), n_kv, hd), None, lens)
    before = [pool.read(0, s) for s in range(n)]
    new = [7] * (n - 1) + [1200]
    kept = [[0, 2, 5]] * (n - 1) + [list(range(0, 1200, 2)) + [1199]]
    pool.keep(np.arange(n), new, kept)
    for s in (0, 1, 200, 398, 399):
        at = list(range(lens[s] - new[s])) + [lens[s] - new[s] + j for j in kept[s]]
        for a, b in zip(pool.read(0, s), before[s]):
            assert np.array_equal(a, b[at])


def test_keep_refuses_capture():
    pool, _ = filled(1, 64, [100], 1)
    s = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with pytest.raises(engine.EngineError, match="captured"):
        with torch.cuda.graph(g, stream=s):
            pool.keep([0], [5], [[1]])
    torch.cuda.synchronize()
    assert pool.length(0) == 100
    pool.keep([0], [5], [[1]])
    assert pool.length(0) == 96


# --------------------------------------------------------------- together --

def test_a_run_of_steps():
    """Steps as a server takes them: extend, rotate and append, attend, verify, keep; two layers.  The cache then holds
    what appending the accepted tokens one by one would have left, bit for bit, and attention over it is the plain
    form's."""
    hd, n_kv, rep, layers, vocab, slots = 64, 2, 2, 2, 200, [2, 0]
    r = np.random.default_rng(3)
    rope = draft.Rope(hd, base=10000.0, scaling="bands", factor=4.0, context=256.0)
    pool, single = (kv4.KvPool(layers, n_kv, hd, 30, 3, 10) for _ in range(2))
    emb = [[torch.from_numpy(r.standard_normal((vocab, h, hd)).astype(np.float32)).cuda() for h in (rep * n_kv, n_kv, n_kv)] for _ in range(layers)]
    head = torch.from_numpy(r.standard_normal((rep * n_kv * hd, vocab)).astype(np.float32) * 0.3).cuda()
    last, taken = {s: int(r.integers(vocab)) for s in slots}, 0
    for s in slots:                                   # something cached already, shared with a fork that stays as it is
        n = 70 + s
        tok = torch.from_numpy(r.integers(0, vocab, n)).cuda()
        for p in (pool, single):
            p.extend([s], [n])
            for l in range(layers):
                p.append_rope(l, rope, None, emb[l][1][tok], emb[l][2][tok], [s], [n])
    pool.fork([0], [1])
    kept_fork = [pool.read(l, 1) for l in range(layers)]
    for step in range(12):
        new = [int(x) for x in r.integers(1, 12, len(slots))]
        parents = [random_tree(r, n) for n in new]
        parents = [[-1 if j == 0 else max(p, 0) for j, p in enumerate(t)] for t in parents]
        tokens = [[last[s]] + [int(x) for x in r.integers(0, vocab, n - 1)] for s, n in zip(slots, new)]
        depth, mask = draft.tree(parents)
        tok = torch.tensor([t for ts in tokens for t in ts], device="cuda")
        pool.extend(slots, new)
        out = None
        for l in range(layers):
            q = pool.append_rope(l, rope, emb[l][0][tok], emb[l][1][tok], emb[l][2][tok], slots, new, depth=depth)
            out = pool.attend_tree(l, q, slots, new, mask)
        vals = {s: tuple(x.astype(np.float64) for x in pool.read(layers - 1, s)) for s in slots}
        masks = [[int(x) for x in draft.tree(p, device=None)[1].view(np.uint64)] for p in parents]
        tree_check(pool, vals, q, slots, new, masks, out)
        logits = out.flatten(1) @ head
        u, un = (torch.from_numpy(r.random(m, dtype=np.float32)).cuda() for m in (sum(new), len(slots)))
        temp = torch.tensor([0.0 if step % 3 == 0 else 2.0, 4.0], device="cuda")
        flat = [p for t in parents for p in t]
        first = np.cumsum([0] + new)
        t32 = tok.int()
        kept, n_kept, nxt = draft.verify(logits, t32, torch.tensor(flat, dtype=torch.int32, device="cuda"), new, u, un, temperature=temp)
        want = verify_plain(logits.double().cpu().numpy(), t32.cpu().numpy(), flat, new, u.double().cpu().numpy(), un.double().cpu().numpy(),
                            temp.double().cpu().numpy(), None)
        assert kept.tolist() == want[0] and n_kept.tolist() == want[1] and nxt.tolist() == want[2]
        # (whatever was accepted, a path of the tree is kept: here the verified one, or every third step another)
        paths = []
        for i in range(len(slots)):
            path = kept[first[i]:first[i] + int(n_kept[i])].tolist()
            if step % 3 == 1:
                j, path = new[i] - 1, []
                while j >= 0:
                    path.append(j)
                    j = parents[i][j]
                path = path[::-1]
            paths.append(path)
        pool.keep(slots, new, paths)
        for s, path, ts, x in zip(slots, paths, tokens, nxt.tolist()):
            for j in path:
                single.extend([s], [1])
                t = torch.tensor([ts[j]], device="cuda")
                for l in range(layers):
                    single.append_rope(l, rope, None, emb[l][1][t], emb[l][2][t], [s], [1])
            last[s] = x
            taken += len(path)
    for s in slots:
        assert pool.length(s) == single.length(s)
        for l in range(layers):
            for a, b in zip(pool.read(l, s), single.read(l, s)):
                assert np.array_equal(a, b)
    for l in range(layers):
        for a, b in zip(pool.read(l, 1), kept_fork[l]):
            assert np.array_equal(a, b)
    assert taken > 40


def test_wrappers_refuse():
    pool = kv4.KvPool(1, 2, 64, 4, 2, 4)
    pool.extend([0, 1], [20, 20])
    rope, E = draft.Rope(64), engine.EngineError
    q, k = torch.zeros(5, 4, 64, device="cuda"), torch.zeros(5, 2, 64, device="cuda")
    i32 = torch.zeros(5, dtype=torch.int32, device="cuda")
    ok = pool.append_rope(0, rope, q, k, k, [0, 1], [3, 2], depth=i32)
    assert ok.shape == q.shape
    for args, kw in [((q, k, k, [0, 1], [3, 3]), {}), ((q, k, k, [0], [3, 2]), {}), ((q.half(), k, k, [0, 1], [3, 2]), {}), ((q[:4], k, k, [0, 1], [3, 2]), {}),
                     ((q, k, k.half(), [0, 1], [3, 2]), {}), ((q, k, k, [0, 1], [3, 2]), dict(depth=i32.long())), ((q, k, k, [0, 1], [3, 2]), dict(depth=i32[:4])),
                     ((q, k, k, [0, 1], [3, 2]), dict(depth=i32.cpu())), ((q, k, k, [0, 1], [3, 2]), dict(k_out=k)), ((None, k, k, [0, 1], [3, 2]), dict(q_out=q)),
                     ((q, k, k, [0, 1], [3, 2]), dict(q_out=q.half())), ((q.cpu(), k, k, [0, 1], [3, 2]), {}), ((q[..., :32], k, k, [0, 1], [3, 2]), {})]:
        with pytest.raises(E):
            pool.append_rope(0, rope, *args, **kw)
    m = torch.zeros(5, dtype=torch.int64, device="cuda")
    for args, kw in [((q, [0, 1], [3, 1]), {}), ((q, [0], [3, 2]), {}), ((q, [0, 1], [3, 2], m.int()), {}), ((q, [0, 1], [3, 2], m[:4]), {}),
                     ((q, [0, 1], [3, 2], m.cpu()), {}), ((q, [0, 1], [3, 2], m), dict(out=q.half())), ((q, [0, 1], [3, 2], m), dict(out=q[:4])),
                     ((q, [0, 1], [3, 2], m), dict(ws=m)), ((q, [0, 0], [3, 2], m), {}), ((q[:, :3], [0, 1], [3, 2], m), {})]:
        with pytest.raises(E):
            pool.attend_tree(0, *args, **kw)
    lg, f5, f2 = torch.zeros(5, 30, device="cuda"), torch.zeros(5, device="cuda"), torch.zeros(2, device="cuda")
    good = dict(logits=lg, tokens=i32, parents=i32, n_row=[3, 2], u=f5, u_next=f2)
    draft.verify(**good)
    for over in (dict(logits=lg.double()), dict(logits=lg[:4]), dict(logits=lg.cpu()), dict(logits=lg.t()), dict(tokens=i32.long()), dict(parents=i32[:4]), dict(u=f2),
                 dict(u_next=f5), dict(u=f5.half()), dict(temperature=f5), dict(draft=lg.half()), dict(draft=lg[:, :29]), dict(kept=f5), dict(n_kept=i32), dict(next=i32),
                 dict(n_row=[3, 1]), dict(n_row=[3.5, 1.5]), dict(u=None), dict(tokens=None)):
        with pytest.raises(E):
            draft.verify(**{**good, **over})
    pool.close()
    for call in (lambda: pool.attend_tree(0, q, [0, 1], [3, 2]), lambda: pool.append_rope(0, rope, q, k, k, [0, 1], [3, 2]), lambda: pool.keep([0], [1], [[0]])):
        with pytest.raises(E):
            call()


def test_tree_wait_that_gives_up():
    """Operands that never come: the kernel ends, the status says so, and the next call is right again."""
    hd, n_kv, rep, lens, new = 128, 8, 8, [2000] * 4, [16] * 4
    pool, vals = filled(n_kv, hd, lens, 3)
    _, mask = make(8, new)
    q = rows(5, sum(new), n_kv * rep, hd).half()
    want = pool.attend_tree(0, q, [0, 1, 2, 3], new, mask)
    kv4.prompt_status()
    engine.set_wait_ns(50_000_000)
    try:
        engine.inject_tree_timeout()
        pool.attend_tree(0, q, [0, 1, 2, 3], new, mask)
        with pytest.raises(engine.EngineError, match="bounded wait"):
            kv4.prompt_status()
    finally:
        engine.set_wait_ns(2_000_000_000)
    kv4.prompt_status()
    assert torch.equal(pool.attend_tree(0, q, [0, 1, 2, 3], new, mask), want)
    with pytest.raises(engine.EngineError):
        engine.inject_tree_timeout(99)
