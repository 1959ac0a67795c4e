"""The paged 4-bit K/V cache and the prompt attention on the GPU, against
plain 64-bit forms of the same definitions.

Tolerances, from the arithmetic (h = half a step of a type, relative):
  * stored values are decided exactly: equal bit for bit;
  * a score is a dot of hd products in fp32: hd / 16 matrix steps, each adding
    a tree of at most 8 roundings or cuts of 2^-23 of the partial sums, which
    are at most A = max_t sum_d |q_d k_td|; the split of an fp32 query leaves
    2^-22 of its largest element, 2^-22 * A at most counted twice.  With the
    scale and the base-2 exponential (2^-21 relative each):
    ds = |scale| * A * 2^-23 * (hd / 2 + 16) + 2^-20;
  * a weight is then off by 2 * ds (numerator and sum), a sum of n weighted
    rows by 2^-23 * (n / 16 + 64): both times max |v|;
  * 16-bit forms round weights once more before their product with V: h of
    the type that they are rounded to (fp16 for the cache, q's own for the
    prompt) times sum p |v|, plus fp16's smallest step at the top of its
    range; and every output by h of its type.
"""
import math

import numpy as np
import pytest
import torch

from distcomp_b200 import engine, kv4

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.float16, torch.bfloat16]
PAGE = 64
H16 = 2.0 ** -11


@pytest.fixture(autouse=True)
def _quiet():
    yield
    torch.cuda.synchronize()


def rows(seed, *shape, spread=1.0):
    g = np.random.default_rng(seed)
    x = g.standard_normal(shape) * spread
    x[..., :: 13] *= 6.0
    return torch.from_numpy(x.astype(np.float32)).cuda()


def quantised(x):
    """The definition in 64 bits: (codes, fp16 scales) of rows [..., hd]."""
    x = x.double().cpu().numpy()
    b = x.reshape(*x.shape[:-1], -1, 32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        mag = np.where(np.isnan(b), -1, np.abs(b))
        m = np.take_along_axis(b, np.argmax(mag, -1)[..., None], -1)
        d = np.clip(m / -8.0, -65504, 65504).astype(np.float32).astype(np.float16)
        fine = np.isfinite(b).all(-1, keepdims=True)
        d = np.where(fine, np.where(d == 0, np.float16(0), d), np.float16(np.nan))
        use = fine & (d != 0)
        code = np.where(use, np.clip(np.floor(b / np.where(use, d, 1).astype(np.float64) + 8.5), 0, 15), 8)
    return code.astype(np.int64), d[..., 0]


def stored(x):
    code, d = quantised(x)
    return ((code - 8) * d[..., None].astype(np.float64)).reshape(x.shape)


def place(t, b, nb):
    return b ^ ((t >> 1) & 3) if nb == 4 else b ^ ((t >> 2) & 1) if nb == 2 else b


def filled(n_kv, hd, lens, seed, pool_pages=None, layers=1, layer=0, dtype=torch.float32, gap=3):
    """A pool whose sequences hold `lens` positions (pages interleaved), and their values in 64 bits."""
    lens = list(lens)
    width = max(1, max(-(-v // PAGE) for v in lens))
    need = sum(-(-v // PAGE) for v in lens) + gap
    pool = kv4.KvPool(layers, n_kv, hd, pool_pages or need, max(1, len(lens)), width)
    kd = torch.as_tensor(kv4._Memory(pool.info().data, (layers * pool.n_pages * kv4.page_bytes(n_kv, hd) // 4,), pool), device="cuda")
    kd.fill_(-1)                                     # codes 15, NaN scales: what nothing may read
    held, vals = [0] * len(lens), [([], []) for _ in lens]
    step, k = 0, 0
    while any(h < v for h, v in zip(held, lens)):
        for i, v in enumerate(lens):
            n = min([37, 64, 1, 130][(step + i) % 4] if v < 600 else 1000, v - held[i])
            if n <= 0:
                continue
            kk, vv = rows(seed + 2 * k, n, n_kv, hd).to(dtype), rows(seed + 2 * k + 1, n, n_kv, hd, spread=0.3).to(dtype)
            k += 1
            pool.extend([i], [n])
            pool.append(layer, kk, vv, [i], [n])
            vals[i][0].append(stored(kk)), vals[i][1].append(stored(vv))
            held[i] += n
        step += 1
    return pool, [tuple(np.concatenate(s) if s else np.zeros((0, n_kv, hd)) for s in v) for v in vals]


def reference(q, k, v, scale, ds_extra, hw, hout, causal_from=None):
    """(out, tolerance) in 64 bits of query rows q [r, H, hd] over k, v [n, Hkv, hd]; row i sees causal_from + i keys."""
    r, H, hd = q.shape
    n, kv = k.shape[0], k.shape[1]
    out, tol = np.zeros((r, H, hd)), np.zeros((r, H, hd))
    for h in range(H):
        kh, vh = k[:, h // (H // kv)], v[:, h // (H // kv)]
        s = q[:, h] @ kh.T * scale
        A = np.max(np.abs(q[:, h]) @ np.abs(kh).T, axis=1, initial=0.0)
        ds = abs(scale) * A * 2.0 ** -23 * (hd / 2 + 16) + 2.0 ** -20
        seen = np.full(r, n) if causal_from is None else np.maximum(0, causal_from + np.arange(r))
        s = np.where(np.arange(n)[None] < seen[:, None], s, -np.inf)
        live = seen > 0
        if not live.any():
            continue
        p = np.exp(s[live] - s[live].max(1, keepdims=True))
        p /= p.sum(1, keepdims=True)
        out[live, h] = p @ vh
        vmax = np.abs(vh).max(initial=0.0)
        tol[live, h] = (vmax * (2 * ds[live] + 2.0 ** -23 * (n / 16 + 64)))[:, None] + hw * (p @ np.abs(vh)) + hout * np.abs(out[live, h])
        tol[live, h] += vmax * ds_extra
    return out, tol


def check(got, want, tol):
    got = got.double().cpu().numpy()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    err = np.nan_to_num(np.abs(got - want))
    worst = np.max(err / np.where(tol > 0, tol, 1e-30), initial=0.0)
    assert worst <= 1.0, f"worst error {worst:.3g} of the tolerance, {err.max():.3g} absolute"


def attend_check(pool, vals, q, seq, out, scale=None):
    hd = q.shape[-1]
    half = torch.finfo(q.dtype).eps / 2
    wide = q.dtype == torch.float32
    for i, s in enumerate(seq):
        k, v = vals[s]
        want, tol = reference(q[i:i + 1].double().cpu().numpy(), k, v, hd ** -0.5 if scale is None else scale,
                              0.0 if wide else 2.0 ** -24, 0.0 if wide else H16, half)
        check(out[i:i + 1], want, tol)


# ---------------------------------------------------------------- append ---

@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", TYPES)
def test_append_stores_the_definition(hd, dtype):
    """Every stored byte of the rows, the values handed back, and nothing else changed."""
    n_kv, nb, lens = 3, hd // 32, [1, 64, 130, 63]
    pool = kv4.KvPool(2, n_kv, hd, 9, 4, 3)
    data = torch.as_tensor(kv4._Memory(pool.info().data, (2, 9, kv4.page_bytes(n_kv, hd) // 4), pool), device="cuda")
    data.fill_(0x5A5A5A5A)
    pool.extend([2, 0, 3, 1], [lens[s] for s in (2, 0, 3, 1)])
    n_new = [1, 5, 130, 0]
    seq = [2, 1, 0, 3]
    counts = [130, 5, 1, 0]
    total = sum(counts)
    wide = rows(5, total, 2 * n_kv * hd + 24).to(dtype)       # k and v side by side, an odd distance apart
    if dtype != torch.float32:
        wide[3, 7:9] = wide[3, 9:11].abs().max() * 8          # equal magnitudes: the first decides
        wide[3, 8] = -wide[3, 7]
    k, v = wide[:, :n_kv * hd], wide[:, n_kv * hd + 8:2 * n_kv * hd + 8]
    ko, vo = (torch.empty(total, n_kv, hd, device="cuda", dtype=torch.float32) for _ in range(2))
    pool.append(1, k, v, seq, counts, k_out=ko, v_out=vo)
    for x, o in ((k, ko), (v, vo)):
        want = stored(x.reshape(total, n_kv, hd))
        assert np.array_equal(o.double().cpu().numpy(), want)
    raw = data.cpu().numpy().view(np.uint8).reshape(2, 9, n_kv, 72 * hd)
    assert (raw[0] == 0x5A).all()
    want = np.full((9, n_kv, 72 * hd), 0x5A, dtype=np.uint8)
    r = 0
    for s, c in zip(seq, counts):
        for pos in range(lens[s] - c, lens[s]):
            page, t = pool.pages(s)[pos // PAGE], pos % PAGE
            for side, x in ((0, k), (1, v)):
                code, d = quantised(x[r].reshape(n_kv, hd))
                for h in range(n_kv):
                    for b in range(nb):
                        at = side * 32 * hd + t * (hd // 2) + place(t, b, nb) * 16
                        want[page, h, at:at + 16] = code[h, b, 0::2] | code[h, b, 1::2] << 4
                        at = 64 * hd + side * 4 * hd + (t * nb + b) * 2
                        want[page, h, at:at + 2] = np.frombuffer(d[h, b].tobytes(), np.uint8)
            r += 1
    assert np.array_equal(raw[1], want)
    kr, vr = pool.read(1, 2)
    assert np.array_equal(kr.astype(np.float64), stored(k[:130].reshape(130, n_kv, hd)))
    assert np.array_equal(vr.astype(np.float64), stored(v[:130].reshape(130, n_kv, hd)))


def test_append_unusual_values():
    """Borders between codes, zeros, subnormals, huge, infinite and NaN values."""
    hd, n_kv = 64, 1
    x = torch.zeros(40, n_kv, hd)
    g = torch.Generator().manual_seed(1)
    for r in range(12):                              # multiples of half a scale: every border
        d = float(torch.tensor(2.0 ** (r - 14) * (1 + r / 16)).half())
        x[r, 0, :32] = (torch.arange(32).float() - 16) / 2 * d
        x[r, 0, 0] = -8 * d
        x[r, 0, 32:] = torch.nextafter(x[r, 0, :32], torch.full((32,), 1e9))
        x[r, 0, 32] = -8 * d
    x[12, 0, 3] = 1e-9                               # a scale that rounds to zero
    x[13, 0, 5] = -3e-7                              # a subnormal scale
    x[14] = torch.randn(n_kv, hd, generator=g) * 1e-6
    x[15] = torch.randn(n_kv, hd, generator=g) * 3e38
    x[16, 0, 9], x[17, 0, 40], x[18, 0, 0] = float("inf"), float("nan"), float("-inf")
    x[19, 0, :] = 600000.0
    x[20, 0, 4], x[20, 0, 2] = 5.0, -5.0
    x[21:] = torch.randn(19, n_kv, hd, generator=g)
    pool = kv4.KvPool(1, n_kv, hd, 1, 1, 1)
    pool.extend([0], [40])
    k = x.cuda()
    ko, vo = torch.empty_like(k), torch.empty_like(k)
    pool.append(0, k, -k, [0], [40], k_out=ko, v_out=vo)
    assert np.array_equal(ko.double().cpu().numpy(), stored(k), equal_nan=True)
    assert np.array_equal(vo.double().cpu().numpy(), stored(-k), equal_nan=True)
    kr, _ = pool.read(0, 0)
    assert np.array_equal(kr.astype(np.float64), stored(k), equal_nan=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_append_rows_at_any_address(dtype):
    """Rows that begin between 16-byte boundaries, and values handed back there."""
    hd, n_kv = 64, 2
    flat = rows(3, 7 * 133 + 1).to(dtype)
    k = flat[1:].as_strided((7, n_kv * hd), (133, 1), 1)
    out = torch.zeros(2 * 7 * n_kv * hd + 1, device="cuda", dtype=dtype)
    ko, vo = out[1:1 + 7 * n_kv * hd].view(7, n_kv, hd), out[1 + 7 * n_kv * hd:].view(7, n_kv, hd)
    pool = kv4.KvPool(1, n_kv, hd, 1, 1, 1)
    pool.extend([0], [7])
    pool.append(0, k, k, [0], [7], k_out=ko, v_out=vo)
    want = torch.from_numpy(stored(k.reshape(7, n_kv, hd))).float().to(dtype)
    assert torch.equal(ko.cpu(), want) and torch.equal(vo.cpu(), want)


def test_append_more_sequences_than_one_launch_lists():
    n, hd = 1500, 32
    pool = kv4.KvPool(1, 1, hd, n + 40, n, 2)
    counts = [1 + (i * 7) % 3 for i in range(n)]
    pool.extend(range(n), counts)
    k = rows(9, sum(counts), 1, hd)
    pool.append(0, k, k + 1, None, counts)
    want_k, want_v = stored(k), stored(k + 1)
    at = np.cumsum([0] + counts)
    for s in (0, 1, 1023, 1024, 1025, n - 1):
        kr, vr = pool.read(0, s)
        assert np.array_equal(kr.astype(np.float64), want_k[at[s]:at[s + 1]])
        assert np.array_equal(vr.astype(np.float64), want_v[at[s]:at[s + 1]])
    q = rows(10, n, 2, hd)
    out = pool.attend(0, q, None)
    vals = {s: (want_k[at[s]:at[s + 1]], want_v[at[s]:at[s + 1]]) for s in range(n)}
    attend_check(pool, vals, q, range(n), out)


# ---------------------------------------------------------------- attend ---

LENS = [1, 0, 31, 32, 33, 63, 64, 65, 96, 127, 128, 129, 200, 333]


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rep", [1, 4])
def test_attend_lengths(hd, dtype, rep):
    n_kv = 2
    pool, vals = filled(n_kv, hd, LENS, seed=hd + rep, layers=2, layer=1)
    seq = list(range(len(LENS)))[::-1] + [3, 3, 12]
    q = rows(77, len(seq), rep * n_kv, hd, spread=1.5).to(dtype)
    out = torch.full_like(q, float("nan"))
    assert pool.attend(1, q, seq, out=out) is out
    attend_check(pool, vals, q, seq, out)


@pytest.mark.parametrize("rep", [2, 3, 5, 6, 7, 8, 9, 16, 33])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_attend_head_groups(rep, dtype):
    lens, hd, n_kv = [70, 1, 259], 64 if rep % 2 else 128, 2
    pool, vals = filled(n_kv, hd, lens, seed=rep)
    q = rows(rep, 3, rep * n_kv, hd).to(dtype)
    attend_check(pool, vals, q, [0, 1, 2], pool.attend(0, q))


@pytest.mark.parametrize("n_kv, rep, lens", [(1, 4, [40001]), (8, 4, [9000, 17, 3000]), (2, 8, [1, 1, 20011, 1])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attend_long(n_kv, rep, lens, dtype):
    """Rows whose positions many CTAs share, next to short ones."""
    pool, vals = filled(n_kv, 128, lens, seed=4)
    q = rows(8, len(lens), rep * n_kv, 128, spread=2.0).to(dtype)
    out = pool.attend(0, q)
    attend_check(pool, vals, q, range(len(lens)), out)
    for _ in range(3):                               # the same bits whatever the order in which the CTAs end
        assert torch.equal(pool.attend(0, q), out)


@pytest.mark.parametrize("hd, rep", [(32, 3), (64, 8), (96, 5), (96, 1), (128, 9)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_attend_long_other_shapes(hd, rep, dtype):
    """Rows across many CTAs at every head size, padded head groups, and a negative scale."""
    lens = [9001, 40, 3000]
    pool, vals = filled(1, hd, lens, seed=hd)
    q = rows(8, 3, rep, hd).to(dtype)
    for scale in (hd ** -0.5, -0.05):
        attend_check(pool, vals, q, [2, 0, 1], pool.attend(0, q, [2, 0, 1], scale=scale), scale=scale)


def test_attend_zero_and_tiny_rows():
    """Keys, values or queries of zeros, and V scales from fp16's smallest to its largest, in one sequence."""
    hd, n = 64, 300
    pool = kv4.KvPool(1, 1, hd, 6, 2, 5)
    k, v = rows(1, n, 1, hd), rows(2, n, 1, hd)
    k[:64], v[32:96] = 0, 0
    v[128:160] *= 1e-6
    v[200:210] *= 3e4
    pool.extend([0, 1], [n, 33])
    pool.append(0, torch.cat([k, torch.zeros(33, 1, hd, device="cuda")]), torch.cat([v, torch.zeros(33, 1, hd, device="cuda")]),
                [0, 1], [n, 33])
    q = rows(3, 2, 2, hd)
    q[:, 1] = 0
    out = pool.attend(0, q)
    assert (out[1] == 0).all()
    attend_check(pool, [(stored(k), stored(v))], q[:1], [0], out[:1])


def test_attend_many_short():
    r = np.random.default_rng(0)
    lens = [int(v) for v in r.integers(0, 150, 300)]
    pool, vals = filled(2, 64, lens, seed=21)
    q = rows(8, 300, 4, 64).half()
    attend_check(pool, vals, q, range(300), pool.attend(0, q))


def test_attend_strided_scaled_and_misaligned():
    lens = [100, 65]
    pool, vals = filled(2, 64, lens, seed=2)
    wide = rows(5, 2, 4 * 64 + 131)
    q = wide[:, 3:3 + 256]
    buf = torch.zeros(2, 300, device="cuda")
    out = buf[:, 5:261]
    pool.attend(0, q, [1, 0], out=out, scale=0.5)
    attend_check(pool, vals, q.reshape(2, 4, 64), [1, 0], out.reshape(2, 4, 64), scale=0.5)
    assert (buf[:, :5] == 0).all() and (buf[:, 261:] == 0).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_attend_peaked_flat_and_far_values(dtype):
    """Scores that leave one position, queries of zero, values far apart in size."""
    hd, n = 64, 200
    pool = kv4.KvPool(1, 1, hd, 4, 1, 4)
    k, v = rows(1, n, 1, hd), rows(2, n, 1, hd)
    k[50] *= 30
    v[:100] *= 1e-4
    v[150:] *= 200
    pool.extend([0], [n])
    pool.append(0, k, v, [0], [n])
    q = torch.stack([rows(3, 1, hd) * 10, torch.zeros(1, hd, device="cuda"), rows(4, 1, hd) * 1e-6]).to(dtype)
    vals = [(stored(k), stored(v))]
    attend_check(pool, vals, q, [0, 0, 0], pool.attend(0, q, [0, 0, 0]))


def test_attend_nan_rows_stay_in_their_sequence():
    """A row that is not finite reads as NaN, in the sequences that hold it only; what lies past a length is never read."""
    hd = 64
    pool, vals = filled(1, hd, [70, 80], seed=3)     # unwritten positions hold NaN scales
    k, v = rows(5, 1, 1, hd), rows(6, 1, 1, hd)
    v[0, 0, 40] = float("inf")
    pool.extend([0], [1])
    pool.append(0, k, v, [0], [1])
    q = rows(7, 2, 2, hd)
    out = pool.attend(0, q)
    attend_check(pool, vals, q[1:], [1], out[1:])
    assert torch.isnan(out[0, :, 32:]).all() and torch.isfinite(out[0, :, :32]).all()
    pool.truncate([0], [70])
    attend_check(pool, vals, q, [0, 1], pool.attend(0, q))


def nan_check(pool, vals, q, out):
    """Sequence 0's row: NaN where the definition is NaN, the rest as without the values that are not finite."""
    n_kv, rep = pool.n_head_kv, q.shape[1] // pool.n_head_kv
    k, v = vals
    for g in range(n_kv):
        hs = slice(g * rep, (g + 1) * rep)
        bad_v = np.isnan(v[:, g]).any(0)
        want_nan = np.broadcast_to(bad_v | np.isnan(k[:, g]).any(), (rep, pool.head_dim))
        got = out[0, hs].double().cpu().numpy()
        assert np.array_equal(np.isnan(got), want_nan), f"KV head {g}"
        if np.isnan(k[:, g]).any():
            continue
        half, wide = torch.finfo(q.dtype).eps / 2, q.dtype == torch.float32
        want, tol = reference(q[:1, hs].double().cpu().numpy(), k[:, g:g + 1], np.nan_to_num(v[:, g:g + 1]), pool.head_dim ** -0.5,
                              0.0 if wide else 2.0 ** -24, 0.0 if wide else H16, half)
        fine = ~bad_v
        assert (np.abs(got[:, fine] - want[0][:, fine]) <= tol[0][:, fine]).all()


@pytest.mark.parametrize("n_kv, rep", [(1, 4), (2, 1), (8, 4), (8, 8)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, first, count", [(33, 32, 1), (65, 64, 1), (65, 0, 1), (96, 32, 32), (5000, 4992, 8), (5000, 1000, 32)])
def test_attend_keys_that_are_not_finite(n_kv, rep, dtype, n, first, count):
    """A key that is not finite makes its head's row NaN, wherever it lies: alone in its warp's part of the row, as a
    whole unit, or in one CTA's part of many."""
    hd = 64
    pool = kv4.KvPool(1, n_kv, hd, 80, 1, 80)
    k, v = rows(n, n, n_kv, hd), rows(n + 1, n, n_kv, hd)
    k[first:first + count, n_kv - 1, 3] = float("nan")
    pool.extend([0], [n])
    pool.append(0, k, v, [0], [n])
    q = rows(9, 1, rep * n_kv, hd).to(dtype)
    nan_check(pool, (stored(k), stored(v)), q, pool.attend(0, q))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n, at", [(33, 32), (33, 0), (65, 40), (5000, 4999), (5000, 7)])
def test_attend_values_that_are_not_finite_and_weigh_nothing(dtype, n, at):
    """A value that is not finite makes its dimensions NaN however small its weight is: 0 * NaN is NaN."""
    hd, n_kv = 64, 8
    pool = kv4.KvPool(1, n_kv, hd, 80, 1, 80)
    k, v = rows(n, n, n_kv, hd), rows(n + 1, n, n_kv, hd)
    unit = slice(at // 32 * 32, min(n, at // 32 * 32 + 32))
    k[unit, 5] = 0
    k[unit, 5, 0] = -400                             # the whole unit far below the others: its weights are zero
    v[at, 5, 40] = float("inf")
    pool.extend([0], [n])
    pool.append(0, k, v, [0], [n])
    q = rows(9, 1, 4 * n_kv, hd)
    q[:, :, 0] = 20                                  # scores of -1000
    q = q.to(dtype)
    nan_check(pool, (stored(k), stored(v)), q, pool.attend(0, q))


def test_attend_beyond_32_bits():
    """Pages further than 4 GB into the layer."""
    hd, n_kv = 128, 8
    far = (5 << 30) // kv4.page_bytes(n_kv, hd)
    pool = kv4.KvPool(1, n_kv, hd, far + 4, 2, far)
    pool.extend([0, 1], [far * PAGE, 100])
    k, v = rows(1, 100, n_kv, hd), rows(2, 100, n_kv, hd)
    pool.append(0, k, v, [1], [100])
    assert pool.pages(1) == [far, far + 1]
    q = rows(3, 1, 2 * n_kv, hd)
    vals = {1: (stored(k), stored(v))}
    attend_check(pool, vals, q, [1], pool.attend(0, q, [1]))
    pool.free([0])
    assert pool.compact() == 2 and pool.pages(1) == [0, 1]
    attend_check(pool, vals, q, [1], pool.attend(0, q, [1]))


def test_attend_captured_follows_the_lengths():
    """A captured step (append, attend) replayed as the sequences grow; two graphs with workspaces of their own."""
    hd, n_kv, n = 128, 2, 3
    lens = [62, 1, 500]
    pool, vals = filled(n_kv, hd, lens, seed=1, pool_pages=40)
    vals = [list(v) for v in vals]
    big = kv4.KvPool(1, n_kv, hd, 40, n, 20)
    big.extend([0, 1, 2], lens)
    kd, vd = (torch.from_numpy(np.concatenate([v[j] for v in vals])).float().cuda() for j in (0, 1))
    big.append(0, kd, vd, [0, 1, 2], lens)
    for i in range(n):                               # stored values are stored again as they are read
        a = big.read(0, i)
        vals[i] = [a[0].astype(np.float64), a[1].astype(np.float64)]
    k, v, q = (torch.zeros(n, h, hd, device="cuda") for h in (n_kv, n_kv, 2 * n_kv))
    out = torch.zeros_like(q)
    big.extend([0, 1, 2], [1, 1, 1])
    with pytest.raises(engine.EngineError, match="workspace of its own"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            big.attend(0, q, out=out)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        ws = big.workspace()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            big.append(0, k, v, None, [1, 1, 1])
            big.attend(0, q, out=out, ws=ws)
        graphs.append((gr, ws))
    for step in range(5):
        if step:
            big.extend([0, 1, 2], [1, 1, 1])
        k.copy_(rows(100 + step, n, n_kv, hd)), v.copy_(rows(200 + step, n, n_kv, hd)), q.copy_(rows(300 + step, n, 2 * n_kv, hd))
        graphs[step % 2][0].replay()
        for i in range(n):
            vals[i][0] = np.concatenate([vals[i][0], stored(k[i:i + 1])])
            vals[i][1] = np.concatenate([vals[i][1], stored(v[i:i + 1])])
        attend_check(big, vals, q, [0, 1, 2], out)
    with pytest.raises(engine.EngineError, match="cannot be captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            big.free([0])
    torch.cuda.synchronize()
    assert big.length(0) == lens[0] + 5


def test_attend_on_two_streams():
    """Overlapping calls on two streams take workspaces of their own."""
    pool, vals = filled(1, 128, [30000, 29000], seed=6)
    q = rows(3, 1, 4, 128)
    want = [pool.attend(0, q, [s]).clone() for s in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[torch.empty_like(q) for _ in range(20)] for _ in range(2)]
    for j in range(20):
        for s in (0, 1):
            pool.attend(0, q, [s], out=outs[s][j], stream=streams[s].cuda_stream)
    torch.cuda.synchronize()
    for s in (0, 1):
        for o in outs[s]:
            assert torch.equal(o, want[s])


# ----------------------------------------------------------------- pages ---

def test_attend_keeps_a_workspace_a_stream():
    """The pool's own workspaces go by the stream, not by its handle: the per-thread default stream has one handle for
    all threads, and two threads' calls may overlap."""
    import threading
    hd, n_kv, n = 64, 2, 3000
    pool, vals = filled(n_kv, hd, [n], 5)
    q = rows(6, 1, n_kv, hd)
    want = pool.attend(0, q, [0])
    torch.cuda.synchronize()
    per = pool.ws_bytes()
    for _ in range(2):
        pool.attend(0, q, [0], stream=2)                  # this thread's own default stream
    before = pool.info().device_bytes
    outs, errors = [torch.zeros_like(q) for _ in range(2)], []

    def work(out):
        try:
            for _ in range(20):
                pool.attend(0, q, [0], out=out, stream=2)
        except Exception as e:
            errors.append(e)
    for o in outs:                                        # one after the other on the host; their kernels may overlap
        t = threading.Thread(target=work, args=(o,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert not errors and all(torch.equal(o, want) for o in outs)
    assert pool.info().device_bytes == before + 2 * per
    streams = [torch.cuda.Stream(priority=p) for _ in range(32) for p in (0, -1)]
    outs = []
    for s in streams:                                     # more than the pool keeps
        outs.append(torch.zeros_like(q))
        s.wait_stream(torch.cuda.current_stream())
        pool.attend(0, q, [0], out=outs[-1], stream=s.cuda_stream)
        assert pool.info().device_bytes <= before + 16 * per
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    pool.close()


def test_pages_follow_their_sequences():
    """Forks, copies on write, truncations and compactions leave every sequence's rows as they were."""
    hd, n_kv, layers, slots = 64, 2, 3, 6
    pool = kv4.KvPool(layers, n_kv, hd, 40, slots, 8)
    r = np.random.default_rng(3)
    held = [[np.zeros((0, 2, n_kv, hd)) for _ in range(layers)] for _ in range(slots)]
    for step in range(120):
        s = int(r.integers(slots))
        what = r.choice(["grow", "grow", "fork", "cut", "free", "compact"])
        if what == "grow":
            n = int(r.integers(1, 90))
            try:
                pool.extend([s], [n])
            except engine.EngineError:
                continue
            for l in range(layers):
                k, v = rows(step * 10 + l, n, n_kv, hd), rows(step * 10 + l + 5, n, n_kv, hd)
                pool.append(l, k, v, [s], [n])
                held[s][l] = np.concatenate([held[s][l], np.stack([stored(k), stored(v)], 1)])
        elif what == "fork":
            d = int(r.integers(slots))
            if d != s and pool.length(d) == 0:
                pool.fork([s], [d])
                held[d] = [x.copy() for x in held[s]]
        elif what == "cut" and pool.length(s):
            n = int(r.integers(0, pool.length(s) + 1))
            pool.truncate([s], [n])
            held[s] = [x[:n] for x in held[s]]
        elif what == "free" and r.random() < 0.3:
            pool.free([s])
            held[s] = [x[:0] for x in held[s]]
        elif what == "compact":
            pool.compact()
            assert all(p < pool.used for i in range(slots) for p in pool.pages(i))
        if step % 10 == 9:
            table, lens = pool.table.cpu().numpy(), pool.lengths.cpu().numpy()
            for i in range(slots):
                n = pool.length(i)
                assert lens[i] == n and list(table[i]) == pool.pages(i) + [-1] * (8 - len(pool.pages(i)))
                for l in range(layers):
                    k, v = pool.read(l, i)
                    assert np.array_equal(k.astype(np.float64), held[i][l][:, 0]), (step, i, l)
                    assert np.array_equal(v.astype(np.float64), held[i][l][:, 1]), (step, i, l)


def test_pages_of_a_failed_change():
    """A change whose first launch fails leaves the device's tables and pages to the sequences that had them."""
    hd, n_kv = 64, 2
    pool, vals = filled(n_kv, hd, [70, 130, 5], seed=4, gap=8)
    q = rows(5, 3, 4, hd)
    want, table, lens = pool.attend(0, q).clone(), pool.table.clone(), pool.lengths.clone()
    for f in (lambda: pool.extend([0, 2], [100, 1]), lambda: pool.truncate([1], [3]), lambda: pool.free([0, 2])):
        pool.inject_failure()
        with pytest.raises(engine.EngineError, match="injected"):
            f()
        assert torch.equal(pool.table, table) and torch.equal(pool.lengths, lens)
        assert torch.equal(pool.attend(0, q), want)
    pool.free([0])
    pool.inject_failure()
    with pytest.raises(engine.EngineError, match="injected"):
        pool.compact()
    assert torch.equal(pool.attend(0, q[1:], [1, 2]), want[1:])
    assert pool.compact() > 0
    attend_check(pool, vals, q[1:], [1, 2], pool.attend(0, q[1:], [1, 2]))


def test_pages_many_at_once():
    """More copies and words than one launch's argument holds."""
    hd, n_kv, n = 32, 1, 1500
    pool = kv4.KvPool(1, n_kv, hd, 4 * n, 2 * n, 2)
    pool.extend(range(n), [70] * n)
    k, v = rows(1, 70 * n, n_kv, hd), rows(2, 70 * n, n_kv, hd)
    pool.append(0, k, v, None, [70] * n)
    pool.fork(range(n), range(n, 2 * n))
    pool.extend(range(n, 2 * n), [1] * n)
    pool.free(range(0, n))
    assert pool.used == 2 * n and pool.compact() > 0
    table = pool.table.cpu().numpy()
    assert (table[:n] == -1).all() and sorted(table[n:].ravel()) == list(range(2 * n))
    want_k, want_v = stored(k), stored(v)
    for i in (0, 1, 700, n - 1):
        kr, vr = pool.read(0, n + i, 0, 70)
        assert np.array_equal(kr.astype(np.float64), want_k[70 * i:70 * i + 70])
        assert np.array_equal(vr.astype(np.float64), want_v[70 * i:70 * i + 70])


# ---------------------------------------------------------------- prompt ---

def prompt_check(q, k, v, out, cu_q, cu_k, scale=None):
    hd, half = q.shape[-1], torch.finfo(q.dtype).eps / 2
    for s in range(len(cu_q) - 1):
        a, b, c, d = cu_q[s], cu_q[s + 1], cu_k[s], cu_k[s + 1]
        if a == b:
            continue
        want, tol = reference(*(x.double().cpu().numpy() for x in (q[a:b], k[c:d], v[c:d])), hd ** -0.5 if scale is None else scale,
                              2.0 ** -24, half, half, causal_from=(d - c) - (b - a) + 1)
        check(out[a:b], want, tol)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rep", [1, 2, 3, 4])
def test_prompt_lengths(hd, dtype, rep):
    lens = [1, 127, 0, 128, 129, 2, 255, 256, 257, 300]
    past = [0, 5, 3, 0, 128, 127, 0, 1, 0, 200]
    n_kv = 2
    cu_q, cu_k = np.cumsum([0] + lens), np.cumsum([0] + [a + b for a, b in zip(lens, past)])
    q = rows(1, cu_q[-1], rep * n_kv, hd, spread=1.5).to(dtype)
    k, v = rows(2, cu_k[-1], n_kv, hd).to(dtype), rows(3, cu_k[-1], n_kv, hd).to(dtype)
    out = kv4.prompt_attention(q, k, v, cu_q, cu_k)
    prompt_check(q, k, v, out, cu_q, cu_k)
    assert torch.equal(kv4.prompt_attention(q, k, v, cu_q, cu_k), out)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_strided_rows_and_what_lies_behind(dtype):
    """q, k and v side by side in one buffer; rows behind the last, and other buffers' columns, left alone."""
    n, H, kv, hd = 150, 4, 2, 128
    width = (H + 2 * kv) * hd + 8
    buf = rows(4, n + 140, width).to(dtype)
    buf[n:] = float("nan")
    q, k, v = (buf[:n, a * hd:b * hd].unflatten(1, (b - a, hd)) for a, b in ((0, H), (H, H + kv), (H + kv, H + 2 * kv)))
    ob = torch.full((n + 9, H * hd + 16), 7.0, device="cuda", dtype=dtype)
    out = ob[:n, 8:8 + H * hd].unflatten(1, (H, hd))
    kv4.prompt_attention(q, k, v, [0, 20, 150], out=out, scale=0.2)
    prompt_check(q, k, v, out, [0, 20, 150], [0, 20, 150], scale=0.2)
    assert (ob[n:] == 7).all() and (ob[:, :8] == 7).all() and (ob[:, 8 + H * hd:] == 7).all()


def test_prompt_rows_that_see_nothing():
    """Fewer keys than queries: the first rows see none and become zeros."""
    hd = 64
    q, k, v = rows(1, 200, 2, hd).half(), rows(2, 30, 1, hd).half(), rows(3, 30, 1, hd).half()
    out = torch.full_like(q, float("nan"))
    cu_q, cu_k = [0, 150, 160, 200], [0, 20, 20, 30]
    kv4.prompt_attention(q, k, v, cu_q, cu_k, out=out)
    assert (out[:130] == 0).all() and (out[150:190] == 0).all()
    prompt_check(q, k, v, out, cu_q, cu_k)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_prompt_masked_places_have_no_effect(hd, bad):
    """Keys and values that are not finite reach the rows that see them and no other: within a tile, behind a
    sequence's end, and in the next sequence."""
    lens = [100, 70, 140]
    cu = np.cumsum([0] + lens)
    q, k, v = rows(1, 310, 2, hd).bfloat16(), rows(2, 310, 2, hd).bfloat16(), rows(3, 310, 2, hd).bfloat16()
    want = kv4.prompt_attention(q, k, v, cu)
    v2, k2 = v.clone(), k.clone()
    v2[60, 0, 5] = bad                               # seen by rows 60..99 of the first sequence, KV head 0
    v2[100 + 69, 1, 7] = bad                         # the second one's last row
    k2[170 + 139, 0, 3] = float("nan")               # the third one's last key
    out = kv4.prompt_attention(q, k2, v2, cu)
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[60:100, 0, 5] = True
    hit[169, 1, 7] = True
    hit[309, 0, :] = True
    assert torch.equal(out[~hit], want[~hit])
    assert not torch.isfinite(out[hit]).any()
    if bad != bad:
        assert torch.isnan(out[hit]).all()
    else:
        assert (out[60:100, 0, 5] == bad).all() and out[169, 1, 7] == bad


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_masked_places_of_the_largest_values(hd, dtype):
    """The largest finite keys and values in masked places, one of them at every place of a tile, weigh nothing."""
    n, big = 300, torch.finfo(dtype).max
    q, k, v = rows(1, n, 2, hd).to(dtype), rows(2, n, 2, hd).to(dtype), rows(3, n, 2, hd).to(dtype)
    want = kv4.prompt_attention(q, k, v, [0, n])
    for first in (40, 150):
        k2, v2 = k.clone(), v.clone()
        k2[first:] = big
        v2[first:] = -big
        assert torch.equal(kv4.prompt_attention(q, k2, v2, [0, n])[:first], want[:first])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_weights_that_vanish(dtype):
    """A key 2^369 ahead of all the others: their values, however large, add nothing.  The key lies at every place.
    (Where it comes in the second tile of 128 keys, the first one's sum comes before it: 128 of the largest bf16
    values, 2^135, are past fp32, so they are 2^100 there.)"""
    n, hd = 200, 64
    q = torch.zeros(n, 1, hd, device="cuda", dtype=dtype)
    k = torch.zeros(n * n, 1, hd, device="cuda", dtype=dtype)
    v = torch.full((n * n, 1, hd), torch.finfo(dtype).max, device="cuda", dtype=dtype)
    at = torch.arange(n, device="cuda") * (n + 1)
    q[:, 0, 0] = 16
    k[at, 0, 0] = 16
    if dtype is torch.bfloat16:
        v[128 * n:] = 2.0 ** 100
    v[at] = 1
    out = kv4.prompt_attention(q, k, v, range(n + 1), range(0, n * n + 1, n), scale=1.0)
    assert (out == 1).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_infinite_scores(dtype):
    """A score of -inf weighs nothing; of +inf, or -inf alone, the softmax is NaN.  At every place of a tile."""
    n, hd = 200, 64
    cu_q, cu_k = range(n + 1), range(0, n * n + 1, n)
    q, k, v = rows(1, n, 1, hd), rows(2, n * n, 1, hd), rows(3, n * n, 1, hd).to(dtype)
    q[:, 0, 0] = q[:, 0, 0].abs() + 0.5
    q, k = q.to(dtype), k.to(dtype)
    at = torch.arange(n, device="cuda") * (n + 1)
    k[at, 0, 0] = float("inf")
    assert torch.isnan(kv4.prompt_attention(q, k, v, cu_q, cu_k)).all()
    k[at, 0, 0] = float("-inf")
    v[at] = torch.finfo(dtype).max
    out = kv4.prompt_attention(q, k, v, cu_q, cu_k)
    rest = torch.ones(n * n, dtype=torch.bool, device="cuda")
    rest[at] = False
    prompt_check(q, k[rest], v[rest], out, list(cu_q), list(range(0, n * (n - 1) + 1, n - 1)))
    k[:, 0, 0] = float("-inf")
    assert torch.isnan(kv4.prompt_attention(q, k, v, cu_q, cu_k)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_prompt_large_scores(dtype):
    """Scores in the hundreds, one key that takes all, rows of equal scores."""
    n, hd = 300, 128
    q, k, v = rows(1, n, 1, hd).to(dtype) * 8, rows(2, n, 1, hd).to(dtype) * 4, rows(3, n, 1, hd).to(dtype)
    q[10:20] = 0
    out = kv4.prompt_attention(q, k, v, [0, n])
    prompt_check(q, k, v, out, [0, n], [0, n])


def test_prompt_many_sequences():
    r = np.random.default_rng(1)
    lens = [int(x) for x in r.integers(0, 4, 2100)]
    lens[1500] = 400
    cu = np.cumsum([0] + lens)
    q, k, v = rows(1, cu[-1], 2, 64).half(), rows(2, cu[-1], 1, 64).half(), rows(3, cu[-1], 1, 64).half()
    out = kv4.prompt_attention(q, k, v, cu)
    prompt_check(q, k, v, out, cu, cu)


def test_prompt_long():
    """One long prompt: rows from its start, its middle and its end against 64 bits."""
    n, H, hd = 5000, 4, 128
    q, k, v = rows(1, n, H, hd).bfloat16(), rows(2, n, 2, hd).bfloat16(), rows(3, n, 2, hd).bfloat16()
    out = kv4.prompt_attention(q, k, v, [0, n])
    for a, b in ((0, 40), (2500, 2540), (4960, 5000)):
        prompt_check(q[a:b], k[:b], v[:b], out[a:b], [0, b - a], [0, b])


def test_prompt_captured_and_on_a_stream():
    n, hd = 333, 64
    q, k, v = rows(1, n, 2, hd).half(), rows(2, n, 1, hd).half(), rows(3, n, 1, hd).half()
    want = kv4.prompt_attention(q, k, v, [0, 33, n])
    out = torch.zeros_like(q)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        kv4.prompt_attention(q, k, v, [0, 33, n], out=out)
    gr.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    side = torch.cuda.Stream()
    out2 = torch.zeros_like(q)
    torch.cuda.synchronize()
    kv4.prompt_attention(q, k, v, [0, 33, n], out=out2, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out2, want)


# -------------------------------------------------------------- together ---

def test_prompts_then_steps():
    """What a server does: prompts written and attended, a fork, single tokens, the pool closed up in between."""
    hd, n_kv, rep = 128, 2, 4
    lens = [150, 64, 33]
    pool = kv4.KvPool(1, n_kv, hd, 30, 5, 6)
    pool.extend([0, 1, 2], lens)
    cu, n = np.cumsum([0] + lens), sum(lens)
    q, k, v = rows(1, n, rep * n_kv, hd).half(), rows(2, n, n_kv, hd).half(), rows(3, n, n_kv, hd).half()
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    pool.append(0, k, v, [0, 1, 2], lens, k_out=ko, v_out=vo)
    out = kv4.prompt_attention(q, ko, vo, cu)
    prompt_check(q, ko, vo, out, cu, cu)
    hist = [[stored(x[cu[i]:cu[i + 1]]) for x in (k, v)] for i in range(3)]
    pool.fork([0, 0], [3, 4])
    hist += [[x.copy() for x in hist[0]] for _ in range(2)]
    pool.free([1])
    live = [0, 2, 3, 4]
    for step in range(4):
        if step == 2:                                # sequence 2's page becomes a hole in front of a copied one
            live.remove(2)
            pool.free([2])
        m = len(live)
        pool.extend(live, [1] * m)
        k1, v1, q1 = (rows(50 + 3 * step + j, m, h, hd).half() for j, h in enumerate((n_kv, n_kv, rep * n_kv)))
        pool.append(0, k1, v1, live, [1] * m)
        if step == 2:
            assert pool.compact() == 1
        for i, s in enumerate(live):
            hist[s] = [np.concatenate([a, stored(b[i:i + 1])]) for a, b in zip(hist[s], (k1, v1))]
        attend_check(pool, hist, q1, live, pool.attend(0, q1, live))


# -------------------------------------------------------------- refusals ---

def test_wrappers_refuse():
    """What only the tensors show: types, devices, shapes, strides, sizes."""
    hd, n_kv = 64, 2
    pool = kv4.KvPool(1, n_kv, hd, 4, 3, 2)
    pool.extend([0, 1], [5, 70])
    k = rows(1, 5, n_kv, hd)
    cpu, wide = k.cpu(), rows(2, 5, n_kv, 2 * hd)
    bad = engine.EngineError
    for kk, vv in ((cpu, k), (k, cpu), (k.double(), k.double()), (k, k.half()), (k[:4], k[:4]), (k[:, :1], k[:, :1]),
                   (wide[..., :hd], k), (k.transpose(0, 1), k), (k.transpose(1, 2).contiguous().transpose(1, 2), k),
                   (k[0], k[0]), (k.flatten(1)[:, 1:], k)):
        with pytest.raises(bad):
            pool.append(0, kk, vv, [0], [5])
    for seq, n_new in (([0], [5, 0]), ([0.5], [5]), ([[0]], [[5]]), ([1 << 33], [5]), ([0, 0], [3, 2]), ([2], [5])):
        with pytest.raises(bad):
            pool.append(0, k, k, seq, n_new)
    out = torch.empty_like(k)
    for ko, vo in ((out, None), (None, out), (out[:4], out[:4]), (out, out.half()), (out.cpu(), out), (wide[..., :hd], out)):
        with pytest.raises(bad):
            pool.append(0, k, k, [0], [5], k_out=ko, v_out=vo)
    q = rows(3, 2, 4, hd)
    for qq, kw in ((q.cpu(), {}), (q.double(), {}), (q[:, :3], {}), (q, {"out": q.half()}), (q, {"out": q[:1]}),
                   (q, {"seq": [0]}), (q, {"seq": [0, 3]}), (q, {"ws": torch.zeros(8, device="cuda")}),
                   (q, {"ws": pool.workspace().cpu()}), (q, {"scale": float("inf")}), (q[..., :32], {})):
        with pytest.raises(bad):
            pool.attend(0, qq, **{"seq": [0, 1], **kw})
    for l in (-1, 1):
        with pytest.raises(bad):
            pool.attend(l, q, [0, 1])
    h = rows(4, 6, 2, hd).half()
    for a, b, c, cu, kw in ((h.cpu(), h, h, [0, 6], {}), (h.float(), h.float(), h.float(), [0, 6], {}), (h, h, h, [0, 5], {}),
                            (h, h[:5], h, [0, 6], {}), (h, h, h.bfloat16(), [0, 6], {}), (h, h, h, [0, 6], {"cu_k": [0, 3, 6]}),
                            (h, h, h, [], {}), (h, h, h, [0, 6], {"out": h[:5]}), (h, h, h, [0, 6], {"scale": -1.0}),
                            (h[:, :, :32], h, h, [0, 6], {}), (h, h, h, [0, 7, 6], {})):
        with pytest.raises(bad):
            kv4.prompt_attention(a, b, c, cu, **kw)
    flat = torch.zeros(6 * 2 * hd + 1, device="cuda", dtype=torch.float16)[1:].view(6, 2, hd)
    with pytest.raises(bad, match="16-byte aligned"):
        kv4.prompt_attention(flat, flat, flat, [0, 6])
    with pytest.raises(bad):
        kv4.KvPool(1, n_kv, hd, 4, 3, 2, data=torch.zeros(100, device="cuda"))
    assert pool.length(0) == 5 and pool.used == 3


def test_pool_over_given_memory_and_its_end():
    """Pages in the caller's memory stay as they are; a closed pool answers with errors."""
    hd, n_kv = 32, 1
    data = torch.full((2, 3, kv4.page_bytes(n_kv, hd)), 7, dtype=torch.uint8, device="cuda")
    pool = kv4.KvPool(2, n_kv, hd, 3, 2, 2, data=data)
    assert (data == 7).all()
    pool.extend([1], [3])
    k = rows(1, 3, n_kv, hd)
    pool.append(1, k, k, [1], [3])
    assert (data[0] == 7).all() and (data[1, 1:] == 7).all() and not (data[1, 0] == 7).all()
    pool.close()
    pool.close()
    for f in (pool.info, lambda: pool.length(0), lambda: pool.extend([0], [1]), lambda: pool.compact(),
              lambda: pool.append(0, k, k, [1], [3]), lambda: pool.attend(0, k, [1, 1, 1])):
        with pytest.raises(engine.EngineError):
            f()
    assert (data[0] == 7).all()
    for f in (lambda: pool.table, lambda: pool.lengths, lambda: pool.read(0, 1)):
        with pytest.raises(engine.EngineError):
            f()


THREADS = '''
import sys, threading
sys.path[:0] = sys.argv[1:]
import torch
from distcomp_b200 import draft, kv4
hd, n_kv, n = 64, 2, 3000
pool = kv4.KvPool(1, n_kv, hd, 120, 2, 60)
pool.extend([0, 1], [n, 100])
k, q = torch.randn(n, n_kv, hd, device="cuda"), torch.randn(16, n_kv, hd, device="cuda")
pool.append(0, k, k, [0], [n])
logits, zero = torch.randn(16, 5000, device="cuda"), torch.zeros(16, device="cuda")
rope, ints = draft.Rope(hd), torch.zeros(16, dtype=torch.int32, device="cuda")
calls = [lambda: pool.attend(0, q[:1], [0], stream=2),
         lambda: pool.append(0, k[:16], k[:16], [1], [16], stream=2),
         lambda: pool.append_rope(0, rope, q, k[:16], k[:16], [1], [16], stream=2),
         lambda: pool.attend_tree(0, q, [0], [16], stream=2),
         lambda: draft.verify(logits, ints, ints, [16], zero, zero[:1], stream=2),
         lambda: kv4.prompt_attention(k, k, k, [0, n], stream=2)]
torch.cuda.synchronize()

def work(call):
    for _ in range(20):
        call()
for call in calls * 3:                                # one after the other on the host, each ended with work under way
    t = threading.Thread(target=work, args=(call,))
    t.start()
    t.join()
torch.cuda.synchronize()
print("all through")
'''


def test_threads_that_end_with_work_under_way():
    """Calls on the default streams of threads that end at once, while the next thread calls: in a process of its own,
    which a limit ends where the threads would wait for one another."""
    import subprocess
    import sys
    from pathlib import Path
    root = Path(kv4.__file__).resolve().parents[1]
    for _ in range(4):
        r = subprocess.run([sys.executable, "-c", THREADS, str(root)], capture_output=True, text=True, timeout=120)
        assert r.returncode == 0 and "all through" in r.stdout, r.stderr[-2000:]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,lens", [(64, [150] * 8), (128, [6000]), (96, [700, 1, 90])])
@pytest.mark.parametrize("top", [18, 20, 24, 27, 30])
def test_attend_scores_past_what_a_float_steps_over(dtype, hd, lens, top):
    """Scores around 2^top and beyond: rows stay finite, and one whose largest score is clear of all rounding shows its
    value (its weight and the output are rounded once each, the weights' sum is not)."""
    n_kv, rep = 2, 8
    pool = kv4.KvPool(1, n_kv, hd, sum(-(-n // PAGE) for n in lens), len(lens), -(-max(lens) // PAGE))
    n, half = max(lens), torch.finfo(dtype).eps / 2
    k, v, q = rows(1, n, n_kv, hd), rows(2, n, n_kv, hd), rows(5, len(lens), n_kv * rep, hd).to(dtype)
    k[70] *= 2.0 ** 12
    pool.extend(range(len(lens)), lens)
    for s, m in enumerate(lens):
        pool.append(0, k[:m], v[:m], [s], [m])
    kn, vn = (torch.from_numpy(stored(x)).cuda().repeat_interleave(rep, 1) for x in (k, v))
    scale = 2.0 ** top / float(torch.einsum("rhd,hd->rh", q.double(), kn[70]).abs().median())
    got, clear_rows = pool.attend(0, q, list(range(len(lens))), scale=scale), 0
    assert torch.isfinite(got).all()
    for s, m in enumerate(lens):
        sc = torch.einsum("hd,thd->ht", q[s].double(), kn[:m]) * scale
        size = (torch.einsum("hd,thd->ht", q[s].double().abs(), kn[:m].abs()) * scale).amax(-1)
        two = torch.cat((sc, torch.full_like(sc[:, :1], -math.inf)), 1).topk(2, -1)
        clear = two.values[:, 0] - two.values[:, 1] > 2 * size * 2.0 ** -23 * (hd / 2 + 16) + 64
        want = vn[two.indices[:, 0], torch.arange(n_kv * rep, device="cuda")]
        tol = (half + (2.0 ** -20 if dtype == torch.float32 else H16)) * want.abs() + 2.0 ** -20
        assert ((got[s].double() - want).abs() <= tol)[clear].all()
        clear_rows += int(clear.sum())
    assert clear_rows > 0.2 * q.shape[0] * q.shape[1]


@pytest.mark.parametrize("dtype", TYPES[1:])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("top", [18, 20, 24, 27, 30])
def test_prompt_scores_past_what_a_float_steps_over(dtype, hd, top):
    """As test_attend_scores_past_what_a_float_steps_over, of a prompt: rows stay finite, and one whose largest score is
    clear of all rounding shows its value."""
    n, n_kv, rep, half = 600, 2, 4, torch.finfo(dtype).eps / 2
    k, v, q = rows(1, n, n_kv, hd).to(dtype), rows(2, n, n_kv, hd).to(dtype), rows(3, n, n_kv * rep, hd).to(dtype)
    k[70] *= 2.0 ** 10
    kk, vv = k.double().repeat_interleave(rep, 1), v.double().repeat_interleave(rep, 1)
    sc = torch.einsum("rhd,thd->rht", q.double(), kk)
    scale = 2.0 ** top / float(sc[100:].abs().amax(-1).median())
    unseen = torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1)[:, None]
    size = (torch.einsum("rhd,thd->rht", q.double().abs(), kk.abs()) * scale).masked_fill(unseen, 0.0).amax(-1)
    two = (sc * scale).masked_fill(unseen, -math.inf).topk(2, -1)
    clear = two.values[..., 0] - two.values[..., 1] > 2 * size * 2.0 ** -23 * (hd / 2 + 16) + 64
    want = vv[two.indices[..., 0], torch.arange(n_kv * rep, device="cuda")[None]]
    got = kv4.prompt_attention(q, k, v, [0, n], scale=scale)
    assert torch.isfinite(got).all()
    assert clear.sum() > 0.2 * clear.numel()
    assert ((got.double() - want).abs() <= 2 * half * want.abs() + 2.0 ** -20)[clear].all()
