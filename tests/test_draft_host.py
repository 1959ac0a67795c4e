"""Steps with drafted tokens, the part that needs no GPU: rotations, trees, what
the calls refuse, and the pool's bookkeeping of kept rows."""
import ctypes as C
import math
from pathlib import Path

import numpy as np
import pytest

from distcomp_b200 import draft, engine, kv4

PAGE = 64


def error():
    return engine.last_error()


# -------------------------------------------------------------- rotation ---

def turns_of(freq):
    """Radians a position as 64-bit fractions of a turn, in whole-number arithmetic."""
    two_pi = 6283185307179586476925286766559005768      # 2 pi * 10^36
    out = []
    for f in freq:
        num, den = float(f).as_integer_ratio()
        out.append(((num * 10 ** 36 << 64) // (den * two_pi)) % (1 << 64))
    return out


def close(turns, freq):
    """Within one unit for each 2^-63 of the frequency's own rounding in 64 bits of mantissa."""
    for t, w, f in zip(turns, turns_of(freq), freq):
        gap = (int(t) - w) % (1 << 64)
        assert min(gap, (1 << 64) - gap) <= 2 + abs(f) * 8, (int(t), w)


def formula(rot, base, scaling=None, factor=1.0, context=0.0, slow=1.0, fast=4.0):
    f = base ** (-2.0 * np.arange(rot // 2) / rot)
    if scaling is None:
        return f, 1.0
    if scaling == "linear":
        return f / factor, 1.0
    if scaling == "bands":
        w = np.clip((context * f / (2 * math.pi) - slow) / (fast - slow), 0, 1)
        return w * f + (1 - w) * f / factor, 1.0
    at = [rot * math.log(context / (t * 2 * math.pi)) / (2 * math.log(base)) for t in (fast, slow)]
    lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), rot - 1)
    w = np.clip((np.arange(rot // 2) - lo) / (hi - lo if hi != lo else 0.001), 0, 1)
    return f / factor * w + f * (1 - w), 0.1 * math.log(factor) + 1


@pytest.mark.parametrize("rot,base,kw", [
    (128, 500000.0, {}), (2, 10000.0, {}), (20, 10000.0, dict(scaling="linear", factor=4.0)),
    (128, 500000.0, dict(scaling="bands", factor=8.0, context=8192.0)), (64, 10000.0, dict(scaling="yarn", factor=16.0, context=4096.0, fast=32.0)),
    (64, 10000.0, dict(scaling="yarn", factor=1.0, context=2048.0, fast=8.0, slow=2.0))])
def test_rotation_follows_its_formula(rot, base, kw):
    r = draft.Rope(128, rot=rot, base=base, **kw)
    f, factor = formula(rot, base, **kw)
    assert r.rot == rot and r.factor == pytest.approx(factor, rel=1e-15)
    # pow differs by a few units of its last place between libraries
    for t, w, x in zip(r.turns, turns_of(f), f):
        assert abs(int(t) - w) <= 2 ** 64 * x / (2 * math.pi) * 2.0 ** -48 + 2
    close(draft.Rope(128, rot=rot, freq=f).turns, f)


def test_rotation_of_own_frequencies():
    f = [0.0, 1.0, 2 * math.pi, -0.25, 7.5]
    r = draft.Rope(64, rot=10, freq=f, factor=1.5, interleaved=True)
    close(r.turns, f)
    assert r.factor == 1.5
    assert draft.Rope(64, rot=0, freq=[]).rot == 0


@pytest.mark.parametrize("kw", [dict(rot=3), dict(rot=130), dict(rot=-2), dict(rot=66), dict(base=1.0), dict(base=math.nan), dict(scaling="other"),
                                dict(scaling="linear", factor=0.5), dict(scaling="linear", factor=math.inf), dict(scaling="bands", factor=2.0),
                                dict(scaling="bands", factor=2.0, context=100.0, slow=4.0, fast=4.0), dict(scaling="yarn", factor=math.nan, context=9.0),
                                dict(freq=[1.0]), dict(freq=[math.nan] * 32), dict(freq=[1.0] * 32, factor=math.inf),
                                dict(freq=[1.0] * 32, scaling="linear")])
def test_rotation_refuses(kw):
    with pytest.raises(engine.EngineError):
        draft.Rope(64, **kw)


def test_tree():
    depth, mask = draft.tree([-1, 0, 0, 1, 3, -1], device=None)
    assert depth.tolist() == [0, 1, 1, 2, 3, 0] and mask.tolist() == [1, 3, 5, 11, 27, 32]
    depth, mask = draft.tree([[-1, 0], [], list(range(-1, 63))], device=None)
    assert depth.tolist() == [0, 1] + list(range(64)) and mask.view(np.uint64).tolist() == [1, 3] + [(2 << j) - 1 for j in range(64)]
    for bad in ([0], [-1, 1], [-2], [-1] * 65, [-1, 0.5]):
        with pytest.raises(engine.EngineError):
            draft.tree(bad, device=None)


# ---------------------------------------------------------------- refusals --

def pool(n=4, n_kv=2, hd=64, pages=12, width=6):
    return kv4.KvPool(1, n_kv, hd, pages, n, width, device=-1)


def ints(*a):
    return np.array(a, dtype=np.int32)


def ptr(a):
    return a.ctypes.data if a is not None else None


ROPE = draft.Rope(64)
WIDE = draft.EcuRope(rot=96)


def append_args(p, **over):
    a = dict(h=p.h, layer=0, rope=ROPE.at, dtype=0, q=1 << 12, k=2 << 12, v=3 << 12, n_head=4, qs=256, ks=128, vs=128, seq=ints(0, 1), n_new=ints(3, 2), n=2,
             depth=None, qo=4 << 12, qos=256, od=0, ko=None, vo=None)
    a.update(over)
    return engine.lib().ecu_kv_append_rope(a["h"], a["layer"], a["rope"], a["dtype"], a["q"], a["k"], a["v"], a["n_head"], a["qs"], a["ks"], a["vs"],
                                           ptr(a["seq"]), ptr(a["n_new"]), a["n"], a["depth"], a["qo"], a["qos"], a["od"], a["ko"], a["vo"], None)


@pytest.mark.parametrize("over,why", [
    (dict(h=None), "null"), (dict(rope=None), "null"), (dict(n_new=None), "null"), (dict(n=-1), "negative"), (dict(layer=1), "layer 1 of 1"),
    (dict(dtype=3), "element type"), (dict(od=-1), "element type"), (dict(n_head=3), "3 query heads"), (dict(n_head=0), "query heads"), (dict(qo=None), "alone"),
    (dict(q=None), "alone"), (dict(seq=ints(0, 0)), "twice"), (dict(seq=ints(0, 9)), "no sequence 9"), (dict(n_new=ints(3, 200)), "200 rows"),
    (dict(n_new=ints(-1, 2)), "-1 rows"), (dict(k=None), "null rows"), (dict(v=None), "null rows"), (dict(ko=1 << 13), "alone"), (dict(ks=127), "overlap"),
    (dict(vs=0), "overlap"), (dict(qs=255), "overlap"), (dict(qos=-256), "overlap"), (dict(q=(1 << 12) + 2), "aligned"), (dict(depth=2), "aligned"),
    (dict(qo=1 << 12, qos=260), "in place"), (dict(rope=C.addressof(WIDE)), "96 turning"), (dict(), "no device")])
def test_append_rope_refuses(over, why):
    p = pool()
    p.extend([0, 1], [100, 50])
    assert append_args(p, **over) == -1 and why in error()


def test_append_rope_to_own_pages_only():
    p = pool()
    p.extend([0, 1], [100, 50])
    p.fork([0], [2])
    assert append_args(p) == -1 and "other sequences hold" in error()
    p.extend([2], [3])                                # a copy of the partly filled page
    assert append_args(p, seq=ints(2, 1)) == -1 and "no device" in error()
    assert append_args(p, n=0) == 0 and append_args(p, n_new=ints(0, 0), k=None) == 0


def tree_args(p, **over):
    a = dict(h=p.h, layer=0, dtype=0, q=1 << 12, out=2 << 12, n_head=4, qs=256, os=256, seq=ints(0, 1), n_new=ints(3, 2), n=2, mask=None, scale=0.1, ws=None)
    a.update(over)
    return engine.lib().ecu_kv_attend_tree(a["h"], a["layer"], a["dtype"], a["q"], a["out"], a["n_head"], a["qs"], a["os"], ptr(a["seq"]), ptr(a["n_new"]),
                                           a["n"], a["mask"], a["scale"], a["ws"], None)


@pytest.mark.parametrize("over,why", [
    (dict(h=None), "null"), (dict(n_new=None), "null"), (dict(n=-1), "negative"), (dict(layer=-1), "layer -1"), (dict(dtype=7), "element type"),
    (dict(n_head=5), "5 query heads"), (dict(n_head=2 * 4097), "query heads"), (dict(scale=math.inf), "finite"), (dict(seq=ints(1, 1)), "twice"),
    (dict(seq=ints(-1, 1)), "no sequence -1"), (dict(n_new=ints(3, 65)), "64 drafted"), (dict(n_new=ints(3, 51)), "51 rows"), (dict(n_new=ints(-3, 1)), "-3 rows"),
    (dict(q=None), "null rows"), (dict(out=None), "null rows"), (dict(qs=128), "overlap"), (dict(os=0), "overlap"), (dict(out=(2 << 12) + 1), "aligned"),
    (dict(mask=4), "aligned"), (dict(ws=8), "aligned"), (dict(), "no device")])
def test_attend_tree_refuses(over, why):
    p = pool()
    p.extend([0, 1], [100, 50])
    assert tree_args(p, **over) == -1 and why in error()


def test_attend_tree_of_nothing():
    p = pool()
    p.extend([0], [100])
    assert tree_args(p, n=0, q=None) == 0 and tree_args(p, n_new=ints(0, 0), out=None) == 0
    assert engine.lib().ecu_kv_tree_ws_bytes(p.h) == 0 and engine.lib().ecu_kv_tree_ws_bytes(None) == 0


def verify_args(**over):
    a = dict(dtype=0, logits=1 << 12, stride=100, vocab=100, draft=None, ds=0, token=1 << 12, parent=1 << 12, n_row=ints(2, 3), n=2, u=1 << 12, un=1 << 12,
             temp=None, kept=1 << 12, nk=1 << 12, next=1 << 12, device=0)
    a.update(over)
    return engine.lib().ecu_draft_verify(a["dtype"], a["logits"], a["stride"], a["vocab"], a["draft"], a["ds"], a["token"], a["parent"], ptr(a["n_row"]), a["n"],
                                         a["u"], a["un"], a["temp"], a["kept"], a["nk"], a["next"], a["device"], None)


@pytest.mark.parametrize("over,why", [
    (dict(dtype=9), "element type"), (dict(n=-1), "negative"), (dict(vocab=0), "vocabulary"), (dict(n_row=None), "null"), (dict(un=None), "null"),
    (dict(nk=None), "null"), (dict(next=None), "null"), (dict(n_row=ints(2, 65)), "64 at most"), (dict(n_row=ints(-1, 1)), "-1 rows"), (dict(logits=None), "null rows"),
    (dict(token=None), "null rows"), (dict(parent=None), "null rows"), (dict(u=None), "null rows"), (dict(kept=None), "null rows"), (dict(stride=99), "overlap"),
    (dict(draft=1 << 12, ds=99), "overlap"), (dict(logits=(1 << 12) + 2), "aligned"), (dict(u=(1 << 12) + 1), "aligned"), (dict(device=-1), "not available"),
    (dict(device=99), "not available")])
def test_verify_refuses(over, why):
    assert verify_args(**over) == -1 and why in error()


def test_verify_refuses_a_vocabulary_past_counting():
    assert verify_args(vocab=2 ** 30 + 1, stride=2 ** 30 + 1) == -1 and "2^30" in error()


def test_verify_of_nothing():
    assert verify_args(n=0) == 0


@pytest.mark.parametrize("parents", [None, 5, iter([-1]), [None], [[-1], None], [[-1], 3], [-1, [0]], [[[-1]]], "ab"])
def test_tree_refuses_what_are_no_lists(parents):
    with pytest.raises(engine.EngineError):
        draft.tree(parents, device=None)


# ------------------------------------------------------------------ verify ---

def statements(text):
    """What stands outside of all braces."""
    depth, out = 0, []
    for c in text:
        depth += c == "{"
        if depth == 0:
            out.append(c)
        depth -= c == "}"
    return "".join(out)


def test_verify_meets_between_the_table_and_its_readers():
    """Eight of a block's sixteen warps write the exponential's table, all read it from the first row on: the block meets in
    between (the missing barrier cannot be made to show: the logits' loads hide it)."""
    source = (Path(engine.__file__).parent / "csrc" / "ecu_verify.cuh").read_text()
    kernel = source[source.index("k_draft_verify("):]
    written, read = kernel.index("table[tid] ="), kernel.index("open_row(0)")
    assert written < read and "__syncthreads();" in statements(kernel[written:read])


# ------------------------------------------------------------------- keep ---

def test_keep_gives_the_rest_back():
    p = pool()
    p.extend([0, 1, 2], [60, 64, 10])
    p.extend([0, 1], [64, 5])
    assert p.used == 5
    p.keep([1, 0], [5, 64], [[], [0, 3, 63]])
    assert [p.length(s) for s in range(3)] == [63, 64, 10] and p.used == 3
    p.keep([2], [10], [list(range(10))])              # all of it
    p.keep([2], [0], [[]])
    p.keep([], [], [])
    assert p.length(2) == 10
    p.keep([2], [10], [[9]])
    assert p.length(2) == 1
    p.keep([2], [1], [[]])
    assert p.length(2) == 0 and p.used == 2


@pytest.mark.parametrize("seq,n_new,kept,why", [
    ([0, 0], [1, 1], [[0], [0]], "twice"), ([5], [1], [[0]], "no sequence 5"), ([0], [101], [[0]], "100 positions"), ([0], [-1], [[]], "positions"),
    ([0], [3], [[0, 1, 2, 2]], "4 rows of 3"), ([0], [3], [[0, 3]], "rising"), ([0], [3], [[1, 1]], "rising"), ([0], [3], [[2, 1]], "rising"),
    ([0], [3], [[-1]], "rising"), ([1, 0], [2, 3], [[0], [0, 5]], "rising")])
def test_keep_refuses_whole(seq, n_new, kept, why):
    p = pool()
    p.extend([0, 1], [100, 50])
    with pytest.raises(engine.EngineError, match=why):
        p.keep(seq, n_new, kept)
    assert [p.length(s) for s in (0, 1)] == [100, 50] and p.used == 3


def test_keep_moves_rows_of_own_pages_only():
    p = pool()
    p.extend([0], [100])
    p.fork([0], [1])
    with pytest.raises(engine.EngineError, match="other sequences hold"):
        p.keep([0], [5], [[0, 2]])
    p.keep([0], [5], [[0, 1]])                        # nothing moves
    assert p.length(0) == 97 and p.length(1) == 100
    p.extend([0], [5])                                # its own copy now
    p.keep([0], [5], [[1, 4]])
    assert p.length(0) == 99


def test_keep_whose_launch_fails_is_taken_back():
    p = pool()
    p.extend([0, 1], [130, 50])
    before = [(p.length(s), p.pages(s)) for s in (0, 1)]
    p.inject_failure()
    with pytest.raises(engine.EngineError, match="injected"):
        p.keep([0, 1], [70, 3], [[5, 9], [2]])
    assert [(p.length(s), p.pages(s)) for s in (0, 1)] == before
    p.keep([0, 1], [70, 3], [[5, 9], [2]])
    assert [p.length(s) for s in (0, 1)] == [62, 48]


def test_keep_refuses_lists():
    p = pool()
    p.extend([0], [10])
    for args in (([0], [1, 1], [[0]]), ([0], [1], []), ([0], [2 ** 32], [[0]]), ([0], [2], [[0.5]])):
        with pytest.raises(engine.EngineError):
            p.keep(*args)
    L = engine.lib()
    one = ints(1)
    assert L.ecu_kv_keep(p.h, ptr(ints(0)), ptr(one), None, ptr(one), 1, None) == -1
    assert L.ecu_kv_keep(p.h, ptr(ints(0)), ptr(one), None, None, 1, None) == -1
    assert L.ecu_kv_keep(p.h, None, ptr(one), ptr(one), ptr(one), 1, None) == -1
    assert L.ecu_kv_keep(None, ptr(ints(0)), ptr(one), ptr(ints(0)), ptr(one), 1, None) == -1
    p.keep([0], [1], [[0]])


def test_keep_refuses_what_are_no_lists_of_rows():
    p = pool()
    p.extend([0], [10])
    for kept in ([0], [None], [iter([0])], [np.array(0)], [[[0]]], [["0"]], None, 7, iter([[0]])):
        with pytest.raises(engine.EngineError):
            p.keep([0], [1], kept)
    assert p.length(0) == 10
    p.keep([0], [1], [(0,)])
