"""The page pool's bookkeeping against a plain model of it, and what the 4-bit
cache's and the prompt attention's entry points refuse.  No kernel runs here:
a pool of device -1 is the bookkeeping alone, and every refusal comes before
the device is used."""
import ctypes as C
import random

import numpy as np
import pytest

from distcomp_b200 import engine, kv4

PAGE = 64


class Model:
    """Lists of pages and counts, the rules written out."""

    def __init__(self, pages, slots, per):
        self.ref, self.per = [0] * pages, per
        self.pages, self.len = [[] for _ in range(slots)], [0] * slots

    def take(self):
        p = self.ref.index(0)
        self.ref[p] = 1
        return p

    def extend(self, s, n):
        if self.len[s] % PAGE and n and self.ref[self.pages[s][-1]] > 1:
            old = self.pages[s][-1]
            self.pages[s][-1] = self.take()
            self.ref[old] -= 1
        while len(self.pages[s]) * PAGE < self.len[s] + n:
            self.pages[s].append(self.take())
        self.len[s] += n

    def need(self, s, n):
        return (self.len[s] % PAGE and n and self.ref[self.pages[s][-1]] > 1) + max(
            0, -(-(self.len[s] + n) // PAGE) - len(self.pages[s]))

    def fork(self, a, b):
        self.pages[b], self.len[b] = list(self.pages[a]), self.len[a]
        for p in self.pages[a]:
            self.ref[p] += 1

    def truncate(self, s, n):
        while len(self.pages[s]) * PAGE - PAGE >= n and self.pages[s]:
            self.ref[self.pages[s].pop()] -= 1
        self.len[s] = n

    def compact(self):
        used = sum(r > 0 for r in self.ref)
        holes = [p for p in range(used) if not self.ref[p]]
        tops = [p for p in range(used, len(self.ref)) if self.ref[p]]
        to = dict(zip(tops, holes))
        self.pages = [[to.get(p, p) for p in q] for q in self.pages]
        for a, b in to.items():
            self.ref[b], self.ref[a] = self.ref[a], 0
        return len(to)


def same(pool, m):
    assert pool.used == sum(r > 0 for r in m.ref)
    for s in range(len(m.len)):
        assert pool.length(s) == m.len[s] and pool.pages(s) == m.pages[s], s


@pytest.mark.parametrize("seed", range(6))
def test_bookkeeping_follows_the_model(seed):
    r = random.Random(seed)
    pages, slots, per = r.choice([5, 64, 65, 200]), r.choice([1, 3, 17]), r.choice([1, 4, 30])
    pool, m = kv4.KvPool(2, 2, 64, pages, slots, per, device=-1), Model(pages, slots, per)
    for _ in range(300):
        what, s = r.choice(["extend", "extend", "fork", "truncate", "free", "compact"]), r.randrange(slots)
        if what == "extend":
            n = r.choice([0, 1, 2, 63, 64, 65, r.randint(0, 300)])
            if m.len[s] + n > per * PAGE or m.need(s, n) > m.ref.count(0):
                with pytest.raises(engine.EngineError, match="cannot grow|no free page"):
                    pool.extend([s], [n])
            else:
                pool.extend([s], [n])
                m.extend(s, n)
        elif what == "fork":
            d = r.randrange(slots)
            if d == s or m.len[d]:
                with pytest.raises(engine.EngineError, match="not empty"):
                    pool.fork([s], [d])
            else:
                pool.fork([s], [d])
                m.fork(s, d)
        elif what == "truncate":
            n = r.randint(0, m.len[s])
            pool.truncate([s], [n])
            m.truncate(s, n)
        elif what == "free":
            pool.free([s, s])
            m.truncate(s, 0)
        else:
            assert pool.compact() == m.compact()
        same(pool, m)


def test_lists_run_in_order_and_fail_whole():
    pool, m = kv4.KvPool(1, 1, 64, 6, 4, 8, device=-1), Model(6, 4, 8)
    pool.extend([0, 0, 1], [10, 60, 64])             # one slot twice: 70 positions
    for s, n in ((0, 10), (0, 60), (1, 64)):
        m.extend(s, n)
    pool.fork([0, 2], [2, 3])                        # a copy, and a copy of the copy
    m.fork(0, 2), m.fork(2, 3)
    same(pool, m)
    with pytest.raises(engine.EngineError, match="no free page for sequence 0"):
        pool.extend([2, 3, 0, 1, 0], [1, 1, 1, 64, 200])    # the last one does not fit: nothing is done
    same(pool, m)
    with pytest.raises(engine.EngineError, match="not empty"):
        pool.fork([0, 0], [1, 2])
    with pytest.raises(engine.EngineError, match="no sequence 4"):
        pool.truncate([0, 4], [1, 1])
    with pytest.raises(engine.EngineError, match="has 70 positions"):
        pool.truncate([1, 0], [3, 71])
    with pytest.raises(engine.EngineError, match="no sequence -1"):
        pool.free([0, -1])
    same(pool, m)
    pool.extend([2, 3, 0], [1, 1, 1])                # two copies; the last holder keeps the page
    for s in (2, 3, 0):
        m.extend(s, 1)
    same(pool, m)


def test_open_refuses():
    ok = dict(n_layer=1, n_head_kv=2, head_dim=64, n_pages=4, n_seq=2, max_pages=2, device=-1)
    kv4.KvPool(**ok).close()
    for k, v in (("n_layer", 0), ("n_head_kv", 0), ("head_dim", 48), ("head_dim", 256), ("n_pages", 0), ("n_seq", 0),
                 ("n_seq", 70000), ("max_pages", 0), ("max_pages", 1 << 30)):
        with pytest.raises(engine.EngineError):
            kv4.KvPool(**{**ok, k: v})
    with pytest.raises(engine.EngineError, match="not available"):
        kv4.KvPool(**{**ok, "device": 99})
    h = C.c_void_p()
    err = C.create_string_buffer(200)
    assert engine.lib().ecu_kv_open(C.byref(h), 1, 1, 64, 1, 1, 1, -1, 24, err, 200) == -1 and b"aligned" in err.value
    assert engine.lib().ecu_kv_open(None, 1, 1, 64, 1, 1, 1, -1, None, err, 200) == -1
    assert kv4.page_bytes(8, 128) == 72 * 128 * 8 and kv4.page_bytes(8, 80) == 0
    L = engine.lib()
    assert L.ecu_kv_get_info(None, None) == -1 and L.ecu_kv_len(None, 0, None, 0) == -1
    for f in (L.ecu_kv_extend, L.ecu_kv_fork, L.ecu_kv_truncate):
        assert f(None, None, None, 0, None) == -1
    assert L.ecu_kv_free(None, None, 0, None) == -1 and L.ecu_kv_compact(None, None) == -1
    L.ecu_kv_close(None)


A = 0x10000                                          # an address that no call here reads


def ints(*v):
    return np.array(v, dtype=np.int32)


def append(pool, layer=0, dtype=0, k=A, v=A, ks=128, vs=128, seq=(0,), n_new=(1,), n=None, od=0, ko=None, vo=None):
    s, c = ints(*seq), ints(*n_new)
    return engine.lib().ecu_kv_append(pool.h, layer, dtype, k, v, ks, vs, s.ctypes.data, c.ctypes.data,
                                      len(s) if n is None else n, od, ko, vo, None)


@pytest.mark.parametrize("over, why", [
    (dict(layer=2), "layer 2 of 2"), (dict(layer=-1), "layer -1"), (dict(dtype=3), "unknown element type"),
    (dict(od=7), "unknown element type"), (dict(seq=(4,)), "no sequence 4"), (dict(seq=(-1,)), "no sequence -1"),
    (dict(seq=(0, 0), n_new=(1, 1)), "comes twice"), (dict(n_new=(71,)), "71 rows for sequence 0 of 70"),
    (dict(n_new=(-1,)), "-1 rows"), (dict(seq=(2,), n_new=(6,)), "other sequences hold"), (dict(k=0), "null rows"),
    (dict(n_new=(2,), ks=127), "rows overlap"), (dict(k=A + 2), "not aligned"), (dict(ko=A), "one of k_out and v_out"),
    (dict(ko=A, vo=A + 1), "not aligned"), (dict(n=-1), "negative count"), (dict(), "no device")])
def test_append_refuses(over, why):
    pool = kv4.KvPool(2, 2, 64, 8, 4, 4, device=-1)
    pool.extend([0, 1], [70, 70])
    pool.fork([1], [2])
    pool.extend([2], [5])                            # its own copy of the second page, the first page shared
    pool.fork([2], [3])
    assert append(pool, **over) == -1
    assert why in engine.last_error()


def test_append_to_own_pages_only():
    """The positions from a shared page on are refused until an extend has made the page the sequence's own."""
    pool = kv4.KvPool(1, 1, 64, 8, 2, 4, device=-1)
    pool.extend([0], [60])
    pool.fork([0], [1])
    assert append(pool, seq=(1,), n_new=(1,)) == -1 and "other sequences hold" in engine.last_error()
    pool.extend([1], [1])
    for s in (0, 1):
        assert append(pool, seq=(s,), n_new=(1,)) == -1 and "no device" in engine.last_error()
    assert append(pool, seq=(0, 1), n_new=(0, 0)) == 0      # no rows: nothing to do


def attend(pool, layer=0, dtype=0, q=A, out=A, heads=4, qs=256, os=256, seq=(0,), n=None, scale=0.1, ws=None):
    s = ints(*seq)
    return engine.lib().ecu_kv_attend(pool.h, layer, dtype, q, out, heads, qs, os, s.ctypes.data,
                                      len(s) if n is None else n, scale, ws, None)


@pytest.mark.parametrize("over, why", [
    (dict(layer=1), "layer 1 of 1"), (dict(dtype=-1), "unknown element type"), (dict(heads=3), "3 query heads"),
    (dict(heads=0), "0 query heads"), (dict(seq=(2,)), "no sequence 2"), (dict(q=0), "null rows"),
    (dict(out=0), "null rows"), (dict(seq=(0, 1), qs=255), "rows overlap"), (dict(q=A + 1), "not aligned"),
    (dict(ws=A + 8), "not aligned"), (dict(scale=float("nan")), "not finite"), (dict(n=-2), "negative count"),
    (dict(), "no device")])
def test_attend_refuses(over, why):
    pool = kv4.KvPool(1, 2, 64, 8, 2, 4, device=-1)
    assert attend(pool, **over) == -1
    assert why in engine.last_error()
    assert attend(pool, seq=()) == 0


def test_null_list_is_the_first_slots():
    pool = kv4.KvPool(1, 2, 64, 8, 2, 4, device=-1)
    L = engine.lib()
    assert L.ecu_kv_attend(pool.h, 0, 0, A, A, 4, 256, 256, None, 3, 0.1, None, None) == -1
    assert "3 sequences of 2 slots" in engine.last_error()


def prompt(dtype=1, q=A, k=A, v=A, out=A, heads=4, kv=2, hd=64, st=(256, 128, 128, 256), cu_q=(0, 5), cu_k=None, n=None,
           scale=0.1, device=99):
    cq = ints(*cu_q)
    ck = None if cu_k is None else ints(*cu_k)
    return engine.lib().ecu_attn_prompt(dtype, q, k, v, out, heads, kv, hd, *st, cq.ctypes.data,
                                        None if ck is None else ck.ctypes.data, len(cq) - 1 if n is None else n, scale,
                                        device, None)


@pytest.mark.parametrize("over, why", [
    (dict(dtype=0), "ECU_F16 or ECU_BF16"), (dict(hd=96), "head_dim 96"), (dict(heads=5), "5 query heads"),
    (dict(kv=0), "0 KV heads"), (dict(cu_q=(1, 5)), "begin at 0"), (dict(cu_q=(0, 5, 4)), "decrease"),
    (dict(cu_q=(0, 5), cu_k=(0, -1)), "decrease"), (dict(q=0), "null rows"), (dict(v=0), "null rows"),
    (dict(st=(248, 128, 128, 256)), "rows overlap"), (dict(st=(256, 120, 128, 256)), "rows overlap"),
    (dict(st=(260, 128, 128, 256)), "not 16-byte aligned"), (dict(k=A + 8), "not 16-byte aligned"),
    (dict(scale=float("inf")), "positive finite"), (dict(scale=0.0), "positive finite"), (dict(n=-1), "negative count"),
    (dict(), "device 99 not available")])
def test_prompt_refuses(over, why):
    assert prompt(**over) == -1
    assert why in engine.last_error()


def test_prompt_of_nothing():
    assert prompt(cu_q=(0,)) == 0 and prompt(cu_q=(0, 0, 0), cu_k=(0, 3, 3)) == 0


def test_open_refuses_pools_past_64_bits():
    """Pages whose bytes pass 2^64 are no pool of what is left of them."""
    with pytest.raises(engine.EngineError, match="too large"):
        kv4.KvPool(65535, 4096, 128, 2 ** 31 - 1, 1, 1, device=-1)


def test_attend_refuses_rows_past_32_bits():
    pool = kv4.KvPool(1, 4096, 128, 1, 1, 1, device=-1)
    assert attend(pool, heads=4096 * 4096) == -1 and "16777216 query heads" in engine.last_error()


def test_numbers_past_32_bits():
    """ctypes passes the low 32 bits of a number: such ones are refused, not taken for others."""
    big = 1 << 32
    for at in range(7):
        size = [1, 2, 64, 8, 2, 4, -1]
        size[at] += big
        with pytest.raises(engine.EngineError):
            kv4.KvPool(*size[:6], device=size[6])
    pool = kv4.KvPool(1, 2, 64, 8, 2, 4, device=-1)
    pool.extend([0], [5])
    for f in (lambda: pool.length(big), lambda: pool.pages(big), lambda: pool.extend([big], [1]), lambda: pool.extend([0], [big + 1]),
              lambda: pool.read(0, 0, big, 1), lambda: pool.read(big, 0), lambda: kv4.page_bytes(big + 2, 64),
              lambda: pool.free(np.array([big], dtype=np.int64)), lambda: pool.truncate([0], [big])):
        with pytest.raises(engine.EngineError):
            f()
    assert pool.length(0) == 5


def test_prompt_status_refuses_devices():
    L = engine.lib()
    assert L.ecu_attn_prompt_status(99, None) == -1 and "not available" in engine.last_error()
    assert L.ecu_attn_prompt_status(-1, None) == -1
    for d in (-1, 32):
        with pytest.raises(engine.EngineError):
            engine.inject_prompt_timeout(d)


@pytest.mark.parametrize("seed", range(4))
def test_a_change_whose_launch_fails_is_taken_back(seed):
    """Every kind of change, its device update refused, leaves tables, lengths and the pages that come next as they were."""
    r = random.Random(100 + seed)
    pages, slots, per = r.choice([40, 70, 200]), 9, 12
    pool, m = kv4.KvPool(2, 2, 64, pages, slots, per, device=-1), Model(pages, slots, per)
    failed = {k: 0 for k in ("extend", "fork", "truncate", "free", "compact")}
    for _ in range(400):
        what, s = r.choice(list(failed) + ["extend"]), r.randrange(slots)
        if what == "extend":
            n = r.choice([1, 2, 64, 65, r.randint(1, 300)])
            if m.len[s] + n > per * PAGE or m.need(s, n) > m.ref.count(0):
                continue
            call, do = (lambda: pool.extend([s], [n])), (lambda: m.extend(s, n))
        elif what == "fork":
            d = r.randrange(slots)
            if d == s or m.len[d] or not m.len[s]:
                continue
            call, do = (lambda: pool.fork([s], [d])), (lambda: m.fork(s, d))
        elif what == "compact":
            if not any(m.ref[p] and p >= sum(x > 0 for x in m.ref) for p in range(pages)):
                continue
            call, do = pool.compact, m.compact
        else:
            if not m.len[s]:
                continue
            n = 0 if what == "free" else r.randrange(m.len[s])
            call, do = (lambda: pool.free([s]) if what == "free" else pool.truncate([s], [n])), (lambda: m.truncate(s, n))
        for _ in range(r.choice([0, 1, 2])):
            pool.inject_failure()
            with pytest.raises(engine.EngineError, match="injected"):
                call()
            failed[what] += 1
            same(pool, m)
        call()
        do()
        same(pool, m)
    assert all(failed.values()), failed


def test_a_change_cut_off_between_launches_ends_the_pool():
    """A later launch of a long list fails: nothing after it works on tables that are neither old nor new."""
    n = 1500                                         # two words a sequence: two launches
    pool = kv4.KvPool(1, 1, 64, 2 * n, n, 2, device=-1)
    with pytest.raises(engine.EngineError):
        pool.inject_failure(-1)
    pool.inject_failure(2)
    pool.extend(range(n), [1] * n)                   # has no third launch
    pool.extend([0], [1])
    pool.inject_failure(1)
    with pytest.raises(engine.EngineError, match="injected"):
        pool.free(range(n))
    for f in (lambda: pool.extend([0], [1]), lambda: pool.fork([0], [1]), lambda: pool.truncate([0], [0]), lambda: pool.free([0]),
              pool.compact, lambda: pool.read(0, 0, 0, 0)):
        with pytest.raises(engine.EngineError, match="can only be closed"):
            f()
    for rc in (append(pool, ks=64, vs=64), attend(pool, heads=1, qs=64, os=64)):
        assert rc == -1 and "can only be closed" in engine.last_error()
    pool.length(0), pool.used
    pool.close()
