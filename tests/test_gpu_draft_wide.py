"""Steps with drafted tokens in 16 bits and of many columns, where the attention
runs on tensor memory, by the forms and tolerances of test_gpu_draft.py: which
kernel ran is asserted, the calls are captured, run on several streams, far
into memory and in a run of steps.  And what a rotated append hands back, in
every pair of types."""
import numpy as np
import pytest
import torch

from distcomp_b200 import draft, engine, kv4
from test_gpu_draft import PAGE, TYPES, _quiet, freq_of, held, make, random_tree, same, tree_check, turned, verify_plain  # noqa: F401
from test_gpu_kv4 import H16, filled, rows, stored

pytestmark = pytest.mark.gpu

WIDE = [(hd, dtype) for hd in (64, 128) for dtype in TYPES[1:]]
KV, REP = 8, 8


def on_tensor_memory(call):
    """A call's rows, which the kernel on tensor memory has to have made: the other one's, of the same call, differ in
    their last bits (keys and values are rounded in the first alone)."""
    engine.inject_tree_registers()
    other = call().clone()
    got = call().clone()
    torch.cuda.synchronize()
    assert not torch.equal(got, other), "the call did not run on tensor memory"
    return got


@pytest.mark.parametrize("hd,dtype", WIDE)
def test_a_build_with_other_registers(hd, dtype):
    """Where the kernel on tensor memory was compiled to other registers than its roles share, the other one takes the
    call; the next one is on tensor memory again."""
    lens, new = [700, 200, 1000, 64] * 3, [16, 24, 9, 40] * 3
    pool, vals = filled(KV, hd, lens, 3)
    masks, mask = make(8, new)
    q = rows(5, sum(new), KV * REP, hd).to(dtype)
    engine.inject_tree_registers()
    got = pool.attend_tree(0, q, range(12), new, mask)
    tree_check(pool, vals, q, range(12), new, masks, got, every=13)
    again = pool.attend_tree(0, q, range(12), new, mask)
    tree_check(pool, vals, q, range(12), new, masks, again, every=13)
    assert not torch.equal(got, again)
    with pytest.raises(engine.EngineError):
        engine.inject_tree_registers(-1)


@pytest.mark.parametrize("hd,dtype", WIDE)
def test_captured_follows_the_lengths(hd, dtype):
    """append_rope and attend_tree in two graphs with workspaces of their own, replayed at other lengths than those at
    the capture: around the borders of pages and units, nothing but the drafts, and longer than before."""
    new, seq = [40, 24, 30, 33], [2, 0, 3, 1]
    total = sum(new)
    pool = kv4.KvPool(1, KV, hd, 200, 4, 48)
    parents = [random_tree(np.random.default_rng(i), m) for i, m in enumerate(new)]
    depth, mask = draft.tree(parents)
    masks = [[int(x) for x in draft.tree(p, device=None)[1].view(np.uint64)] for p in parents]
    rope, f = draft.Rope(hd), freq_of(hd)
    q, k, v = (torch.zeros(total, h, hd, device="cuda", dtype=dtype) for h in (REP * KV, KV, KV))
    s = torch.cuda.Stream()

    def step(lens, seed):
        """The sequences at these lengths, and rows to put at their ends."""
        pool.truncate(seq, [0] * 4)
        pool.extend(seq, lens)
        pool.append(0, rows(seed, sum(lens), KV, hd).to(dtype), rows(seed + 1, sum(lens), KV, hd, spread=0.3).to(dtype), seq, lens)
        for i, t in enumerate((q, k, v)):
            t.copy_(rows(seed + 2 + i, *t.shape, spread=[1.5, 1.0, 0.3][i]))
        torch.cuda.synchronize()

    def graph(out, ws):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            tq = pool.append_rope(0, rope, q, k, v, seq, new, depth=depth)
            pool.attend_tree(0, tq, seq, new, mask, out=out, ws=ws)
        return g, tq

    step([2900, 1300, 2600, 2500], 1)
    wss = [pool.tree_workspace() for _ in range(3)]  # (kept as long as the graphs)
    for ws in wss:
        ws.fill_(255)
    outs = [torch.zeros_like(q) for _ in range(3)]
    engine.inject_tree_registers()
    other = graph(outs[2], wss[2])
    graphs = [graph(o, ws) for o, ws in zip(outs[:2], wss)]
    for g, _ in [other] + graphs:
        g.replay()
    torch.cuda.synchronize()
    assert not torch.equal(outs[2], outs[0])          # (made on tensor memory: the other kernel's differ)
    for i, lens in enumerate(([2900, 1300, 2600, 2500], [64, 128, 30, 33], [65, 129, 127, 63], [191, 192, 193, 257], new, [2944, 30, 3000, 64])):
        step(lens, 10 * i + 7)
        for o in outs:
            o.fill_(77.0)
        for g, _ in graphs + [other]:
            g.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1])
        vals = {x: tuple(y.astype(np.float64) for y in pool.read(0, x)) for x in seq}
        pos = np.concatenate([n - m + np.array(draft.tree(p, device=None)[0]) for n, m, p in zip(lens, new, parents)])
        wk, r = held(turned(k.double().cpu().numpy(), pos, f, 1.0, False)[0]), np.cumsum([0] + new)
        for j, x in enumerate(seq):
            same(vals[x][0][-new[j]:], wk[r[j]:r[j + 1]])
        for (_, tq), o in zip([graphs[0], other], (outs[0], outs[2])):
            tree_check(pool, vals, tq, seq, new, masks, o, every=17)


@pytest.mark.parametrize("hd,dtype", WIDE)
def test_on_many_streams(hd, dtype):
    """Calls on streams of their own, which may run at the same time: the bits of a call alone."""
    new = [40, 50]
    pool, vals = filled(KV, hd, [5000, 4500], 3)
    masks, mask = make(3, new)
    q = rows(4, sum(new), KV * REP, hd).to(dtype)
    want = on_tensor_memory(lambda: pool.attend_tree(0, q, [0, 1], new, mask))
    tree_check(pool, vals, q, [0, 1], new, masks, want, every=19)
    streams, outs = [torch.cuda.Stream() for _ in range(18)], []       # more than the pool keeps workspaces for
    for _ in range(2):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            outs.append(torch.zeros_like(q))
            pool.attend_tree(0, q, [0, 1], new, mask, out=outs[-1], stream=s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    pool.close()


def test_beyond_32_bits():
    """Pages further than 4 GB into the layer."""
    hd, n = 128, 6000
    far = (5 << 30) // kv4.page_bytes(KV, hd)
    pool = kv4.KvPool(1, KV, hd, far + 100, 2, far)
    pool.extend([0, 1], [far * PAGE, n])
    k, v, q = rows(1, n, KV, hd), rows(2, n, KV, hd), rows(3, 40, KV * REP, hd).bfloat16()
    pool.append(0, k, v, [1], [n])
    assert min(pool.pages(1)) >= far
    masks, mask = make(3, [40])
    got = on_tensor_memory(lambda: pool.attend_tree(0, q, [1], [40], mask))
    tree_check(pool, {1: (stored(k), stored(v))}, q, [1], [40], masks, got, every=19)


@pytest.mark.parametrize("hd,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_more_sequences_than_a_short_list(hd, dtype):
    """More than the 64 that a launch's short list holds, lengths of 0 and 1 and sequences without rows among them."""
    r, n = np.random.default_rng(hd), 150
    lens = [int(x) for x in r.integers(1, 400, n)]
    lens[3], lens[77] = 1, 0
    new = [int(min(l, x)) for l, x in zip(lens, r.integers(0, 24, n))]
    pool, vals = filled(KV, hd, lens, 3)
    masks, mask = make(3, new)
    q = rows(4, sum(new), KV * REP, hd).to(dtype)
    out = torch.full((sum(new) + 1, KV * REP, hd), 77.0, dtype=dtype, device="cuda")
    got = on_tensor_memory(lambda: pool.attend_tree(0, q, None, new, mask, out=out[:-1]))
    tree_check(pool, vals, q, range(n), new, masks, got, every=31)
    assert (out[-1] == 77).all()


@pytest.mark.parametrize("hd,dtype", WIDE)
def test_a_large_draft_beside_small_rows(hd, dtype):
    """A draft of values past 2^15 takes its unit's keys and values 2^-4 smaller for all rows, those that do not see it
    too.  An operand is (code - 8) * scale, both rounded to multiples of 2^-24 where they are that small: by half of one
    8 times and once more, 9 * 2^-25, which is 9 * 2^-21 of what it stands for.  Rows that do not see the draft are off
    by no more than that beside what test_gpu_draft.py allows; those that see it are as ever."""
    count, n, m, delta = 8, 150, 64, 9 * 2.0 ** -21
    pool = kv4.KvPool(1, KV, hd, 3 * count, count, 3)
    pool.extend(range(count), [n] * count)
    k, v = rows(1, n, KV, hd) * 2.0 ** -13, rows(2, n, KV, hd) * 2.0 ** -14
    k[-3], v[-3] = rows(3, KV, hd) * 30000.0, rows(4, KV, hd) * 30000.0
    for s in range(count):
        pool.append(0, k, v, [s], [n])
    kn, vn = stored(k), stored(v)
    masks = [(1 << j + 1) - 1 & ~(1 << m - 3) for j in range(m)]
    masks[m - 2] = 1 << m - 3                         # sees the large one, and the cached positions
    mask = torch.from_numpy(np.array(masks * count, dtype=np.uint64).view(np.int64)).cuda()
    q = rows(5, m * count, KV * REP, hd).to(dtype) * 1024
    got = on_tensor_memory(lambda: pool.attend_tree(0, q, range(count), [m] * count, mask)).double().cpu().numpy()
    scale, half, worst, qn = hd ** -0.5, torch.finfo(dtype).eps / 2, 0.0, q.double().cpu().numpy()
    for s in (0, count - 1):
        for j in [x for x in range(m) if x != m - 2]:
            see = np.ones(n, bool)
            see[n - m:] = [masks[j] >> t & 1 for t in range(m)]
            for h in range(0, KV * REP, 9):
                kk, vv, x = kn[see, h // REP], vn[see, h // REP], qn[s * m + j, h]
                sc = kk @ x * scale
                p = np.exp(sc - sc.max())
                p /= p.sum()
                want = p @ vv
                ds = scale * (np.max(np.abs(kk) @ np.abs(x)) * (2.0 ** -23 * (hd / 2 + 16) + H16) + np.abs(x).sum() * delta) + 2.0 ** -20
                tol = np.abs(vv).max() * (2 * ds + 2.0 ** -23 * (n / 16 + 64) + 2.0 ** -24) + 2 * H16 * (p @ np.abs(vv)) + delta + half * np.abs(want)
                if dtype == torch.float16:
                    tol = tol + 2.0 ** -25            # half a step of small results
                worst = max(worst, (np.abs(got[s * m + j, h] - want) / tol).max())
    assert worst <= 1.0, worst
    if dtype == torch.bfloat16:                       # (fp16 ends at 65504)
        assert np.isfinite(got).all()


@pytest.mark.parametrize("hd,dtype", [(64, torch.float16), (128, torch.bfloat16)])
def test_a_run_of_steps(hd, dtype):
    """Steps as a server takes them: extend, rotate and append, attend, verify, keep.  The cache then holds what
    appending the accepted tokens one by one would have left."""
    vocab, slots = 300, [2, 0, 1]
    r = np.random.default_rng(hd)
    rope = draft.Rope(hd, base=500000.0, scaling="yarn", factor=4.0, context=512.0)
    pool, single = (kv4.KvPool(1, KV, hd, 100, 3, 30) for _ in range(2))
    emb = [torch.from_numpy(r.standard_normal((vocab, h, hd)).astype(np.float32)).to(dtype).cuda() for h in (REP * KV, KV, KV)]
    last = {s: int(r.integers(vocab)) for s in slots}
    for s in slots:                                   # something cached already
        n = 1430 + 30 * s
        tok = torch.from_numpy(r.integers(0, vocab, n)).cuda()
        for p in (pool, single):
            p.extend([s], [n])
            p.append_rope(0, rope, None, emb[1][tok], emb[2][tok], [s], [n])
    for step in range(6):
        new = [int(x) for x in r.integers(28, 44, 3)]
        parents = [[-1] + [max(p, 0) for p in random_tree(r, n)[1:]] for n in new]
        tokens = [[last[s]] + [int(x) for x in r.integers(0, vocab, n - 1)] for s, n in zip(slots, new)]
        depth, mask = draft.tree(parents)
        tok = torch.tensor([t for ts in tokens for t in ts], device="cuda")
        pool.extend(slots, new)
        q = emb[0][tok]
        assert pool.append_rope(0, rope, q, emb[1][tok], emb[2][tok], slots, new, depth=depth, q_out=q) is q
        out = on_tensor_memory(lambda: pool.attend_tree(0, q, slots, new, mask))
        vals = {s: tuple(x.astype(np.float64) for x in pool.read(0, s)) for s in slots}
        masks = [[int(x) for x in draft.tree(p, device=None)[1].view(np.uint64)] for p in parents]
        tree_check(pool, vals, q, slots, new, masks, out, every=29)
        logits = (out.flatten(1)[:, :vocab] * 8).to(dtype)
        u, un = (torch.from_numpy(r.random(m, dtype=np.float32)).cuda() for m in (sum(new), 3))
        temp = torch.tensor([0.0 if step % 3 == 0 else 2.0, 4.0, 1.0], device="cuda")
        flat, first = [p for t in parents for p in t], np.cumsum([0] + new)
        kept, n_kept, nxt = draft.verify(logits, tok.int(), torch.tensor(flat, dtype=torch.int32, device="cuda"), new, u, un, temperature=temp)
        want = verify_plain(logits.double().cpu().numpy(), tok.cpu().numpy(), flat, new, u.double().cpu().numpy(), un.double().cpu().numpy(),
                            temp.double().cpu().numpy(), None)
        assert kept.tolist() == want[0] and n_kept.tolist() == want[1] and nxt.tolist() == want[2]
        paths = []
        for i, n in enumerate(new):                   # (whatever was accepted, a path of the tree is kept: here or there another)
            path = kept[first[i]:first[i] + int(n_kept[i])].tolist()
            if step % 2:
                j, path = n - 1, []
                while j >= 0:
                    path.insert(0, j)
                    j = parents[i][j]
            paths.append(path)
        pool.keep(slots, new, paths)
        for s, path, ts, x in zip(slots, paths, tokens, nxt.tolist()):
            for j in path:
                t = torch.tensor([ts[j]], device="cuda")
                single.extend([s], [1])
                single.append_rope(0, rope, None, emb[1][t], emb[2][t], [s], [1])
            last[s] = x
    for s in slots:
        assert pool.length(s) == single.length(s)
        for a, b in zip(pool.read(0, s), single.read(0, s)):
            assert np.array_equal(a, b)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("out_dtype", TYPES)
def test_rows_handed_back_in_every_type(dtype, out_dtype):
    """What the cache holds, rounded once to the type that is asked for; 16-bit outputs in wide and in odd places."""
    hd, n_kv, new = 96, 3, [70, 5]
    rope, f, n = draft.Rope(hd, rot=64), freq_of(64), sum(new)
    k, v = rows(1, n, n_kv, hd).to(dtype), rows(2, n, n_kv, hd).to(dtype)
    pos = np.concatenate([np.arange(m) for m in new])
    want = [torch.from_numpy(held(x)).to(out_dtype) for x in (turned(k.double().cpu().numpy(), pos, f, 1.0, False)[0], v.double().cpu().numpy())]
    for odd in (0, 1):
        pool = kv4.KvPool(1, n_kv, hd, 4, 2, 2)
        pool.extend([0, 1], new)
        base = [torch.full((n * n_kv * hd + 8,), 7.0, dtype=out_dtype, device="cuda") for _ in range(2)]
        ko, vo = (b[odd:odd + n * n_kv * hd].view(n, n_kv, hd) for b in base)
        pool.append_rope(0, rope, None, k, v, [0, 1], new, k_out=ko, v_out=vo)
        assert torch.equal(ko.cpu(), want[0]) and torch.equal(vo.cpu(), want[1])
        assert all((b[:odd] == 7).all() and (b[odd + n * n_kv * hd:] == 7).all() for b in base)
