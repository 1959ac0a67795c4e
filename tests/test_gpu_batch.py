"""Many sequences over one model (ecu_batch): prompts, single tokens, forks and
the pool's upkeep against a plain 64-bit forward of the same model whose keys
and values go through the cache's 4-bit definition.

The bar: the GEMMs keep about 22 bits, the prompt attention's operands 11
(2^-12 of each element, averaged over keys and dimensions), so states agree to
a few 1e-4 of the vector's scale; where a key or value lies that near to the
border of two codes it may take the other one, a step of 1/8 of its block's
largest value in one of thousands of products.  1e-2 of the scale covers both;
the 4-bit cache itself moves these logits by more, which the test checks too.
"""
import numpy as np
import pytest

from distcomp_b200 import gguf as G
from distcomp_b200 import synth
from test_gpu_kv4 import stored

pytestmark = pytest.mark.gpu
REL = 1e-2


class Plain:
    """A llama forward in 64 bits; 4-bit keys and values unless told otherwise."""

    def __init__(self, spec, buf, port, four_bits=True):
        self.s, self.port, self.four = spec, port, four_bits
        self.tab = G.read_tensor_table(buf)
        self.dims = {name: (dims, t) for name, dims, t in synth.tensor_list(self.s)}
        self.w = {}

    def weight(self, name):
        if name not in self.w:
            dims, t = self.dims[name]
            n = int(np.prod(dims))
            rc, v = self.port.dequant(t, np.frombuffer(self.tab[name][2], np.uint8), n, 0, n)
            assert rc == 0
            self.w[name] = np.asarray(v, dtype=np.float64).reshape(dims[::-1])
        return self.w[name]

    def keep(self, x):
        import torch
        return stored(torch.from_numpy(x.astype(np.float32))) if self.four else x

    def forward(self, tokens, cache=None):
        """Logits of every position of `tokens` after those in `cache` (grown in place)."""
        s = self.s
        hd, H, KV = s.head_dim or s.n_embd // s.n_head, s.n_head, s.n_head_kv
        cache = {} if cache is None else cache
        x = self.weight("token_embd.weight")[list(tokens)]
        pos0 = len(cache.get((0, "k"), ()))
        pos = pos0 + np.arange(len(tokens))
        ang = pos[:, None] * s.rope_base ** (-2.0 * np.arange(hd // 2) / hd)[None]
        c, sn = np.cos(ang)[:, None], np.sin(ang)[:, None]

        def norm(x):
            return x / np.sqrt((x * x).mean(-1, keepdims=True) + s.eps)

        def turn(x):
            a, b = x[..., :hd // 2], x[..., hd // 2:]
            return np.concatenate([a * c - b * sn, b * c + a * sn], -1)

        for l in range(s.n_layer):
            y = norm(x) * self.weight(f"blk.{l}.attn_norm.weight")
            q, k, v = (y @ self.weight(f"blk.{l}.attn_{n}.weight").T for n in "qkv")
            if s.qkv_bias:
                q, k, v = (x + self.weight(f"blk.{l}.attn_{n}.bias") for x, n in zip((q, k, v), "qkv"))
            q, k, v = turn(q.reshape(-1, H, hd)), turn(k.reshape(-1, KV, hd)), v.reshape(-1, KV, hd)
            for n, r in (("k", k), ("v", v)):
                old = cache.get((l, n))
                cache[(l, n)] = self.keep(r) if old is None else np.concatenate([old, self.keep(r)])
            K, V = cache[(l, "k")], cache[(l, "v")]
            o = np.empty_like(q)
            seen = np.arange(len(K))[None] <= pos[:, None]
            for h in range(H):
                w = np.where(seen, q[:, h] @ K[:, h // (H // KV)].T / np.sqrt(hd), -np.inf)
                w = np.exp(w - w.max(1, keepdims=True))
                o[:, h] = w @ V[:, h // (H // KV)] / w.sum(1, keepdims=True)
            x = x + o.reshape(len(tokens), -1) @ self.weight(f"blk.{l}.attn_output.weight").T
            y = norm(x) * self.weight(f"blk.{l}.ffn_norm.weight")
            g, u = y @ self.weight(f"blk.{l}.ffn_gate.weight").T, y @ self.weight(f"blk.{l}.ffn_up.weight").T
            x = x + (g / (1 + np.exp(-g)) * u) @ self.weight(f"blk.{l}.ffn_down.weight").T
        return (norm(x) * self.weight("output_norm.weight")) @ self.weight("token_embd.weight" if s.tied else "output.weight").T


def close(got, want, rel=REL):
    err = float(np.max(np.abs(got.astype(np.float64) - want)) / np.max(np.abs(want)))
    assert err <= rel, f"off by {err:.2e} of the scale"
    return err


@pytest.fixture(scope="module")
def setup(eng, oracle_port, model_buf):
    def get(key, **over):
        buf, spec = model_buf(key, **over), synth.spec(key, **over)
        base = eng.LlmCtx(eng.GgufModel(buf), eng.STAGE_FULL)
        return base, Plain(spec, buf, oracle_port), Plain(spec, buf, oracle_port, four_bits=False)
    return get


@pytest.mark.parametrize("key", ["mini-q4", "mini-q8", "mini-q4k"])
def test_feed_matches_the_plain_forward(eng, setup, key):
    """Prompts of different lengths in one call, then single tokens and prompt pieces mixed, 20 steps of them."""
    base, plain, dense = setup(key)
    b = eng.LlmBatch(base, 4, 12)
    r = np.random.default_rng(1)
    V = base.n_vocab
    text = [list(map(int, r.integers(3, V, n))) for n in (40, 1, 17)]
    caches = [{} for _ in text]
    picked, lg = b.feed([2, 0, 1], text, logits=True)
    for i in range(3):
        want = plain.forward(text[i], caches[i])[-1]
        close(lg[i], want)
        assert picked[i] == int(np.argmax(lg[i]))
        far = dense.forward(text[i])[-1]
        if len(text[i]) > 1:
            assert np.max(np.abs(far - want)) / np.max(np.abs(want)) > 1e-3     # the 4-bit cache is in the values
    for step in range(20):
        nxt = [[picked[0]], [int(v) for v in r.integers(3, V, 3)] if step % 5 == 2 else [picked[1]], [picked[2]]]
        picked, lg = b.feed([2, 0, 1], nxt, logits=True)
        for i in range(3):
            close(lg[i], plain.forward(nxt[i], caches[i])[-1])
    assert [b.length(s) for s in (2, 0, 1, 3)] == [60, 29, 37, 0]


def test_biases_and_a_tied_head(eng, setup):
    """A qwen2-style model: Q/K/V biases, the embedding as the head; prompts, and few and many steps."""
    base, plain, _ = setup("mini-q8", arch="qwen2", qkv_bias=True, tied=True)
    n = 18
    b = eng.LlmBatch(base, n, 40)
    r = np.random.default_rng(8)
    text = [[int(v) for v in r.integers(3, base.n_vocab, 2 + i)] for i in range(n)]
    caches = [{} for _ in text]
    for seqs in (range(n), range(n), range(3)):
        toks = [text[i] for i in seqs]
        picked, lg = b.feed(list(seqs), toks, logits=True)
        for i in seqs:
            want = plain.forward(toks[i], caches[i])[-1]
            close(lg[i], want)
            text[i] = [picked[i]]


def test_prompt_pieces_forks_and_upkeep(eng, setup):
    """A prompt in pieces (a later one over a page's border), forks that go different ways, a freed slot fed anew, the
    pool closed up between the steps."""
    base, plain, _ = setup("mini-q4")
    b = eng.LlmBatch(base, 5, 10)
    r = np.random.default_rng(2)
    p = [int(v) for v in r.integers(3, base.n_vocab, 75)]
    b.feed([0], [p[:30]])
    b.feed([0], [p[30:31]])
    picked, lg = b.feed([0], [p[31:]], logits=True)
    cache = {}
    close(lg[0], plain.forward(p, cache)[-1])
    b.fork([0, 0], [3, 1])
    assert b.used() == 2
    tails = {s: [int(v) for v in r.integers(3, base.n_vocab, 6)] for s in (0, 3, 1)}
    caches = {s: dict(cache) for s in tails}
    for j in range(6):
        if j == 3:
            b.truncate([1], [70])
            caches[1] = {k: v[:70] for k, v in caches[1].items()}
        if j == 4:
            b.free([0])
            tails.pop(0)
            assert b.compact() >= 0 and b.used() == 3
            picked, lg = b.feed([0], [p[:5]], logits=True)
            close(lg[0], plain.forward(p[:5])[-1])
        _, lg = b.feed(list(tails), [[t[j]] for t in tails.values()], logits=True)
        for i, s in enumerate(tails):
            close(lg[i], plain.forward([tails[s][j]], caches[s])[-1])


def test_steps_of_many_sequences(eng, setup):
    """More single tokens than go through the projections row by row, forks of one prompt among them, and a prompt
    in the same call."""
    base, plain, _ = setup("mini-q4")
    n = 20
    b = eng.LlmBatch(base, n + 1, 60)
    r = np.random.default_rng(5)
    p = [int(v) for v in r.integers(3, base.n_vocab, 66)]
    cache = {}
    plain.forward(p, cache)
    b.feed([0], [p])
    b.fork([0] * (n - 1), range(1, n))
    tok = [int(v) for v in r.integers(3, base.n_vocab, n)]
    more = [int(v) for v in r.integers(3, base.n_vocab, 9)]
    for seqs, toks in ((list(range(n)), [[t] for t in tok]), (list(range(n + 1)), [[t + 1] for t in tok] + [more])):
        picked, lg = b.feed(seqs, toks, logits=True)
        for i in (0, 1, 7, n - 1):
            c = dict(cache)
            if len(seqs) > n:
                plain.forward([tok[i]], c)
            close(lg[i], plain.forward(toks[i], c)[-1])
            assert picked[i] == int(np.argmax(lg[i]))
    close(lg[n], plain.forward(more)[-1])


def test_feed_refuses_and_keeps_what_it_held(eng, setup):
    base, plain, _ = setup("mini-q4")
    b = eng.LlmBatch(base, 3, 3)
    b.feed([0], [[5] * 60])
    for seq, tok, why in (([0, 0], [[1], [2]], "comes twice"), ([1], [[]], "without tokens"), ([3], [[1]], "no sequence 3"),
                          ([1], [[base.n_vocab]], "outside the vocabulary"), ([0], [[1] * 69], "exceed the context"),
                          ([1, 2], [[1] * 70, [2] * 70], "no free page")):
        with pytest.raises(eng.EngineError, match=why):
            b.feed(seq, tok)
        assert [b.length(s) for s in range(3)] == [60, 0, 0] and b.used() == 1
    assert b.feed([], []) == []
    _, lg = b.feed([0], [[7]], logits=True)
    close(lg[0], plain.forward([5] * 60 + [7])[-1])


def test_batch_refuses_bases(eng, model_buf):
    m = eng.GgufModel(model_buf("tiny"))
    with pytest.raises(eng.EngineError, match="do not cover"):
        eng.LlmBatch(eng.LlmCtx(m, eng.STAGE_FULL), 2, 4)          # head_dim 32
    m4 = eng.GgufModel(model_buf("mini-q4"))
    with pytest.raises(eng.EngineError, match="FULL context"):
        eng.LlmBatch(eng.LlmCtx(m4, eng.STAGE_LAYERS, 0, 1), 2, 4)
    base = eng.LlmCtx(m4, eng.STAGE_FULL)
    for n_seq, n_pages in ((0, 4), (2, 0), (70000, 4)):
        with pytest.raises(eng.EngineError):
            eng.LlmBatch(base, n_seq, n_pages)


def test_batch_outlives_its_base(eng, setup, model_buf):
    base = eng.LlmCtx(eng.GgufModel(model_buf("mini-q4")), eng.STAGE_FULL)
    b = eng.LlmBatch(base, 1, 2)
    first = b.feed([0], [[9, 8, 7]])
    base.close()
    b.free([0])
    assert b.feed([0], [[9, 8, 7]]) == first


@pytest.mark.parametrize("key,n_prompt", [("mini-q4", 100), ("mini-q8", 33), ("mini-q4k", 90)])
def test_prefill_with_tensor_core_attention(eng, model_buf, monkeypatch, key, n_prompt):
    """ECU_PF_ATTN=2 keeps ecu_prefill within its 1e-3 bar of the default, also for a second piece."""
    s = synth.spec(key)
    m = eng.GgufModel(model_buf(key))
    prompt = synth.prompt_tokens(n_prompt, s.n_vocab, seed=4)
    a, b = eng.LlmCtx(m, eng.STAGE_FULL), eng.LlmCtx(m, eng.STAGE_FULL)
    first = a.prefill(prompt)
    want = a.logits().astype(np.float64)
    monkeypatch.setenv("ECU_PF_ATTN", "2")
    b.prefill(prompt[: n_prompt // 3])
    assert b.prefill(prompt[n_prompt // 3:]) == first
    close(b.logits(), want, 1e-3)


def test_batch_refuses_when_closed_and_what_is_no_list(eng, model_buf):
    """A closed batch answers with errors; numbers are not cut to 32 bits or to whole ones."""
    b = eng.LlmBatch(eng.LlmCtx(eng.GgufModel(model_buf("mini-q4")), eng.STAGE_FULL), 2, 4)
    big = 1 << 32
    for f in (lambda: b.feed([big], [[1]]), lambda: b.feed(np.array([big]), [[1]]), lambda: b.feed([0], [np.array([big + 1])]),
              lambda: b.feed([0], [[1.5]]), lambda: b.feed([[0]], [[1]]), lambda: b.length(big), lambda: b.free(np.array([big])),
              lambda: b.truncate([0], [0.5])):
        with pytest.raises(eng.EngineError):
            f()
    b.close()
    for f in (lambda: b.feed([0], [[1]]), lambda: b.fork([0], [1]), lambda: b.truncate([0], [0]), lambda: b.free([0]),
              lambda: b.compact(), lambda: b.length(0), lambda: b.used(), lambda: b.kv):
        with pytest.raises(eng.EngineError):
            f()


class Held(Plain):
    """The plain forward over the rows that a batch's pool holds.  Where a key or value lies within the projections'
    rounding of the border of two codes, either code is right, and the layers after it follow the one taken; so this
    forward takes the pool's, after checking each against its own value: half a code away, a whole one where the code
    ends (7, opposite the largest value), and 5e-3 of the block's largest value for what came before."""

    def __init__(self, plain, eng, batch):
        self.__dict__.update(plain.__dict__)
        self.eng, self.b = eng, batch
        self.hd = self.s.head_dim or self.s.n_embd // self.s.n_head

    def rows(self, seq, layer, pos, n):
        k, v = (np.empty((n, self.s.n_head_kv, self.hd), dtype=np.float32) for _ in range(2))
        assert self.eng.lib().ecu_kv_read(self.b.kv, layer, seq, pos, n, k.ctypes.data, v.ctypes.data, self.b.stream) == 0
        return [x.astype(np.float64) for x in (k, v)]

    def keep(self, x):
        got = self.queue.pop(0)
        m = np.abs(x.reshape(*x.shape[:-1], -1, 32)).max(-1, keepdims=True)
        off = np.abs(got - x).reshape(*x.shape[:-1], -1, 32)
        ends = np.abs(x.reshape(off.shape)) > m * 15 / 16 - 5e-3 * m
        assert (off <= m * (np.where(ends, 1 / 8, 1 / 16) + 5e-3)).all()
        return got

    def last(self, seq, tokens):
        """Logits of the last of `tokens`, a sequence's newest ones, which the pool holds already."""
        past = self.b.length(seq) - len(tokens)
        cache = {}
        self.queue = []
        for l in range(self.s.n_layer):
            for n, old, new in zip("kv", self.rows(seq, l, 0, past), self.rows(seq, l, past, len(tokens))):
                cache[(l, n)] = old
                self.queue.append(new)
        return self.forward(tokens, cache)[-1]


@pytest.mark.parametrize("kv, attn", [(2, None), (4, "0"), (16, "2")])
def test_contexts_of_any_size(eng, setup, monkeypatch, kv, attn):
    """A context past 8192 positions, whatever attention ecu_prefill takes (which the batch does not use): prompts,
    pieces, few and many steps, 8, 4 and 1 query heads a KV head."""
    if attn:
        monkeypatch.setenv("ECU_PF_ATTN", attn)
    base, plain, _ = setup("mini-q8", n_head_kv=kv, n_ff=1024, n_ctx=9000)
    b = eng.LlmBatch(base, 20, 300)
    held = Held(plain, eng, b)
    r = np.random.default_rng(kv)

    def some(n):
        return [int(v) for v in r.integers(3, base.n_vocab, n)]
    text = [some(n) for n in (70, 2, 129)]
    for toks in (text, [some(1), some(3), some(1)], [some(1), some(1), some(1)]):
        _, lg = b.feed([4, 0, 9], toks, logits=True)
        for i, s in enumerate((4, 0, 9)):
            close(lg[i], held.last(s, toks[i]))
    b.fork([4] * 17, [s for s in range(20) if s not in (4, 0, 9)])
    toks = [some(1) for _ in range(20)]
    _, lg = b.feed(range(20), toks, logits=True)
    for s in (4, 0, 9, 19):
        close(lg[s], held.last(s, toks[s]))
    b.free(range(20))
    far = some(8300)
    _, lg = b.feed([0], [far], logits=True)
    close(lg[0], held.last(0, far[-1:]))
    b.feed([1], [far[:8250]])
    _, lg = b.feed([1], [far[8250:]], logits=True)
    close(lg[0], held.last(1, far[8250:]))


@pytest.mark.parametrize("which, rel", [("q", 0.1), ("k", 0.1), ("v", REL)])
def test_values_past_fp16(eng, oracle_port, model_buf, monkeypatch, which, rel):
    """Queries, keys or values of 1e5 (a bias): steps, whose attention is fp32 over the cache's exact values, hold them; a
    prompt or a batch of more steps, whose operands are fp16, fails and leaves the sequences as they were.  (Scores of
    some thousands, 8 * 65504 at most in a key: their fp32 rounding moves a weight by up to some percent.)"""
    over = dict(arch="qwen2", qkv_bias=True)
    buf = np.frombuffer(bytes(model_buf("mini-q4", **over)), np.uint8).copy()
    np.frombuffer(G.read_tensor_table(buf)[f"blk.1.attn_{which}.bias"][2], np.float32)[5] = 1e5
    m = eng.GgufModel(buf)
    base = eng.LlmCtx(m, eng.STAGE_FULL)
    b = eng.LlmBatch(base, 20, 30)
    held = Held(Plain(synth.spec("mini-q4", **over), buf, oracle_port), eng, b)
    r = np.random.default_rng(3)
    toks = [int(t) for t in r.integers(3, base.n_vocab, 24)]
    for i, t in enumerate(toks[:12]):
        _, lg = b.feed([0], [[t]], logits=True)
        assert np.isfinite(lg).all()
        close(lg[0], held.last(0, [t]), rel)
    b.fork([0] * 17, range(1, 18))
    state = [b.length(s) for s in range(20)], b.used()
    for seq, text in (([18], [toks]), ([0], [toks[12:]]), ([0, 18], [toks[12:13], toks])):
        with pytest.raises(eng.EngineError, match="fp16's range"):
            b.feed(seq, text)
        assert [b.length(s) for s in range(20)] == state[0]
    many = list(range(18)), [[toks[12]]] * 18
    if which == "v":
        with pytest.raises(eng.EngineError, match="fp16's range"):
            b.feed(*many)
        assert [b.length(s) for s in range(20)] == state[0]
    else:
        _, lg = b.feed(*many, logits=True)
        close(lg[17], held.last(17, [toks[12]]), rel)
    _, lg = b.feed([3], [[toks[13]]], logits=True)
    close(lg[0], held.last(3, [toks[13]]), rel)
    monkeypatch.setenv("ECU_PF_ATTN", "2")
    with pytest.raises(eng.EngineError, match="fp16's range"):
        base.prefill(toks)


def test_a_prompt_however_it_is_cut(eng, setup):
    """One prompt whole, in pieces and token by token: each agrees with the plain forward over its own pool's rows, and
    the rows with one another to a code (1/8 of their block's largest value; 1e-2 of it for what came before)."""
    base, plain, _ = setup("mini-q4")
    b = eng.LlmBatch(base, 4, 12)
    held = Held(plain, eng, b)
    text = [int(t) for t in np.random.default_rng(12).integers(3, base.n_vocab, 90)]
    for seq, cuts in enumerate(([90], [30, 1, 33, 26], [64, 26], [1] * 90)):
        at = 0
        for n in cuts:
            _, lg = b.feed([seq], [text[at:at + n]], logits=True)
            close(lg[0], held.last(seq, text[at:at + n]))
            at += n
    for layer in range(plain.s.n_layer):
        first = held.rows(0, layer, 0, 90)
        for seq in (1, 2, 3):
            for x, y in zip(first, held.rows(seq, layer, 0, 90)):
                m = np.abs(x).reshape(90, plain.s.n_head_kv, -1, 32).max(-1, keepdims=True)
                assert (np.abs(x - y).reshape(90, plain.s.n_head_kv, -1, 32) <= m * (1 / 8 + 1e-2)).all()
