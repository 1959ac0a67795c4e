"""Cases of the operators that a step with drafted tokens is made of.

Four operators, next to those of ``distcomp_b200.kv4`` that fill and read the
paged 4-bit K/V cache:

  rotate  queries and keys turned by their positions (rotary embedding), the
          keys and values quantised into the cache's pages in the same pass
  tree    attention of several drafted positions per sequence, a tree of them,
          over the sequence's cached positions and the drafted ones
  verify  the drafted tokens held against the target's probabilities with
          given random numbers: the accepted path and the token after it
  keep    the accepted path's rows moved together in the cache, the rest of
          the drafted positions given back

A page holds 64 positions of every KV head of one layer.  Per KV head (72 *
head_dim bytes): K codes of 64 positions, V codes, K scales, V scales.  A
position's codes are head_dim / 32 chunks of 16 bytes, one per block of 32
dimensions in order, low nibble first; chunk b of position t lies at place
b ^ ((t >> 1) & 3) for head_dim 128 and b ^ ((t >> 2) & 1) for 64.  Scales are
fp16 [64][head_dim / 32].  A value is (code - 8) * scale.  A block's scale is
fp16(m / -8), m its value of largest magnitude (the first of equals), its codes
floor(x / scale + 8.5) clamped to 0..15, in exact arithmetic.  Pages are taken
lowest free id first.

Drafts: the newest n positions of a sequence.  Row 0 is the token picked last,
every other row's parent an earlier row; a row stands as many positions behind
the cached ones as it has ancestors, and sees those, itself and what is cached.
"""
import math
import random

import numpy as np
import torch

own = False

PAGE = 64
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# ------------------------------------------------------------------ cases ---

def listed():
    return [
        # one decode step's rows of 64 served sequences, fp32 as the engine's projections leave them
        dict(name="rotate 64x1", op="rotate", n=64, lo=1, hi=1, past=4000, head=32, kv=8, hd=128, rot=128, inter=False, scaling="none",
             base=500000.0, tree=False, dtype="f32", shape=1),
        # packed prompts behind cached ones, far positions of a stretched context, the stored values handed on to the prompt attention
        dict(name="rotate prompts 8k", op="rotate", n=7, lo=200, hi=2100, past=60000, head=32, kv=8, hd=128, rot=128, inter=False,
             scaling="bands", base=500000.0, tree=False, dtype="bf16", shape=2),
        # drafted trees, small heads of which half turns, neighbouring dimensions paired
        dict(name="rotate drafts 24", op="rotate", n=24, lo=3, hi=20, past=2000, head=16, kv=4, hd=64, rot=32, inter=True, scaling="yarn",
             base=10000.0, tree=True, dtype="f16", shape=3),
        # one short chat, a few drafts, as the engine calls it
        dict(name="tree 1x6 of 900", op="tree", n=1, lo=6, hi=6, past_lo=900, past=900, head=32, kv=8, hd=128, dtype="f32", shape=1),
        # a served batch with 8 query heads per KV head (the 70B shape), lengths and trees far apart
        dict(name="tree 32 ragged", op="tree", n=32, lo=1, hi=24, past_lo=1, past=4096, head=64, kv=8, hd=128, dtype="bf16", shape=2),
        # one long document, the widest tree
        dict(name="tree 1x64 of 131k", op="tree", n=1, lo=64, hi=64, past_lo=131025, past=131025, head=32, kv=8, hd=128, dtype="bf16", shape=3),
        # small heads, sequences without drafts or without a past among them
        dict(name="tree 17 hd64", op="tree", n=17, lo=0, hi=16, past_lo=0, past=3000, head=16, kv=4, hd=64, dtype="f16", shape=4),
        # one sequence's chain of five drafts of a deterministic drafter
        dict(name="verify 1x6", op="verify", n=1, lo=6, hi=6, vocab=128256, chain=True, dense=False, greedy=False, dtype="f32", shape=1),
        # a served batch's trees
        dict(name="verify 48 trees", op="verify", n=48, lo=4, hi=16, vocab=128256, chain=False, dense=False, greedy=False, dtype="bf16", shape=2),
        # chains drawn from a small model's distributions
        dict(name="verify 16 drawn", op="verify", n=16, lo=3, hi=8, vocab=32000, chain=True, dense=True, greedy=False, dtype="f32", shape=3),
        # 8 sequences, two layers
        dict(name="keep 8", op="keep", n=8, lo=6, hi=6, past=700, layers=2, kv=8, hd=128, shape=1),
        # a served batch of trees, 32 layers
        dict(name="keep 64 trees", op="keep", n=64, lo=4, hi=24, past=900, layers=32, kv=8, hd=128, shape=2),
    ]


def draw(rng):
    def span(a, b):  # whole numbers, even over the logarithm
        return min(b, max(a, int(round(math.exp(rng.uniform(math.log(a), math.log(b + 0.49)))))))

    hd = rng.choice([64, 128, 128])
    kv = rng.choice([1, 2, 4, 8])
    op = rng.choice(["rotate", "tree", "verify", "keep"])
    shape = rng.randrange(1, 1 << 20)
    if op == "rotate":
        tree = rng.random() < 0.4
        n = span(1, 64)
        hi = max(1, min(span(1, 30 if tree else 1500), 8000 // n))
        rot = rng.choice([hd, hd, hd // 2, 2 * rng.randrange(1, hd // 2 + 1)])
        return dict(op=op, n=n, lo=span(1, hi), hi=hi, past=rng.choice([0, span(1, 100000)]), head=kv * rng.choice([1, 2, 4]), kv=kv, hd=hd,
                    rot=rot, inter=rng.random() < 0.5, scaling=rng.choice(["none", "linear", "bands", "yarn"]),
                    base=rng.choice([10000.0, 500000.0]), tree=tree, dtype=rng.choice(list(TYPES)), shape=shape)
    if op == "tree":
        n = span(1, 40)
        past = span(1, 100000 // n)
        head = kv * rng.choice([1, 2, 3, 4, 6, 8])
        hi = span(1, max(1, min(64, 260000000 // (n * past * head))))
        return dict(op=op, n=n, lo=rng.choice([0, 1, hi]), hi=hi, past_lo=rng.choice([0, past // 2, past]), past=past, head=head, kv=kv, hd=hd,
                    dtype=rng.choice(list(TYPES)), shape=shape)
    if op == "verify":
        n = span(1, 64)
        hi = span(1, max(1, min(24, 768 // n)))
        return dict(op=op, n=n, lo=span(1, hi), hi=hi, vocab=rng.choice([32000, 128256, span(300, 130000)]), chain=rng.random() < 0.4,
                    dense=rng.random() < 0.4, greedy=rng.random() < 0.25, dtype=rng.choice(list(TYPES)), shape=shape)
    n, hi = span(1, 64), span(2, 32)
    return dict(op=op, n=n, lo=rng.choice([1, hi]), hi=hi, past=span(1, 900), layers=span(1, 32), kv=kv, hd=hd, shape=shape)


def lengths(case):
    """(new positions, positions held before) of each sequence, from the case alone."""
    r = random.Random(case["shape"] * 7919 + case["n"])
    new = [r.randint(case["lo"], case["hi"]) for _ in range(case["n"])]
    past = [r.randint(case.get("past_lo", 0), case["past"]) if case.get("past") else 0 for _ in new]
    return new, past


def trees(case):
    """Each sequence's parents: half the rows go on from the newest row, the others branch off an earlier one."""
    r = random.Random(case["shape"] * 104729 + 1)
    out = []
    for n in lengths(case)[0]:
        out.append([-1 if j == 0 else j - 1 if r.random() < 0.5 else r.randrange(max(0, j - 8), j) for j in range(n)])
    return out


def above(parents):
    """(ancestors of each row, as a mask of rows with the row itself, their number without it)"""
    mask, depth = [], []
    for j, p in enumerate(parents):
        mask.append((mask[p] if p >= 0 else 0) | 1 << j)
        depth.append(depth[p] + 1 if p >= 0 else 0)
    return mask, depth


def paths(case):
    """The rows of each sequence that are kept: from row 0 to some row of its tree."""
    r = random.Random(case["shape"] * 15485863 + 2)
    out = []
    for parents in trees(case):
        j, path = r.randrange(len(parents)), []
        while j >= 0:
            path.append(j)
            j = parents[j]
        out.append(path[::-1])
    return out


def pages_of(n):
    return -(-n // PAGE)


def page_bytes(case):
    return 72 * case["hd"] * case["kv"]


def work(case):
    new, past = lengths(case)
    n, rows = case["n"], sum(new)
    size = {"f32": 4, "f16": 2, "bf16": 2}.get(case.get("dtype"), 0)
    if case["op"] == "verify":  # no sequence without its first row's distribution
        return {"bytes": n * case["vocab"] * size + 16 * rows, "flops": 4 * n * case["vocab"]}
    hd, kv = case["hd"], case["kv"]
    if case["op"] == "rotate":  # q, k and v read, q, the stored values and their 4-bit form written
        return {"bytes": rows * hd * (size * (2 * case["head"] + 4 * kv) + 1.125 * kv), "flops": rows * (3 * case["rot"] * (case["head"] + kv) + 6 * hd * kv)}
    if case["op"] == "tree":
        seen = sum(m * p + sum(bin(v).count("1") for v in above(t)[0]) for m, p, t in zip(new, past, trees(case)))
        held = sum(m + p for m, p in zip(new, past) if m)
        return {"bytes": 1.125 * held * kv * hd + 2 * rows * case["head"] * hd * size, "flops": 4 * case["head"] * hd * seen}
    moved = sum(sum(1 for t, j in enumerate(p) if t != j) for p in paths(case))
    return {"bytes": 2 * moved * case["layers"] * kv * hd * 1.125 + 8 * n, "flops": 0}


# ----------------------------------------------------------------- inputs ---

def places(hd):
    """Where chunk b of position t lies, [64][blocks]."""
    nb = hd // 32
    t, b = torch.arange(PAGE, device=DEV)[:, None], torch.arange(nb, device=DEV)[None]
    return b ^ ((t >> 1) & 3) if nb == 4 else b ^ ((t >> 2) & 1) if nb == 2 else b + 0 * t


def to_half(x):
    """64-bit values rounded to fp16 once: through fp32 with the last bit odd where that rounds."""
    f = x.float()
    rest, bits = x - f.double(), f.view(torch.int32)
    odd = bits + torch.where((rest > 0) == (f > 0), 1, -1).to(torch.int32)
    return torch.where((rest != 0) & (bits & 1 == 0) & (f != 0) & rest.isfinite(), odd, bits).view(torch.float32).half()


def quantise(x):
    """Rows [..., hd] as (codes int64 [..., nb, 32], scales fp16 [..., nb])."""
    x = x.double().unflatten(-1, (-1, 32))
    m = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    d = to_half((m / -8).clamp(-65504, 65504))
    d = torch.where(x.isfinite().all(-1, keepdim=True), d, torch.full_like(d, math.nan))
    d = torch.where(d == 0, torch.zeros_like(d), d)
    fine = d.isfinite() & (d != 0)
    q = torch.where(fine, (x / torch.where(fine, d, torch.ones_like(d)).double() + 8.5).floor().clamp(0, 15), torch.full_like(x, 8.0))
    return q.long(), d.squeeze(-1)


def rows_of(gen, n, case, spread=1.0):
    """K or V rows as a projection gives them: normal, a few channels several times larger."""
    x = torch.randn(n, case["kv"], case["hd"], generator=gen, device=DEV)
    big = torch.rand(case["kv"], case["hd"], generator=gen, device=DEV) < 0.03
    return x * torch.where(big, 5.0, 1.0) * spread


def filled(gen, case, pages):
    """`pages` pages of one layer with quantised rows in every position."""
    hd, kv, nb = case["hd"], case["kv"], case["hd"] // 32
    out = torch.empty(max(1, pages), kv, 72 * hd, dtype=torch.uint8, device=DEV)
    at = places(hd)
    for p0 in range(0, pages, 256):
        m = min(256, pages - p0)
        for side in range(2):
            q, d = quantise(rows_of(gen, m * PAGE, case, 1.0 if side == 0 else 0.5).view(m, PAGE, kv, hd).transpose(1, 2))
            b = (q[..., 0::2] | q[..., 1::2] << 4).to(torch.uint8)  # [m, kv, 64, nb, 16]
            c = torch.empty_like(b)
            c.scatter_(3, at[None, None, :, :, None].expand_as(b), b)
            out[p0:p0 + m, :, side * 32 * hd:(side + 1) * 32 * hd] = c.reshape(m, kv, -1)
            out[p0:p0 + m, :, (64 + 4 * side) * hd:(68 + 4 * side) * hd] = d.contiguous().view(torch.uint8).reshape(m, kv, -1)
    return out.view(1, max(1, pages), -1)


def interleaved(lens, step):
    """Sequences that grew in turns: the order in which they take pages, as (sequence, positions) pairs, and the table."""
    width = max(1, max(pages_of(v) for v in lens))
    order, table, held, free = [], [[-1] * width for _ in lens], [0] * len(lens), 0
    while any(h < v for h, v in zip(held, lens)):
        for i, v in enumerate(lens):
            take = min(step, v - held[i])
            if take > 0:
                order.append((i, take))
                for j in range(pages_of(held[i]), pages_of(held[i] + take)):
                    table[i][j] = free
                    free += 1
                held[i] += take
    return order, torch.tensor(table, dtype=torch.int32, device=DEV), free


def frequencies(case):
    """(radians a position of each pair, factor on cos and sin) of a rotary embedding, stretched eightfold from 4096 positions."""
    rot, base, kind, factor, ctx = case["rot"], case["base"], case["scaling"], 8.0, 4096.0
    f = [base ** (-2.0 * i / rot) for i in range(rot // 2)]
    if kind == "linear":  # positions closer together
        return [x / factor for x in f], 1.0
    if kind == "bands":  # slow pairs stretched, fast ones left, those between blended by their wavelength
        out = []
        for x in f:
            turns = ctx * x / (2 * math.pi)
            w = min(1.0, max(0.0, (turns - 1.0) / (4.0 - 1.0)))
            out.append(w * x + (1 - w) * x / factor)
        return out, 1.0
    if kind == "yarn":  # the same by the pair's number, and sharper scores
        def pair(turns):
            return rot * math.log(ctx / (turns * 2 * math.pi)) / (2 * math.log(base))
        lo, hi = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        hi = hi + 0.001 if hi == lo else hi
        out = []
        for i, x in enumerate(f):
            w = min(1.0, max(0.0, (i - lo) / (hi - lo)))
            out.append(x / factor * w + x * (1 - w))
        return out, 0.1 * math.log(factor) + 1.0
    return f, 1.0


def prepare(case, seed):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed)
    new, past = lengths(case)
    op, n = case["op"], case["n"]
    s = {"case": case, "op": op, "new": new}
    if own:
        from distcomp_b200 import draft, kv4
        s["draft"] = draft
    if op == "verify":
        return prepare_verify(s, case, gen, new)
    hd, kv = case["hd"], case["kv"]
    s["seq"], s["n_new"] = np.arange(n, dtype=np.int32), np.array(new, dtype=np.int32)
    if op == "keep":
        layers, kept = case["layers"], paths(case)
        held = [a + b for a, b in zip(new, past)]
        order, table, used = interleaved(past, PAGE * 3)
        total, width = used + sum(pages_of(h) - pages_of(p) for h, p in zip(held, past)), max(pages_of(h) for h in held)
        s["data"] = torch.randint(-1 << 31, 1 << 31, (layers, total, page_bytes(case) // 4), generator=gen, device=DEV, dtype=torch.int64).to(torch.int32)
        s["past"], s["kept"] = np.array(past, dtype=np.int32), kept
        if own:
            s["pool"] = kv4.KvPool(layers, kv, hd, total, n, width, data=s["data"])
            for i, take in order:
                s["pool"].extend([i], [take])
            return s
        s["table"] = torch.full((n, width), -1, dtype=torch.int32, device=DEV)
        s["table"][:, :table.shape[1]] = table
        s["len"] = torch.tensor(past, dtype=torch.int32, device=DEV)
        s["from"] = torch.tensor([(i, past[i] + j, past[i] + t) for i in range(n) for t, j in enumerate(kept[i])], device=DEV)
        s["held"], s["goal"] = (torch.tensor(v, device=DEV) for v in (held, [p + len(k) for p, k in zip(past, kept)]))
        s["chunk"] = places(hd)
        return s
    held = [a + b for a, b in zip(new, past)]
    order, s["table"], used = interleaved(held, 512)
    dt = TYPES[case["dtype"]]
    head, t = case["head"], sum(new)
    s["data"] = filled(gen, case, used) if op == "tree" else torch.zeros(1, max(1, used), page_bytes(case), dtype=torch.uint8, device=DEV)
    if own:
        s["pool"] = kv4.KvPool(1, kv, hd, max(1, used), n, s["table"].shape[1], data=s["data"])
        for i, take in order:
            s["pool"].extend([i], [take])
    up = [above(p) for p in (trees(case) if op == "tree" or case["tree"] else [range(-1, v - 1) for v in new])]
    depth = torch.tensor([d for u in up for d in u[1]], dtype=torch.int32, device=DEV)
    seq = torch.repeat_interleave(torch.arange(n, device=DEV), torch.tensor(new, device=DEV))
    s["len"], s["past"], s["seq_of"] = torch.tensor(held, device=DEV), torch.tensor(past, device=DEV), seq
    # q, k and v of a row lie side by side, as a fused projection leaves them
    qkv = torch.empty(t, (head + 2 * kv) * hd, dtype=dt, device=DEV)
    qkv[:, :head * hd] = torch.randn(t, head * hd, generator=gen, device=DEV).mul_(1.5)
    s["q"] = qkv[:, :head * hd].unflatten(1, (head, hd))
    s["out"] = torch.empty(t, head, hd, dtype=dt, device=DEV)
    if op == "tree":
        mask = [m - (1 << 64) if m >> 63 else m for u in up for m in u[0]]
        s["mask"] = torch.tensor(mask, dtype=torch.int64, device=DEV)
        s["row_at"] = torch.tensor([j for v in new for j in range(v)], device=DEV)
        return s
    qkv[:, head * hd:(head + kv) * hd] = rows_of(gen, t, case).flatten(1)
    qkv[:, (head + kv) * hd:] = rows_of(gen, t, case, 0.5).flatten(1)
    s["k"] = qkv[:, head * hd:(head + kv) * hd].unflatten(1, (kv, hd))
    s["v"] = qkv[:, (head + kv) * hd:].unflatten(1, (kv, hd))
    s["k_out"], s["v_out"] = (torch.empty(t, kv, hd, dtype=dt, device=DEV) for _ in range(2))
    freq, factor = frequencies(case)
    s["depth"] = depth if case["tree"] else None
    if own:
        s["rope"] = draft.Rope(hd, rot=case["rot"], interleaved=case["inter"], freq=freq, factor=factor)
        return s
    place = s["past"][seq] + torch.tensor([j for v in new for j in range(v)], device=DEV)
    s["row_page"], s["row_at"] = s["table"][seq, place // PAGE].long(), place % PAGE
    s["pos"] = s["past"][seq] + depth
    s["freq"], s["factor"], s["chunk"] = torch.tensor(freq, dtype=torch.float64, device=DEV), factor, places(hd)
    return s


def prepare_verify(s, case, gen, new):
    n, vocab, dt, rows = case["n"], case["vocab"], TYPES[case["dtype"]], sum(new)
    parents = [list(range(-1, v - 1)) for v in new] if case["chain"] else trees(case)
    flat = torch.tensor([p for t in parents for p in t], dtype=torch.int32, device=DEV)
    first = np.cumsum([0] + new)
    logits = torch.randn(rows, vocab, generator=gen, device=DEV).mul_(3.0)
    # a drafter that sees about what the target does
    about = (logits + torch.randn(rows, vocab, generator=gen, device=DEV)).softmax(-1)
    s["logits"] = logits.to(dt)
    up = torch.tensor([first[i] + max(p, 0) for i, t in enumerate(parents) for p in t], device=DEV)
    # a row's children are drawn from its distribution; of a deterministic drafter they are its likeliest tokens in order
    if case["dense"]:
        s["q"] = about
        tok = torch.multinomial(about[up], 1, generator=gen)[:, 0]
    else:
        s["q"] = None
        top = about.topk(min(32, vocab), dim=-1).indices
        nth, seen = [], {}
        for i, t in enumerate(parents):
            for p in t:
                seen[i, p] = seen.get((i, p), -1) + 1
                nth.append(seen[i, p])
        tok = top[up, torch.tensor(nth, device=DEV)]
    s["tokens"], s["parents"] = tok.to(torch.int32), flat
    s["n_row"] = np.array(new, dtype=np.int32)
    s["u"], s["u_next"] = torch.rand(rows, generator=gen, device=DEV), torch.rand(n, generator=gen, device=DEV)
    s["temp"] = torch.zeros(n, device=DEV) if case["greedy"] else torch.rand(n, generator=gen, device=DEV).mul_(0.5).add_(0.6)
    s["kept"] = torch.empty(rows, dtype=torch.int32, device=DEV)
    s["n_kept"], s["next"] = (torch.empty(n, dtype=torch.int32, device=DEV) for _ in range(2))
    if not own:
        s["first"], s["count"] = torch.tensor(first[:-1], device=DEV), torch.tensor(new, device=DEV)
    return s


# ------------------------------------------------------------- plain forms --

def turned(s, x):
    """Rows [rows, heads, hd] turned by their positions, in 64 bits."""
    case, rot = s["case"], s["case"]["rot"]
    angle = s["pos"].double()[:, None] * s["freq"]
    c, d = (f(angle)[:, None] * s["factor"] for f in (torch.cos, torch.sin))
    x = x.double()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if case["inter"] else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * c - b * d, b * c + a * d
    y = torch.stack((a, b), -1).flatten(-2) if case["inter"] else torch.cat((a, b), -1)
    return torch.cat((y, x[..., rot:]), -1)


def plain_rotate(s):
    case = s["case"]
    hd, kv = case["hd"], case["kv"]
    page, at = s["row_page"], s["row_at"]
    out = []
    data = s["data"][0].view(-1, kv, 72 * hd)
    head = torch.arange(kv, device=DEV)[None, :, None, None]
    scales = data.view(torch.float16)
    where = s["chunk"][at][:, None, :, None] * 16 + torch.arange(16, device=DEV)  # [rows, 1, nb, 16]

    def side(x, codes_at, scales_at, dt):
        q, d = quantise(x)
        data[page[:, None, None, None], head, codes_at + at[:, None, None, None] * (hd // 2) + where] = (q[..., 0::2] | q[..., 1::2] << 4).to(torch.uint8)
        block = scales_at // 2 + at[:, None, None] * (hd // 32) + torch.arange(hd // 32, device=DEV)
        scales[page[:, None, None], head[..., 0], block] = d
        out.append(((q - 8).float() * d.float()[..., None]).flatten(-2).to(dt))

    side(turned(s, s["k"]), 0, 64 * hd, s["k"].dtype)
    side(s["v"], 32 * hd, 68 * hd, s["v"].dtype)
    return {"q": turned(s, s["q"]).to(s["q"].dtype), "k": out[0], "v": out[1], "cache": s["data"].view(torch.int32)}


def plain_rows(data, hd, kv, side):
    """fp32 rows [pages, 64, kv, hd] of pages [pages, bytes]."""
    d = data.view(-1, kv, 72 * hd)
    c = d[:, :, side * 32 * hd:(side + 1) * 32 * hd].reshape(-1, kv, PAGE, hd // 32, 16)
    c = c.gather(3, places(hd)[None, None, :, :, None].expand_as(c))
    v = torch.stack((c & 15, c >> 4), -1).flatten(-2).float() - 8
    sc = d[:, :, (64 + 4 * side) * hd:(68 + 4 * side) * hd].contiguous().view(torch.float16).view(-1, kv, PAGE, hd // 32, 1)
    return (v * sc.float()).flatten(-2).transpose(1, 2)


def plain_tree(s):
    case = s["case"]
    hd, kv, n, head = case["hd"], case["kv"], case["n"], case["head"]
    rep, most = head // kv, max(1, max(s["new"]))
    page = s["table"].clamp(min=0).long().flatten()
    at = torch.arange(s["table"].shape[1] * PAGE, device=DEV)
    k, v = (plain_rows(s["data"][0][page], hd, kv, side).reshape(n, -1, kv, hd).permute(0, 2, 3, 1) for side in (0, 1))
    q = torch.zeros(n, most, kv, rep, hd, device=DEV)
    q[s["seq_of"], s["row_at"]] = s["q"].float().unflatten(1, (kv, rep))
    q = q.permute(0, 2, 1, 3, 4).reshape(n, kv, most * rep, hd)
    # which keys a row sees: the cached ones, and the drafted ones of its mask
    mask = torch.zeros(n, most, dtype=torch.int64, device=DEV)
    mask[s["seq_of"], s["row_at"]] = s["mask"]
    new = (at[None] - s["past"][:, None])[:, None]
    live = (new < 0) | ((mask[:, :, None] >> new.clamp(0, 63)) & 1).bool() & (new < 64)
    live = (live & (at[None, None] < s["len"][:, None, None]))[:, None, :, None].expand(n, 1, most, rep, at.numel()).flatten(2, 3)
    sc = (q @ k).mul_(hd ** -0.5).masked_fill_(~live, -math.inf)
    p = sc.sub_(sc.amax(-1, keepdim=True).clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (p @ v.masked_fill(at >= s["len"][:, None, None, None], 0).transpose(-1, -2)) / total
    o = o.view(n, kv, most, rep, hd).transpose(1, 2).flatten(2, 3)
    return {"out": o[s["seq_of"], s["row_at"]].to(s["q"].dtype)}


def plain_verify(s):
    case, n, vocab = s["case"], s["case"]["n"], s["case"]["vocab"]
    first, count, tokens, parents = s["first"], s["count"], s["tokens"].long(), s["parents"].long()
    me = torch.arange(n, device=DEV)
    cur, kept = torch.zeros(n, dtype=torch.int64, device=DEV), torch.full_like(s["parents"], -1)
    kept[first], held = 0, torch.ones(n, dtype=torch.int64, device=DEV)

    def target(row):
        x = s["logits"][row].double()
        if case["greedy"]:  # all weight on the first of the largest
            return torch.zeros_like(x).scatter_(1, (x == x.amax(-1, keepdim=True)).int().argmax(-1, keepdim=True), 1.0)
        x = x / s["temp"].double()[:, None]
        e = (x - x.amax(-1, keepdim=True)).exp()
        return e / e.sum(-1, keepdim=True)

    f = target(first)
    for j in range(1, max(s["new"])):
        row = (first + j).clamp(max=tokens.numel() - 1)
        child = (j < count) & (parents[row] == cur)
        tok = tokens[row]
        total = f.sum(-1)
        q = s["q"][first + cur].double() if s["q"] is not None else None
        weight = q[me, tok] if q is not None else torch.ones(n, dtype=torch.float64, device=DEV)
        take = child & (s["u"][row].double() * weight * total < f[me, tok])
        rest = (f / total[:, None] - q).clamp(min=0) if q is not None else f.scatter(1, tok[:, None], 0.0)
        cur = torch.where(take, j, cur)
        f = torch.where(take[:, None], target(first + cur), torch.where((child & ~take)[:, None], rest, f))
        kept[(first + held)[take]] = j
        held = held + take
    sums = f.cumsum(-1)
    nxt = torch.searchsorted(sums, (s["u_next"].double() * sums[:, -1])[:, None], right=True)[:, 0]
    last = vocab - 1 - (f > 0).flip(-1).int().argmax(-1)
    return {"kept": kept, "n_kept": held.int(), "next": torch.minimum(nxt, last).int()}


def plain_keep(s):
    case, table, data = s["case"], s["table"], s["data"]
    n, hd, kv, nb = case["n"], case["hd"], case["kv"], case["hd"] // 32
    col = torch.arange(table.shape[1], device=DEV)[None]
    now = (s["len"].long() + PAGE - 1) // PAGE
    # back to where the step began, and grown by its drafts: the lowest free pages in the sequences' order
    begin = (torch.tensor(s["past"], device=DEV).long() + PAGE - 1) // PAGE
    table.masked_fill_((col >= begin[:, None]) & (col < now[:, None]), -1)
    free = torch.ones(data.shape[1], dtype=torch.bool, device=DEV)
    free[table[table >= 0].long()] = False
    want = (col >= begin[:, None]) & (col < ((s["held"] + PAGE - 1) // PAGE)[:, None])
    table[want] = free.nonzero()[:int(want.sum()), 0].int()
    # the kept rows, all read before any is written
    seq, src, dst = s["from"].unbind(1)
    raw = data.view(torch.uint8).view(data.shape[0], data.shape[1], kv, 72 * hd)
    codes = raw[..., :64 * hd].unflatten(-1, (2, PAGE, nb, 16))
    scales = raw[..., 64 * hd:].unflatten(-1, (2, PAGE, 2 * nb))
    lay = torch.arange(data.shape[0], device=DEV)[:, None, None]
    page, at = table[seq, src // PAGE].long()[None, :, None], (src % PAGE)[None, :, None]
    c = codes[lay, page, :, :, at, s["chunk"][src % PAGE][None]]
    d = scales[lay[..., 0], page[..., 0], :, :, at[..., 0]]
    page, at = table[seq, dst // PAGE].long()[None, :, None], (dst % PAGE)[None, :, None]
    codes[lay, page, :, :, at, s["chunk"][dst % PAGE][None]] = c
    scales[lay[..., 0], page[..., 0], :, :, at[..., 0]] = d
    table.masked_fill_(col >= ((s["goal"] + PAGE - 1) // PAGE)[:, None], -1)
    s["len"].copy_(s["goal"])
    return {"table": table, "len": s["len"], "data": data}


def run(s):
    if own:
        pool = s.get("pool")
        if s["op"] == "rotate":
            pool.append_rope(0, s["rope"], s["q"], s["k"], s["v"], s["seq"], s["n_new"], depth=s["depth"], q_out=s["out"], k_out=s["k_out"], v_out=s["v_out"])
            return {"q": s["out"], "k": s["k_out"], "v": s["v_out"], "cache": s["data"].view(torch.int32)}
        if s["op"] == "tree":
            return {"out": pool.attend_tree(0, s["q"], s["seq"], s["n_new"], s["mask"], out=s["out"])}
        if s["op"] == "verify":
            s["draft"].verify(s["logits"], s["tokens"], s["parents"], s["n_row"], s["u"], s["u_next"], temperature=s["temp"], draft=s["q"], kept=s["kept"],
                              n_kept=s["n_kept"], next=s["next"])
            return {"kept": s["kept"], "n_kept": s["n_kept"], "next": s["next"]}
        pool.truncate(s["seq"], s["past"])
        pool.extend(s["seq"], s["n_new"])
        pool.keep(s["seq"], s["n_new"], s["kept"])
        return {"table": pool.table, "len": pool.lengths, "data": s["data"]}
    return {"rotate": plain_rotate, "tree": plain_tree, "verify": plain_verify, "keep": plain_keep}[s["op"]](s)


# ------------------------------------------------------------------- exact --

def exact(case, seed):
    if case["op"] in ("verify", "keep"):  # whole numbers only
        return None
    s = prepare(case, seed)
    new, past = lengths(case)
    hd, kv, rep = case["hd"], case["kv"], case["head"] // case["kv"]
    if case["op"] == "rotate":
        freq, factor = frequencies(case)
        parents = trees(case) if case["tree"] else None
        pos = np.concatenate([p + (np.array(above(parents[i])[1]) if parents else np.arange(m)) for i, (m, p) in enumerate(zip(new, past))])
        angle = np.fmod(pos.astype(np.longdouble)[:, None] * np.array(freq, dtype=np.longdouble), 2 * np.longdouble("3.14159265358979323846264338327950288"))
        turn = np.exp(1j * angle.astype(np.float64))[:, None] * factor
        rot = case["rot"]
        first = np.arange(0, rot, 2) if case["inter"] else np.arange(rot // 2)
        second = first + (1 if case["inter"] else rot // 2)

        def turn_rows(x):
            x = x.double().cpu().numpy()
            z = (x[..., first] + 1j * x[..., second]) * turn
            x[..., first], x[..., second] = z.real, z.imag
            return x

        def stored(x):
            x = x.reshape(-1, 32)
            m = x[np.arange(len(x)), np.argmax(np.abs(x), axis=1)]
            d = np.clip(m / -8.0, -65504, 65504).astype(np.float16).astype(np.float64)[:, None]
            code = np.clip(np.floor(np.divide(x, d, out=np.zeros_like(x), where=d != 0) + 8.5), 0, 15)
            return ((code - 8) * d).reshape(-1, kv, hd)
        return {"q": turn_rows(s["q"]), "k": stored(turn_rows(s["k"])), "v": stored(s["v"].double().cpu().numpy()), "cache": None}
    out = torch.zeros(sum(new), case["head"], hd, dtype=torch.float64, device=DEV)
    nb, r0 = hd // 32, 0
    dim = torch.arange(hd, device=DEV)
    pages, grown = s["data"][0].view(-1, kv, 72 * hd), trees(case)
    for i, (m, base) in enumerate(zip(new, past)):
        if not m:
            continue
        t = torch.arange(m + base, device=DEV)
        page, at = s["table"][i].long()[t // PAGE], t % PAGE
        turn = {4: (at // 2) % 4, 2: (at // 4) % 2}[nb]
        byte = at[:, None] * (hd // 2) + ((dim // 32)[None] ^ turn[:, None]) * 16 + (dim % 32 // 2)[None]
        seen = torch.ones(m, m + base, dtype=torch.bool, device=DEV)
        for j, p in enumerate(grown[i]):
            seen[j, base:] = seen[p, base:] if p >= 0 else False
            seen[j, base + j] = True
        for h in range(kv):
            side = []
            for j in (0, 1):
                raw = pages[page[:, None], h, byte + j * 32 * hd].long()
                code = torch.where(dim % 2 == 1, raw // 16, raw % 16).double() - 8
                scale = pages[:, h].view(torch.float16)[page[:, None], (32 + 2 * j) * hd + at[:, None] * nb + dim[None] // 32].double()
                side.append(code * scale)
            for g in range(h * rep, (h + 1) * rep):
                w = s["q"][r0:r0 + m, g].double() @ side[0].T / math.sqrt(hd)
                out[r0:r0 + m, g] = torch.softmax(w.masked_fill_(~seen, -math.inf), -1) @ side[1]
        r0 += m
    return {"out": out}
