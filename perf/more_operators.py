"""Cases of the operators on a paged K/V cache held in 8 bits (int8 codes, a scale for each block of
positions and kv head), for measuring them: the append that quantises (`append`), reading rows back
(`read`) and attention over the cache, with or without a prefix that the batch shares (`attention`).
Each case runs either as a plain form in elementary torch operations (32 bits, rounded once at the
end) or, where `own` is true, through this package's entry points.

Lengths of a case follow from its numbers alone (`_lengths`), values and page orders from the
seed. Rows are tokens; a sequence of the batch brings q >= 0 new rows, which are the last of its kv
own positions."""
import math
import os
import sys

import numpy as np
import torch

own = False

_context = None


def _binding():
    """The package's binding and one context for the process, as a user's program holds it."""
    global _context
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-omni-inference-rs_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import lq8
    if _context is None:
        _context = lq8.Context(0)
    return lq8, _context


# ---------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------

def listed():
    return [
        # one decode step of 8 sequences from f32 projection rows, q/k norm weights; the blocks that
        # the step touched are read back, as a check of what the cache holds does
        dict(name="append decode 8 rows", op="append", src="f32", seqs=8, heads=64, kv_heads=8, head_dim=128, page=16,
             block=16, own=1500, chunk=1, axes=0, norm=True),
        # prompt chunks of 12 sequences, multi-axis positions, bf16 rows; read back for the chunks' own attention
        dict(name="append chunks 12 seqs", op="append", src="bf16", seqs=12, heads=32, kv_heads=8, head_dim=128, page=64,
             block=64, own=700, chunk=511, axes=3, norm=True),
        # a large prefill from f32 rows, no norm weights, blocks of 128
        dict(name="append prefill 16 seqs", op="append", src="f32", seqs=16, heads=32, kv_heads=8, head_dim=128,
             page=128, block=128, own=100, chunk=2000, axes=3, norm=False),
        # the last rows of two sequences
        dict(name="read 2 seqs", op="read", out="bf16", seqs=2, kv_heads=8, head_dim=128, page=16, block=16, own=60,
             chunk=40),
        # ragged ends of 40 sequences, f32, head dimension 64
        dict(name="read 40 seqs f32 d64", op="read", out="f32", seqs=40, kv_heads=4, head_dim=64, page=32, block=32,
             own=500, chunk=901),
        # whole long sequences into another cache's type
        dict(name="read 24 seqs", op="read", out="bf16", seqs=24, kv_heads=8, head_dim=128, page=64, block=16, own=1,
             chunk=9000),
        # the smallest attention call: two sequences, a short prefix that ends inside a page
        dict(name="attn decode 2 seqs", op="attention", seqs=2, heads=16, kv_heads=8, head_dim=128, page=16, block=16,
             prefix=100, own=40, chunk=1),
        # one decode step of 64 sequences with long contexts of their own
        dict(name="attn decode 64 seqs long", op="attention", seqs=64, heads=64, kv_heads=8, head_dim=128, page=64,
             block=16, prefix=0, own=8000, chunk=1),
        # plain paged decode, head dimension 64, pages of 128 with a scale each
        dict(name="attn decode 48 seqs d64", op="attention", seqs=48, heads=32, kv_heads=4, head_dim=64, page=128,
             block=128, prefix=0, own=4000, chunk=1),
        # one decode step of 64 sequences behind an 8191-token system prompt
        dict(name="attn decode 64 seqs prefix", op="attention", seqs=64, heads=32, kv_heads=8, head_dim=128, page=16,
             block=16, prefix=8191, own=1000, chunk=1),
        # the largest: 128 sequences that share a 32768-token document
        dict(name="attn decode 128 seqs 32k", op="attention", seqs=128, heads=64, kv_heads=8, head_dim=128, page=64,
             block=64, prefix=32768, own=1000, chunk=1),
        # chunks of new tokens (prompt continuations next to decode rows), ragged, prefix 2049
        dict(name="attn chunks 10 seqs", op="attention", seqs=10, heads=32, kv_heads=8, head_dim=128, page=32, block=32,
             prefix=2049, own=1500, chunk=500),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(16, 8), (32, 8), (64, 8), (32, 4), (12, 4), (5, 1), (28, 4), (8, 8), (14, 2), (16, 1)]


def draw(rng):
    op = rng.choice(["append", "read", "attention", "attention"])
    heads, kv_heads = rng.choice(_HEADS)
    head_dim, page = rng.choice([64, 128, 128]), rng.choice([16, 32, 64, 128, 256])
    block = rng.choice([b for b in (16, 32, 64, 128) if b <= page])
    c = dict(op=op, kv_heads=kv_heads, head_dim=head_dim, page=page, block=block)
    if op == "append":
        chunk = rng.choice([1, 1, _log(rng, 2, 2000)])
        seqs = _log(rng, 1, 256 if chunk == 1 else max(1, min(32, 24000 // chunk)))
        return dict(c, src=rng.choice(["f32", "bf16"]), seqs=seqs, heads=heads, own=_log(rng, 1, 2000), chunk=chunk,
                    axes=rng.choice([0, 1, 3]), norm=rng.random() < 0.7)
    if op == "read":
        chunk = _log(rng, 2, 9000)
        return dict(c, out=rng.choice(["bf16", "f32"]), seqs=_log(rng, 1, max(1, min(64, 100000 // chunk))),
                    own=_log(rng, 1, 2000), chunk=chunk)
    chunk = rng.choice([1, 1, 1, rng.randint(2, 4), _log(rng, 5, 500)])
    c.update(seqs=_log(rng, 1, 128 if chunk == 1 else 16), heads=heads, chunk=chunk,
             prefix=rng.choice([0, 0, _log(rng, 1, 32768), _log(rng, 1, 32768)]), own=_log(rng, 1, 8000))
    most = work(listed()[10])["flops"]
    while (work(c)["flops"] > most or c["seqs"] * c["chunk"] * heads * (c["prefix"] + c["own"] + c["chunk"]) > 4e8 or
           c["seqs"] * c["own"] * kv_heads * head_dim > 64 * 8000 * 1024):
        if c["prefix"] >= c["own"]:
            c["prefix"] = c["prefix"] * 2 // 3
        else:
            c["own"] = c["own"] * 2 // 3
    return c


def _lengths(case):
    """(q, past) of each sequence: new rows and positions before them, from the case alone.
    Decode steps bring one row a sequence; chunked ones 0 to `chunk` rows, a fifth of them none."""
    b = np.arange(case["seqs"], dtype=np.int64)
    past = (b * 7919 + 37) % 101 * case["own"] // 100
    if case["chunk"] == 1:
        return np.ones_like(b), past
    q = 1 + (b * 4099 + 96) % 97 * (case["chunk"] - 1) // 96
    return np.where(b % 5 == 3, 0, q), past


_TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
_SIZE = {"bf16": 2, "f32": 4}
_POSITIONS = 40960  # rows of the cos/sin tables


def _touched(case):
    """Rows that an append's read-back covers: from the beginning of the first block that each
    sequence's new rows touch."""
    q, past = _lengths(case)
    return np.where(q > 0, q + past % case["block"], 0)


def work(case):
    q, past = _lengths(case)
    rows, D, Hkv = int(q.sum()), case["head_dim"], case["kv_heads"]
    if case["op"] == "read":
        n = 2 * rows * Hkv * D
        return {"bytes": n + n * _SIZE[case["out"]] + 4 * n // (D * case["block"]), "flops": n}
    Hq = case["heads"]
    if case["op"] == "append":
        read = int(_touched(case).sum())  # rows of the touched blocks: new ones, and older ones that may be rounded again
        kv = 2 * Hkv * D
        return {"bytes": rows * (Hq + 2 * Hkv) * D * _SIZE[case["src"]] + 2 * rows * Hq * D + rows * kv + (read - rows) * kv +
                         2 * read * kv + min(_POSITIONS, rows) * D * 4 + 4 * case["axes"] * rows,
                "flops": (7 if case["norm"] else 3) * rows * (Hq + Hkv) * D + 4 * rows * Hkv * D}
    kv = case["prefix"] + int(np.where(q > 0, past + q, 0).sum())
    seen = int((q * (case["prefix"] + past) + q * (q + 1) // 2).sum())
    return {"bytes": 2 * kv * Hkv * D + 8 * kv * Hkv // case["block"] + 4 * rows * Hq * D, "flops": 4 * seen * Hq * D}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _axis_of_pair(pairs, axes):
    """The axis whose position turns each rotary pair: a quarter of the pairs, three eighths, three eighths."""
    i = np.arange(pairs)
    if axes == 3:
        return np.where(i < pairs // 4, 0, np.where(i < pairs // 4 + (pairs - pairs // 4) // 2, 1, 2)).astype(np.uint8)
    return np.zeros(pairs, np.uint8)


def _tables(pairs, dev):
    inv = torch.from_numpy(1e6 ** (-np.arange(pairs) / pairs)).to(dev)
    ang = torch.arange(_POSITIONS, device=dev, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _grid_positions(rows, axes, gen, dev):
    """Positions of `axes` axes: runs of text (all axes equal) and of a 24 x 32 grid (its own
    height and width behind a common start)."""
    r = torch.arange(rows, device=dev)
    start = torch.randint(0, 64, (1,), generator=gen, device=dev)
    grid = torch.stack([r // 768, r // 32 % 24, r % 32])[:axes] if axes > 1 else r[None] % (_POSITIONS - 64)
    return (grid + start).to(torch.int32).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed) * 1000003 + 17)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dtype)

    s = {"case": dict(case)}
    q, past = _lengths(case)
    kv = past + q
    B, D, Hkv, page, block = case["seqs"], case["head_dim"], case["kv_heads"], case["page"], case["block"]
    prefix = case.get("prefix", 0)
    prefix_pages, own_pages = -(-prefix // page), -(-kv // page)
    n_pages = int(prefix_pages + own_pages.sum()) + 3
    ids = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32).cpu().numpy()
    table = np.zeros((B, max(1, int(own_pages.max()))), np.int32)
    at = np.concatenate([[0], np.cumsum(own_pages)]) + prefix_pages
    for b in range(B):
        table[b, :own_pages[b]] = ids[at[b]:at[b + 1]]
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)  # noqa: E731
    start = lambda a: put(np.concatenate([[0], np.cumsum(a)]))  # noqa: E731
    s["table"], s["kv_len"] = put(table), put(kv)
    s["prefix_table"] = put(ids[:prefix_pages]) if prefix else None
    s["q_start"] = start(q)
    s["max_q"], s["max_kv"] = max(1, int(q.max())), max(1, int(kv.max()))
    rows = s["rows"] = int(q.sum())
    # what the pages hold: values whose size differs from head to head and from dim to dim
    for name in ("k", "v"):
        gain = torch.exp(0.4 * normal(Hkv, 1, D, dtype=torch.float32))
        x = torch.randn(n_pages, Hkv, page, D, generator=gen, device=dev, dtype=torch.float32)
        x *= gain
        x = x.view(n_pages, Hkv, page // block, block * D)
        scale = x.abs().amax(-1) / 127
        x /= scale[..., None]
        s[name] = x.round_().clamp_(-127, 127).to(torch.int8).view(n_pages, Hkv, page, D)
        s[name + "_scale"] = scale.contiguous()
        del x
    if case["op"] == "append":
        Hq = case["heads"]
        read = _touched(case)
        s["read_rows"], s["read_start"], s["max_read"] = int(read.sum()), start(read), max(1, int(read.max()))
        s["qkv"] = normal(rows, (Hq + 2 * Hkv) * D, scale=1.1, dtype=_TYPE[case["src"]])
        s["axis"] = _axis_of_pair(D // 2, case["axes"])
        s["cos"], s["sin"] = _tables(D // 2, dev)
        s["pos"] = _grid_positions(rows, case["axes"], gen, dev) if case["axes"] else None
        for name in ("q_norm", "k_norm"):
            s[name] = (1 + 0.1 * normal(D, dtype=torch.float32)).to(torch.bfloat16) if case["norm"] else None
        s["q_out"] = torch.empty(rows, Hq, D, dtype=torch.bfloat16, device=dev)
        s["k_out"], s["v_out"] = (torch.empty(s["read_rows"], Hkv, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    elif case["op"] == "read":
        s["k_out"], s["v_out"] = (torch.empty(rows, Hkv, D, dtype=_TYPE[case["out"]], device=dev) for _ in range(2))
    else:
        s["q"] = normal(rows, case["heads"], D, scale=1.5)
        s["out"] = torch.empty_like(s["q"])
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if not own:
        return {"append": _plain_append, "read": _plain_read, "attention": _plain_attention}[op](s)
    h = s.get("handles")
    if h is None:  # the views of its own buffers that a program keeps: pointers, sizes, strides
        h = s["handles"] = _handles(s)
    if op == "append":
        q = h["cache"].append(s["qkv"], s["case"]["heads"], h["batch"], h["rotary"], pos=s["pos"], q_norm=s["q_norm"],
                              k_norm=s["k_norm"], eps=1e-6, q_out=s["q_out"])
        return (q, *h["cache"].read(h["touched"], s["k_out"], s["v_out"]))
    if op == "read":
        return h["cache"].read(h["batch"], s["k_out"], s["v_out"])
    return h["cache"].attend(s["q"], h["batch"], out=s["out"])


def _handles(s):
    lq8, ctx = _binding()
    c = s["case"]
    h = {"cache": lq8.PagedKvCacheQ8(ctx, s["k"], s["v"], s["k_scale"], s["v_scale"])}
    h["batch"] = lq8.PagedBatch(s["table"], s["kv_len"], q_start=s["q_start"] if c["chunk"] > 1 else None, max_q=s["max_q"],
                                max_kv=s["max_kv"], prefix_table=s["prefix_table"], prefix_len=c.get("prefix", 0))
    if c["op"] == "append":
        h["rotary"] = lq8.Rotary(s["cos"], s["sin"], s["axis"])
        h["touched"] = lq8.PagedBatch(s["table"], s["kv_len"], q_start=s["read_start"], max_q=s["max_read"], max_kv=s["max_kv"])
    return h


def _rows_of(s, q_start, rows):
    """Sequence and own position of every row of a batch whose rows begin at q_start."""
    r = torch.arange(rows, device=q_start.device)
    b = torch.searchsorted(q_start[1:].contiguous(), r.to(torch.int32), right=True)
    return b, (s["kv_len"][b] - q_start[b + 1]).long() + r


def _turn(x, cos, sin):
    """Rotates pairs (i, i + n) of x [rows, heads, D] by rows' angles [rows, n]."""
    n = cos.shape[1]
    a, b = x[..., :n], x[..., n:]
    c, d = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * d, b * c + a * d], dim=-1)


def _plain_append(s):
    c = s["case"]
    D, Hq, Hkv, block = c["head_dim"], c["heads"], c["kv_heads"], c["block"]
    b, at = _rows_of(s, s["q_start"], s["rows"])
    x = s["qkv"].float().view(s["rows"], Hq + 2 * Hkv, D)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_norm"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["k_norm"].float()
    pairs = torch.arange(D // 2, device=b.device)
    pos = (s["pos"] if s["pos"] is not None else at[None]).long()
    pos = pos[torch.from_numpy(s["axis"]).to(b.device).long()].T
    cos, sin = s["cos"][pos, pairs], s["sin"][pos, pairs]
    page, off = s["table"][b, at // c["page"]].long(), at % c["page"]
    slot = off // block
    n_rows = (s["q_start"][1:] - s["q_start"][:-1]).long()
    first = s["kv_len"].long() - n_rows  # a sequence's first new position
    for name, new in (("k", _turn(k, cos, sin)), ("v", v)):
        codes, scale = s[name], s[name + "_scale"]
        flat = ((page * Hkv)[:, None] + torch.arange(Hkv, device=b.device)) * scale.shape[2] + slot[:, None]
        most = torch.zeros_like(scale).view(-1).scatter_reduce(0, flat.view(-1), new.abs().amax(-1).view(-1) / 127, "amax")
        # a block that older positions begin keeps its scale where that is larger, and they are rounded again
        older = (first % block != 0) & (n_rows > 0)
        live = torch.nonzero(older)[:, 0]
        p0 = s["table"][live, first[live] // c["page"]].long()
        o0 = first[live] % c["page"] // block
        heads = torch.arange(Hkv, device=b.device)
        at0 = ((p0 * Hkv)[:, None] + heads) * scale.shape[2] + o0[:, None]
        was = scale.view(-1)[at0]
        now = torch.maximum(was, most[at0])
        most[at0] = now
        old = codes.view(codes.shape[0], Hkv, -1, block, D)[p0[:, None], heads[None], o0[:, None]].float()
        again = torch.round(old * torch.where(now > 0, was / now, torch.zeros_like(now))[..., None, None])
        before = torch.arange(block, device=b.device)[None] < (first[live] % block)[:, None]
        again = torch.where(before[:, None, :, None], again, old).to(torch.int8)
        codes.view(codes.shape[0], Hkv, -1, block, D)[p0[:, None], heads[None], o0[:, None]] = again
        scale.view(-1)[flat.view(-1)] = most[flat.view(-1)]
        size = most[flat][..., None]
        new = torch.round(new / torch.where(size > 0, size, torch.ones_like(size)))
        codes[page, :, off] = new.clamp(-127, 127).to(torch.int8)
    return (_turn(q, cos, sin).to(torch.bfloat16), *_read_rows(s, s["read_start"], s["read_rows"], torch.bfloat16))


def _read_rows(s, q_start, rows, dtype):
    c = s["case"]
    b, at = _rows_of(s, q_start, rows)
    page, off = s["table"][b, at // c["page"]].long(), at % c["page"]
    return [(s[n][page, :, off].float() * s[n + "_scale"][page, :, off // c["block"]][..., None]).to(dtype) for n in ("k", "v")]


def _plain_read(s):
    return tuple(_read_rows(s, s["q_start"], s["rows"], _TYPE[s["case"]["out"]]))


def _pages(s, name, ids):
    """Pages `ids` [..., n] as values [..., n, Hkv, page, D]."""
    c = s["case"]
    codes = s[name][ids].float()
    codes = codes.view(*codes.shape[:-2], c["page"] // c["block"], c["block"], c["head_dim"])
    return (codes * s[name + "_scale"][ids][..., None, None]).flatten(-3, -2)


def _plain_attention(s):
    c = s["case"]
    D, Hq, Hkv, prefix = c["head_dim"], c["heads"], c["kv_heads"], c["prefix"]
    B, G, Q, T = c["seqs"], Hq // Hkv, s["max_q"], s["max_kv"]
    dev = s["q"].device
    b, at = _rows_of(s, s["q_start"], s["rows"])
    j = torch.arange(s["rows"], device=dev) - s["q_start"][b].long()
    # the rows of each sequence side by side: [B, Hkv, G * Q, D]
    q = torch.zeros(B, Q, Hq, D, device=dev)
    q[b, j] = s["q"].float() / math.sqrt(D)
    q = q.view(B, Q, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Q, D)
    ids = s["table"][:, :-(-T // c["page"])].long()
    own_k, own_v = (_pages(s, n, ids).transpose(1, 2).reshape(B, Hkv, -1, D) for n in ("k", "v"))
    t = torch.arange(own_k.shape[2], device=dev)
    first = s["kv_len"].long() - (s["q_start"][1:] - s["q_start"][:-1]).long()
    sees = t[None, None] <= first[:, None, None] + torch.arange(Q, device=dev)[None, :, None]
    sees = (sees & (t[None] < s["kv_len"][:, None].long())[:, None])[:, None].repeat(1, G, 1, 1).view(B, 1, G * Q, -1)
    scores = torch.matmul(q, own_k.transpose(2, 3)).masked_fill(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if prefix:
        pk, pv = (_pages(s, n, s["prefix_table"].long()).transpose(0, 1).reshape(Hkv, -1, D)[:, :prefix] for n in ("k", "v"))
        flat = q.permute(1, 0, 2, 3).reshape(Hkv, B * G * Q, D)
        shared = torch.matmul(flat, pk.transpose(1, 2))
        top = torch.maximum(top, shared.amax(-1, keepdim=True).view(Hkv, B, G * Q, 1).permute(1, 0, 2, 3))
        shared = torch.exp(shared - top.permute(1, 0, 2, 3).reshape(Hkv, -1, 1))
        shared_sum = shared.sum(-1, keepdim=True).view(Hkv, B, G * Q, 1).permute(1, 0, 2, 3)
        shared = torch.matmul(shared, pv).view(Hkv, B, G * Q, D).permute(1, 0, 2, 3)
    p = torch.exp(scores - top.clamp_min(-3e38))
    o, total = torch.matmul(p, own_v), p.sum(-1, keepdim=True)
    if prefix:
        o, total = o + shared, total + shared_sum
    o = o / torch.where(total > 0, total, torch.ones((), device=dev))
    o = o.view(B, Hkv, G, Q, D).permute(0, 3, 1, 2, 4).reshape(B, Q, Hq, D)
    return o[b, j].to(torch.bfloat16)


# ---------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    q, past = _lengths(case)
    D, Hkv, page, block = case["head_dim"], case["kv_heads"], case["page"], case["block"]
    table = s["table"].cpu().numpy()
    dev = s["k"].device
    index = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int64)).to(dev)  # noqa: E731

    def sequence(name, b, n=None):
        """Positions of a sequence (of the prefix for b None) as values [Hkv, positions, D]."""
        ids = s["prefix_table"].long() if b is None else index(table[b, :-(-int(past[b] + q[b]) // page)])
        codes = s[name].transpose(0, 1)[:, ids].reshape(Hkv, -1, D)
        size = s[name + "_scale"].transpose(0, 1)[:, ids].reshape(Hkv, -1)
        x = codes.to(f).view(Hkv, -1, block, D) * size.to(f)[:, :, None, None]
        return x.view(Hkv, -1, D)[:, :n]

    if case["op"] == "read":
        return tuple(torch.cat([sequence(n, b, int(past[b] + q[b]))[:, past[b]:].transpose(0, 1) for b in range(len(q)) if q[b]])
                     for n in ("k", "v"))
    Hq = case["heads"]
    if case["op"] == "append":
        x = s["qkv"].to(f).reshape(-1, Hq + 2 * Hkv, D)
        if s["pos"] is not None:
            pos = s["pos"]
        else:
            pos = index(np.concatenate([np.arange(past[b], past[b] + q[b]) for b in range(len(q))]))[None]
        w = torch.stack([torch.complex(s["cos"][pos[a].long(), i].to(f), s["sin"][pos[a].long(), i].to(f))
                         for i, a in enumerate(s["axis"].tolist())], dim=1)[:, None]
        parts = {"q": x[:, :Hq], "k": x[:, Hq:Hq + Hkv]}
        for name, y in parts.items():
            if case["norm"]:
                y = y / (y.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * s[name + "_norm"].to(f)
            z = torch.complex(y[..., :D // 2], y[..., D // 2:]) * w
            parts[name] = torch.cat([z.real, z.imag], dim=-1)
        out = [parts["q"]]
        begin = np.concatenate([[0], np.cumsum(q)])
        for name, new in (("k", parts["k"]), ("v", x[:, Hq + Hkv:])):
            got = []
            for b in range(len(q)):
                if not q[b]:
                    continue
                lead, n = int(past[b] % block), int(q[b])  # older positions of the first block
                rows = new[begin[b]:begin[b] + n].transpose(0, 1)
                blocks = torch.zeros(Hkv, -(-(lead + n) // block) * block, D, dtype=f, device=dev)
                blocks[:, lead:lead + n] = rows
                blocks = blocks.view(Hkv, -1, block, D)
                size = blocks.abs().amax((2, 3)) / 127
                if lead:
                    pg, o = int(table[b, past[b] // page]), int(past[b] % page) // block
                    was = s[name + "_scale"][pg, :, o].to(f)
                    size[:, 0] = torch.maximum(size[:, 0], was)
                    codes = s[name][pg, :, o * block:o * block + lead].to(f)
                    blocks[:, 0, :lead] = codes * was[:, None, None]
                size = size[:, :, None, None]
                blocks = (blocks / torch.where(size > 0, size, 1.0)).round() * size
                got.append(blocks.view(Hkv, -1, D)[:, :lead + n].transpose(0, 1))
            out.append(torch.cat(got))
        return tuple(out)
    G, prefix, out, start = Hq // Hkv, case["prefix"], [], 0
    pk, pv = (sequence(n, None, prefix) for n in ("k", "v")) if prefix else (None, None)
    for b in range(len(q)):
        if not q[b]:
            continue
        n, kv = int(q[b]), int(past[b] + q[b])
        rows = s["q"][start:start + n].to(f).view(n, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * n, D)
        start += n
        own_k, own_v = sequence("k", b, kv), sequence("v", b, kv)
        score = rows @ own_k.mT / math.sqrt(D)
        hidden = torch.arange(kv, device=dev)[None] > torch.arange(kv - n, kv, device=dev)[:, None]
        score.view(Hkv, G, n, kv).masked_fill_(hidden, -math.inf)
        if prefix:
            score = torch.cat([rows @ pk.mT / math.sqrt(D), score], dim=-1)
        p = torch.softmax(score, dim=-1)
        o = p[..., prefix:] @ own_v
        if prefix:
            o = o + p[..., :prefix] @ pv
        out.append(o.view(Hkv, G, n, D).permute(2, 0, 1, 3).reshape(n, Hq, D))
    return torch.cat(out)
