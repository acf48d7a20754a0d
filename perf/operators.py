"""Cases of the paged-serving operators, for measuring them: rotary positions with several axes
(`mrope`), the append to a paged K/V cache with the rotation on the way (`append`), and attention
over that cache for a batch that shares a prefix (`attention`). Each case runs either as a plain
form in elementary torch operations (32 bits, rounded once at the end) or, where `own` is true,
through this package's entry points.

Lengths of a case follow from its numbers alone (`_lengths`), values and page orders from the
seed. Rows are tokens; a sequence of the batch brings q >= 0 new rows and owns kv positions of
its own, after the prefix that all share."""
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
        # one decode step's q and k heads of 8 sequences (64 + 8 heads): a few hundred KB, latency
        dict(name="mrope decode 8 rows", op="mrope", dtype="bf16", rows=8, heads=72, extra=8, head_dim=128, rot=128,
             axes=3, layout="cyclic"),
        # patches of an image in an encoder: two axes (height, width), each with its own
        # frequencies, a head dimension that is no power of two, f32 activations
        dict(name="mrope patches 4805 rows", op="mrope", dtype="f32", rows=4805, heads=32, extra=16, head_dim=80,
             rot=80, axes=2, layout="per_axis"),
        # a long prompt with video: q and k heads of 32768 tokens
        dict(name="mrope prompt 32768 rows", op="mrope", dtype="bf16", rows=32768, heads=40, extra=8, head_dim=128,
             rot=128, axes=3, layout="blocks"),
        # one decode step of 8 sequences from f32 projection rows, q/k norm weights
        dict(name="append decode 8 rows", op="append", src="f32", dtype="bf16", seqs=8, heads=64, kv_heads=8,
             head_dim=128, page=16, own=1500, chunk=1, axes=0, norm=True),
        # prompt chunks of 12 sequences, multi-axis positions, bf16 rows
        dict(name="append chunks 12 seqs", op="append", src="bf16", dtype="bf16", seqs=12, heads=32, kv_heads=8,
             head_dim=128, page=64, own=700, chunk=511, axes=3, norm=True),
        # a large prefill into an f32 cache, no norm weights
        dict(name="append prefill f32", op="append", src="f32", dtype="f32", seqs=16, heads=32, kv_heads=8,
             head_dim=128, page=32, own=100, chunk=2000, axes=3, norm=False),
        # the smallest attention call: two sequences, a short prefix that ends inside a page
        dict(name="attn decode 2 seqs", op="attention", dtype="bf16", seqs=2, heads=16, kv_heads=8, head_dim=128,
             page=16, prefix=100, own=40, chunk=1),
        # one decode step of 64 sequences behind an 8191-token system prompt
        dict(name="attn decode 64 seqs", op="attention", dtype="bf16", seqs=64, heads=32, kv_heads=8, head_dim=128,
             page=16, prefix=8191, own=1000, chunk=1),
        # the largest: 128 sequences that share a 32768-token document
        dict(name="attn decode 128 seqs 32k", op="attention", dtype="bf16", seqs=128, heads=64, kv_heads=8,
             head_dim=128, page=64, prefix=32768, own=1000, chunk=1),
        # chunks of new tokens (prompt continuations next to decode rows), ragged, prefix 2049
        dict(name="attn chunks 10 seqs", op="attention", dtype="bf16", seqs=10, heads=32, kv_heads=8, head_dim=128,
             page=32, prefix=2049, own=1500, chunk=500),
        # no prefix: plain paged decode, head dimension 64
        dict(name="attn decode no prefix d64", op="attention", dtype="bf16", seqs=48, heads=32, kv_heads=4, head_dim=64,
             page=128, prefix=0, own=4000, chunk=1),
        # the f32 cache of the framework's own model runner, batch 8
        dict(name="attn decode f32 8 seqs", op="attention", dtype="f32", seqs=8, heads=64, kv_heads=8, head_dim=128,
             page=16, prefix=1024, own=600, chunk=1),
    ]


def _log(rng, lo, hi):
    """A whole number from lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


_HEADS = [(16, 8), (32, 8), (64, 8), (32, 4), (12, 4), (5, 1), (28, 4), (8, 8), (14, 2)]


def draw(rng):
    op = rng.choice(["mrope", "append", "attention", "attention"])
    if op == "mrope":
        head_dim = rng.choice([64, 80, 96, 128, 256])
        layout, axes = rng.choice([("blocks", 3), ("cyclic", 3), ("per_axis", 2), ("blocks", 1), ("blocks", 4)])
        rot = head_dim if layout == "per_axis" else rng.choice([head_dim, head_dim // 2])
        heads = rng.randint(1, 72)
        rows = _log(rng, 1, max(1, min(32768, 32768 * 40 * 128 // (2 * heads * head_dim))))
        return dict(op=op, dtype=rng.choice(["bf16", "f32"]), rows=rows, heads=heads, extra=rng.randint(0, 8),
                    head_dim=head_dim, rot=rot, axes=axes, layout=layout)
    heads, kv_heads = rng.choice(_HEADS)
    dtype = rng.choice(["bf16", "bf16", "f32"])
    head_dim, page = rng.choice([64, 128, 128]), rng.choice([8, 16, 32, 64, 128, 256])
    if op == "append":
        chunk = rng.choice([1, 1, _log(rng, 2, 2000)])
        seqs = _log(rng, 1, 256 if chunk == 1 else max(1, min(32, 24000 // chunk)))
        return dict(op=op, src=rng.choice(["f32", "bf16"]), dtype=dtype, seqs=seqs, heads=heads, kv_heads=kv_heads,
                    head_dim=head_dim, page=page, own=_log(rng, 1, 2000), chunk=chunk, axes=rng.choice([0, 1, 3]),
                    norm=dtype == "bf16" and rng.random() < 0.7)
    chunk = rng.choice([1, 1, 1, _log(rng, 2, 500)])
    seqs = _log(rng, 1, 128 if chunk == 1 else 16)
    prefix = rng.choice([0, _log(rng, 1, 32768), _log(rng, 1, 32768)])
    own_ = _log(rng, 1, 4000)
    if dtype == "f32":  # the f32 cache: up to a tenth of the largest case's products
        prefix, own_ = min(prefix, 8192), min(own_, 2000)
    c = dict(op=op, dtype=dtype, seqs=seqs, heads=heads, kv_heads=kv_heads, head_dim=head_dim, page=page,
             prefix=prefix, own=own_, chunk=chunk)
    most = work(listed()[8])["flops"] / (10 if dtype == "f32" else 1)
    while work(c)["flops"] > most or c["seqs"] * c["chunk"] * c["heads"] * (c["prefix"] + c["own"] + c["chunk"]) > 4e8:
        if c["prefix"] >= c["own"]:
            c["prefix"] = c["prefix"] * 2 // 3
        else:
            c["own"] = c["own"] * 2 // 3
    return c


def _lengths(case):
    """(q, past) of each sequence: new rows and positions already cached, from the case alone.
    Decode steps bring one row a sequence; chunked ones 0 to `chunk` rows, a fifth of them none."""
    b = np.arange(case["seqs"], dtype=np.int64)
    past = (b * 7919 + 37) % 101 * case["own"] // 100
    if case["chunk"] == 1:
        return np.ones_like(b), past
    q = 1 + (b * 4099 + 96) % 97 * (case["chunk"] - 1) // 96
    return np.where(b % 5 == 3, 0, q), past


_SIZE = {"bf16": 2, "f32": 4}
_TYPE = {"bf16": torch.bfloat16, "f32": torch.float32}
_POSITIONS = 40960  # rows of the cos/sin tables


def work(case):
    if case["op"] == "mrope":
        n = case["rows"] * case["heads"] * case["head_dim"] * _SIZE[case["dtype"]]
        tables = min(_POSITIONS, case["rows"]) * case["rot"] // 2 * 8
        return {"bytes": 2 * n + tables + 4 * case["axes"] * case["rows"],
                "flops": 3 * case["rows"] * case["heads"] * case["rot"]}
    q, past = _lengths(case)
    rows, D, Hq, Hkv = int(q.sum()), case["head_dim"], case["heads"], case["kv_heads"]
    size = _SIZE[case["dtype"]]
    if case["op"] == "append":
        n = rows * (Hq + 2 * Hkv) * D
        return {"bytes": n * (_SIZE[case["src"]] + size) + min(_POSITIONS, rows) * D * 4 + 4 * case["axes"] * rows,
                "flops": (7 if case["norm"] else 3) * rows * (Hq + Hkv) * D}
    kv = case["prefix"] + int(np.where(q > 0, past + q, 0).sum())
    seen = int((q * (case["prefix"] + past) + q * (q + 1) // 2).sum())
    return {"bytes": 2 * kv * Hkv * D * size + 2 * rows * Hq * D * size, "flops": 4 * seen * Hq * D}


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------

def _axis_of_pair(pairs, axes, layout):
    """The axis whose position turns each rotary pair."""
    i = np.arange(pairs)
    if layout == "cyclic":  # axis 0, 1, 2, 0, 1, 2, ...; what is left over at the end to axis 0
        return np.where(i < pairs // axes * axes - axes, i % axes, 0).astype(np.uint8)
    if layout == "blocks" and axes == 3:  # a quarter, three eighths, three eighths
        return np.where(i < pairs // 4, 0, np.where(i < pairs // 4 + (pairs - pairs // 4) // 2, 1, 2)).astype(np.uint8)
    return np.minimum(i * axes // pairs, axes - 1).astype(np.uint8)


def _tables(pairs, axis, layout, dev):
    i = np.arange(pairs)
    if layout == "per_axis":  # every axis counts its frequencies from the first
        i = i - np.searchsorted(axis, axis)
        pairs = int(i.max()) + 1
    inv = torch.from_numpy(1e6 ** (-i / pairs)).to(dev)
    ang = torch.arange(_POSITIONS, device=dev, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


def _grid_positions(rows, axes, gen, dev):
    """Positions of `axes` axes: runs of text (all axes equal) and of a 24 x 32 grid (its own
    height and width behind a common start)."""
    r = torch.arange(rows, device=dev)
    start = torch.randint(0, 64, (1,), generator=gen, device=dev)
    t = r // 768
    grid = torch.stack([t, r // 32 % 24, r % 32, t])[:axes] if axes > 1 else r[None]
    return ((grid if axes > 1 else r[None] % (_POSITIONS - 64)) + start).to(torch.int32).contiguous()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(int(seed) * 1000003 + 17)

    def normal(*shape, scale=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=gen, device=dev, dtype=torch.float32) * scale).to(dtype)

    s = {"case": dict(case)}
    if case["op"] == "mrope":
        axis = _axis_of_pair(case["rot"] // 2, case["axes"], case["layout"])
        s["cos"], s["sin"] = _tables(case["rot"] // 2, axis, case["layout"], dev)
        s["axis"] = axis
        s["pos"] = _grid_positions(case["rows"], case["axes"], gen, dev)
        # the rotated heads are the first of each projection row
        s["x"] = normal(case["rows"], case["heads"] + case["extra"], case["head_dim"],
                        dtype=_TYPE[case["dtype"]])[:, :case["heads"]]
        s["out"] = torch.empty(s["x"].shape, dtype=s["x"].dtype, device=dev)
        return s

    q, past = _lengths(case)
    kv = past + q
    B, D, Hq, Hkv, page = case["seqs"], case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    dtype = _TYPE[case["dtype"]]
    prefix = case.get("prefix", 0)
    prefix_pages, own_pages = -(-prefix // page), -(-kv // page)
    n_pages = int(prefix_pages + own_pages.sum()) + 3
    ids = torch.randperm(n_pages, generator=gen, device=dev).to(torch.int32).cpu().numpy()
    table = np.zeros((B, max(1, int(own_pages.max()))), np.int32)
    at = np.concatenate([[0], np.cumsum(own_pages)]) + prefix_pages
    for b in range(B):
        table[b, :own_pages[b]] = ids[at[b]:at[b + 1]]
    put = lambda a: torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).to(dev)  # noqa: E731
    s["table"], s["kv_len"] = put(table), put(kv)
    s["prefix_table"] = put(ids[:prefix_pages]) if prefix else None
    s["q_start"] = put(np.concatenate([[0], np.cumsum(q)]))
    s["max_q"], s["max_kv"] = max(1, int(q.max())), max(1, int(kv.max()))
    rows = int(q.sum())
    s["rows"] = rows
    s["k"] = normal(n_pages, Hkv, page, D, dtype=dtype)
    s["v"] = normal(n_pages, Hkv, page, D, dtype=dtype)
    if case["op"] == "append":
        s["qkv"] = normal(rows, (Hq + 2 * Hkv) * D, scale=2.0, dtype=_TYPE[case["src"]])
        axis = _axis_of_pair(D // 2, max(1, case["axes"]), "blocks")
        s["axis"] = axis
        s["cos"], s["sin"] = _tables(D // 2, axis, "blocks", dev)
        s["pos"] = _grid_positions(rows, case["axes"], gen, dev) if case["axes"] else None
        for name in ("q_norm", "k_norm"):
            s[name] = (1 + 0.1 * normal(D, dtype=torch.float32)).to(torch.bfloat16) if case["norm"] else None
        s["q_out"] = torch.empty(rows, Hq, D, dtype=dtype, device=dev)
    else:
        s["q"] = normal(rows, Hq, D, scale=1.5, dtype=dtype)
        s["out"] = torch.empty(rows, Hq, D, dtype=dtype, device=dev)
    return s


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------

def run(s):
    op = s["case"]["op"]
    if not own:
        return {"mrope": _plain_mrope, "append": _plain_append, "attention": _plain_attention}[op](s)
    h = s.get("handles")
    if h is None:  # the views of its own buffers that a program keeps: pointers, sizes, strides
        h = s["handles"] = _handles(s)
    if op == "mrope":
        return h["lq8"].mrope(h["ctx"], s["x"], h["rotary"], s["pos"], out=s["out"])
    if op == "append":
        q = h["cache"].append(s["qkv"], s["case"]["heads"], h["batch"], h["rotary"], pos=s["pos"], q_norm=s["q_norm"],
                              k_norm=s["k_norm"], eps=1e-6, q_out=s["q_out"])
        return q, s["k"], s["v"]
    return h["cache"].attend(s["q"], h["batch"], out=s["out"])


def _handles(s):
    lq8, ctx = _binding()
    h = {"lq8": lq8, "ctx": ctx}
    if "cos" in s:
        h["rotary"] = lq8.Rotary(s["cos"], s["sin"], s["axis"])
    if "k" in s:
        h["cache"] = lq8.PagedKvCache(ctx, s["k"], s["v"])
        h["batch"] = lq8.PagedBatch(s["table"], s["kv_len"], q_start=s["q_start"] if s["case"]["chunk"] > 1 else None,
                                    max_q=s["max_q"], max_kv=s["max_kv"], prefix_table=s["prefix_table"],
                                    prefix_len=s["case"].get("prefix", 0))
    return h


def _turn(x, cos, sin):
    """Rotates pairs (i, i + n) of x [rows, heads, D] by rows' angles [rows, n]; dims past 2n stay."""
    n = cos.shape[1]
    a, b = x[..., :n], x[..., n:2 * n]
    c, d = cos[:, None], sin[:, None]
    return torch.cat([a * c - b * d, b * c + a * d, x[..., 2 * n:]], dim=-1)


def _angles(s, pos):
    """cos and sin [rows, pairs]: pair i at its axis' position."""
    pairs = torch.arange(s["cos"].shape[1], device=pos.device)
    at = pos.long()[torch.from_numpy(s["axis"]).to(pos.device).long()].T
    return s["cos"][at, pairs], s["sin"][at, pairs]


def _plain_mrope(s):
    return _turn(s["x"].float(), *_angles(s, s["pos"])).to(s["x"].dtype)


def _rows_of(s):
    """Sequence and own position of every row."""
    r = torch.arange(s["rows"], device=s["kv_len"].device)
    b = torch.searchsorted(s["q_start"][1:].contiguous(), r.to(torch.int32), right=True)
    return b, (s["kv_len"][b] - s["q_start"][b + 1]).long() + r


def _plain_append(s):
    c = s["case"]
    D, Hq, Hkv = c["head_dim"], c["heads"], c["kv_heads"]
    b, at = _rows_of(s)
    x = s["qkv"].float().view(s["rows"], Hq + 2 * Hkv, D)
    q, k, v = x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]
    if c["norm"]:
        q = q * torch.rsqrt((q * q).mean(-1, keepdim=True) + 1e-6) * s["q_norm"].float()
        k = k * torch.rsqrt((k * k).mean(-1, keepdim=True) + 1e-6) * s["k_norm"].float()
    cos, sin = _angles(s, s["pos"] if s["pos"] is not None else at[None])
    page, off = s["table"][b, at // c["page"]].long(), at % c["page"]
    s["k"][page, :, off] = _turn(k, cos, sin).to(s["k"].dtype)
    s["v"][page, :, off] = v.to(s["v"].dtype)
    return _turn(q, cos, sin).to(s["k"].dtype), s["k"], s["v"]


def _plain_attention(s):
    c = s["case"]
    D, Hq, Hkv, prefix = c["head_dim"], c["heads"], c["kv_heads"], c["prefix"]
    B, G, Q, T = c["seqs"], Hq // Hkv, s["max_q"], s["max_kv"]
    dev = s["q"].device
    b, at = _rows_of(s)
    j = torch.arange(s["rows"], device=dev) - s["q_start"][b].long()
    # the rows of each sequence side by side: [B, Hkv, G * Q, D]
    q = torch.zeros(B, Q, Hq, D, device=dev)
    q[b, j] = s["q"].float() / math.sqrt(D)
    q = q.view(B, Q, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * Q, D)
    pages = -(-T // c["page"])
    own_k = s["k"][s["table"][:, :pages].long()].float().permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    own_v = s["v"][s["table"][:, :pages].long()].float().permute(0, 2, 1, 3, 4).reshape(B, Hkv, -1, D)
    t = torch.arange(own_k.shape[2], device=dev)
    live = t[None] < s["kv_len"][:, None].long()
    own_v = torch.where(live[:, None, :, None], own_v, torch.zeros((), device=dev))
    first = s["kv_len"].long() - (s["q_start"][1:] - s["q_start"][:-1]).long()
    sees = t[None, None] <= first[:, None, None] + torch.arange(Q, device=dev)[None, :, None]
    sees = (sees & live[:, None])[:, None].repeat(1, G, 1, 1).view(B, 1, G * Q, -1)
    scores = torch.matmul(q, own_k.transpose(2, 3)).masked_fill(~sees, -math.inf)
    top = scores.amax(-1, keepdim=True)
    if prefix:
        n = s["prefix_table"].long()
        pk = s["k"][n].float().permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :prefix]
        pv = s["v"][n].float().permute(1, 0, 2, 3).reshape(Hkv, -1, D)[:, :prefix]
        flat = q.permute(1, 0, 2, 3).reshape(Hkv, B * G * Q, D)
        shared = torch.matmul(flat, pk.transpose(1, 2))
        most = shared.amax(-1, keepdim=True).view(Hkv, B, G * Q, 1).permute(1, 0, 2, 3)
        top = torch.maximum(top, most)
        shared = torch.exp(shared - top.permute(1, 0, 2, 3).reshape(Hkv, -1, 1))
        shared_sum = shared.sum(-1, keepdim=True).view(Hkv, B, G * Q, 1).permute(1, 0, 2, 3)
        shared = torch.matmul(shared, pv).view(Hkv, B, G * Q, D).permute(1, 0, 2, 3)
    p = torch.exp(scores - top.clamp_min(-3e38))
    o, total = torch.matmul(p, own_v), p.sum(-1, keepdim=True)
    if prefix:
        o, total = o + shared, total + shared_sum
    o = o / torch.where(total > 0, total, torch.ones((), device=dev))
    o = o.view(B, Hkv, G, Q, D).permute(0, 3, 1, 2, 4).reshape(B, Q, Hq, D)
    return o[b, j].to(s["q"].dtype)


# ---------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    f = torch.float64
    if case["op"] == "mrope":
        return _exact_rotation(s["x"].to(f), s, s["pos"])
    q, past = _lengths(case)
    D, Hq, Hkv, page = case["head_dim"], case["heads"], case["kv_heads"], case["page"]
    table = s["table"].cpu().numpy()
    if case["op"] == "append":
        x = s["qkv"].to(f).reshape(-1, Hq + 2 * Hkv, D)
        position = np.concatenate([np.arange(past[b], past[b] + q[b]) for b in range(len(q))])
        pos = s["pos"] if case["axes"] else torch.from_numpy(position[None]).to(x.device)
        parts = {"q": x[:, :Hq], "k": x[:, Hq:Hq + Hkv]}
        for name in parts:
            y = parts[name]
            if case["norm"]:
                y = y / (y.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * s[name + "_norm"].to(f)
            parts[name] = _exact_rotation(y, s, pos)
        which = np.repeat(np.arange(len(q)), q)
        slot = torch.from_numpy(table[which, position // page].astype(np.int64) * page + position % page).to(x.device)
        out = [parts["q"]]
        for old, new in ((s["k"], parts["k"]), (s["v"], x[:, Hq + Hkv:])):
            flat = old.to(f).transpose(1, 2).reshape(-1, Hkv, D)
            flat[slot] = new
            out.append(flat.reshape(-1, page, Hkv, D).transpose(1, 2).contiguous())
        return tuple(out)
    G, prefix, out, start = Hq // Hkv, case["prefix"], [], 0
    k, v = (t.transpose(0, 1) for t in (s["k"], s["v"]))  # [Hkv, pages, page, D]
    for b in range(len(q)):
        if not q[b]:
            continue
        n, kv = int(q[b]), int(past[b] + q[b])
        rows = s["q"][start:start + n].to(f).view(n, Hkv, G, D).permute(1, 2, 0, 3).reshape(Hkv, G * n, D)
        start += n
        ids = torch.from_numpy(table[b, :-(-kv // page)].astype(np.int64)).to(k.device)
        own_k, own_v = (t[:, ids].reshape(Hkv, -1, D)[:, :kv].to(f) for t in (k, v))
        score = rows @ own_k.mT / math.sqrt(D)
        hidden = torch.arange(kv, device=k.device)[None] > torch.arange(kv - n, kv, device=k.device)[:, None]
        score.view(Hkv, G, n, kv).masked_fill_(hidden, -math.inf)
        if prefix:
            if "pk" not in s:
                ids = s["prefix_table"].long()
                s["pk"], s["pv"] = (t[:, ids].reshape(Hkv, -1, D)[:, :prefix].to(f) for t in (k, v))
            score = torch.cat([rows @ s["pk"].mT / math.sqrt(D), score], dim=-1)
        p = torch.softmax(score, dim=-1)
        o = p[..., prefix:] @ own_v
        if prefix:
            o = o + p[..., :prefix] @ s["pv"]
        out.append(o.view(Hkv, G, n, D).permute(2, 0, 1, 3).reshape(n, Hq, D))
    return torch.cat(out)


def _exact_rotation(x, s, pos):
    """x [rows, heads, D] times the rotation matrices of its rows, as complex numbers."""
    cols = []
    for i, axis in enumerate(s["axis"].tolist()):
        cols.append(torch.complex(s["cos"][pos[axis].long(), i].double(), s["sin"][pos[axis].long(), i].double()))
    w = torch.stack(cols, dim=1)[:, None]
    n = w.shape[-1]
    z = torch.complex(x[..., :n], x[..., n:2 * n]) * w
    return torch.cat([z.real, z.imag, x[..., 2 * n:]], dim=-1)
