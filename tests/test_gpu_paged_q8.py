"""GPU tests of the operators on a paged cache in 8 bits against their definitions in 64 bits.

Tolerances, with u = 2^-8 the unit roundoff of a bf16 output (0 for f32):
- append, query rows: as the f32 and bf16 caches' append, 2^-19 (|x| + |x'|) + u |y| on the normalised
  pair (x, x');
- append, codes: with a the block's largest |y|, a pair's |x| + |x'| is at most 2 a = 254 steps, so that
  y is off by at most 2^-19 254 < 0.0005 steps, and the scale, a / 127, by as much for a code of 127:
  a code is within 0.5 + 0.001 (and 2^-10 for the f32 product by the scale's reciprocal) of the exact
  quotient, the scale within 2^-17 of its own size; given the f32 values, codes and scales are exact;
- codes rounded again, and rows read back: exact, in f32;
- attention with up to 32 stacked rows a kv head: q is rounded to amax / 65024 at most, which moves a
  score by at most d = c amax / 65024 sum |k| and a weight by a factor within e^(+-2d); f32 sums and
  exponentials stay within 2e-5 sum p |v| (the framework's tolerance for its f32 attention), the result
  is rounded once, u |o|. Weights p, times V's scale s, are rounded
  to whole 1 / 32512 parts of the largest p s of their 128 positions (the tiles begin at the prefix's and
  at the own positions' first), half of that at most: codes are up to 127, so that a tile gives at most
  128 127 max(p s) / 65024; w is the sum of 128 127 max(p s) over the tiles;
- attention with more: q is exact, a weight (times V's scale) is rounded to 16 bits once, at most u sum
  p |v|; the rest as above;
- both: a weight below 2^-126 of the largest is zero in f32 (and flushed). Over up to 2^13 positions of
  |v| < 2^3 that is up to 2^-110, where the 64-bit result may be the like of 1e-116."""
import numpy as np
import pytest

from test_gpu_paged import i32, pair_size, randn, turn64, within

pytestmark = pytest.mark.gpu

U = 2.0 ** -8


class Cache:
    """Pages with garbage (codes of any value, scales NaN or infinite) everywhere but where a sequence or the
    prefix has a position; page ids in no order, three pages that nobody owns."""

    def __init__(self, lq8_lib, ctx, kv, q, n_kv, D, page, block, prefix=0, seed=0, layers=1, layer=0):
        import torch
        rng = np.random.default_rng(seed)
        self.kv, self.q = np.asarray(kv, np.int64), np.asarray(q, np.int64)
        self.page, self.block, self.prefix, self.D, self.n_kv, self.seed = page, block, prefix, D, n_kv, seed
        own, pp = -(-self.kv // page), -(-prefix // page)
        self.n_pages = int(own.sum()) + pp + 3
        ids = rng.permutation(self.n_pages)
        self.table = np.full((len(kv), max(1, int(own.max(initial=0)) + 1)), -7, np.int64)  # unused entries: no page
        at = pp
        for b in range(len(kv)):
            self.table[b, :own[b]] = ids[at:at + own[b]]
            at += own[b]
        self.ptable = ids[:pp]
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        codes = torch.randint(-128, 128, (2, self.n_pages, layers, n_kv, page, D), generator=g, device="cuda", dtype=torch.int32).to(torch.int8)
        scales = torch.full((2, self.n_pages, layers, n_kv, page // block), float("nan"), device="cuda")
        scales[:, ::2] = float("inf")
        self.k, self.v, self.ks, self.vs = codes[0][:, layer], codes[1][:, layer], scales[0][:, layer], scales[1][:, layer]
        self.all = codes, scales
        self.start = np.concatenate([[0], np.cumsum(self.q)])
        self.rows = int(self.start[-1])
        self.cache = lq8_lib.PagedKvCacheQ8(ctx, self.k, self.v, self.ks, self.vs)
        assert self.cache.block == block
        one = bool((self.q == 1).all())
        self.batch = lq8_lib.PagedBatch(i32(self.table), i32(self.kv), q_start=None if one else i32(self.start),
                                        max_q=max(1, int(self.q.max(initial=0))), max_kv=int(self.kv.max(initial=0)),
                                        prefix_table=i32(self.ptable) if prefix else None, prefix_len=prefix)

    def slots(self, b=None, n=None):
        """(page, offset) of a sequence's own positions, or of the prefix."""
        n = (self.prefix if b is None else int(self.kv[b])) if n is None else n
        p = np.arange(n)
        t = self.ptable if b is None else self.table[b]
        return t[p // self.page], p % self.page

    def fill(self, lengths=None):
        """Codes and scales for every position of the prefix and of the sequences (of the first lengths[b])."""
        import torch
        for x, sc, size in ((self.k, self.ks, 0.02), (self.v, self.vs, 0.03)):
            for b in [None, *range(len(self.kv))]:
                pg, off = self.slots(b, None if b is None or lengths is None else int(lengths[b]))
                if len(pg):
                    self.seed += 1
                    pg, off = i32(pg).long(), i32(off).long()
                    x[pg, :, off] = torch.clamp(randn(self.seed, len(pg), self.n_kv, self.D, scale=40.0).round(), -127, 127).to(torch.int8)
                    new = size * torch.exp(0.5 * randn(self.seed + 10 ** 6, len(pg), self.n_kv))
                    last = torch.arange(len(pg), device="cuda") // self.block * self.block  # one scale a block
                    sc[pg, :, off // self.block] = new[last]
        return self

    def read(self, which, b=None, n=None):
        """[n_kv, positions, D] in f64."""
        x, sc = (self.k, self.ks) if which == "k" else (self.v, self.vs)
        pg, off = (i32(t).long() for t in self.slots(b, n))
        return (x[pg, :, off].double() * sc[pg, :, off // self.block].double()[..., None]).transpose(0, 1)


# ------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------

def make_rows(lq8_lib, s, src, Hq, Hkv, D, rot, norm, axes, seed, pad=8, offset=0):
    import torch
    n = rot // 2
    axis = None if axes <= 1 else lq8_lib.Rotary.cyclic([n - 2 * (n // 4), n // 4, n // 4])
    rotary = lq8_lib.Rotary.build(n, 5000, 1e4, axis)
    width = (Hq + 2 * Hkv) * D
    qkv = randn(seed, s.rows, width + pad, scale=2.0, dtype=src)[:, offset:offset + width]
    pos = i32(np.random.default_rng(seed).integers(0, 5000, (3, s.rows))) if axes else None
    qn, kn = ((1 + 0.2 * randn(seed + i, D)).to(torch.bfloat16) if norm else None for i in (1, 2))
    return rotary, axis, qkv, pos, qn, kn


def own_positions(s):
    return np.concatenate([np.arange(a - b, a) for a, b in zip(s.kv, s.q)] or [[]]).astype(np.int64)


def append_case(ctx, lq8_lib, src, kv, q, Hq, Hkv, D, page, block, rot, norm, axes, seed=5, layers=1, pad=8, offset=0):
    import torch
    s = Cache(lq8_lib, ctx, kv, q, Hkv, D, page, block, seed=seed, layers=layers, layer=layers - 1)
    s.fill(s.kv - s.q)
    rotary, axis, qkv, pos, qn, kn = make_rows(lq8_lib, s, src, Hq, Hkv, D, rot, norm, axes, seed, pad, offset)
    before = [t.clone() for t in s.all]
    older = {(w, b): s.read(w, b, int(s.kv[b] - s.q[b])) for w in "kv" for b in range(len(kv))}
    was = {"k": s.ks.clone(), "v": s.vs.clone()}
    codes_was = {"k": s.k.clone(), "v": s.v.clone()}
    q_out = s.cache.append(qkv, Hq, s.batch, rotary, pos=pos, q_norm=qn, k_norm=kn, eps=1e-6)
    ctx.device_status()
    assert q_out.dtype == torch.bfloat16
    x = qkv.double().view(s.rows, Hq + 2 * Hkv, D)
    own = own_positions(s)
    at = pos if axes else i32(own[None])

    def exact(y, w):
        if w is not None:
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        return turn64(y, rotary.cos, rotary.sin, at, axis), pair_size(y, rot // 2)

    want, size = exact(x[:, :Hq], qn)
    within(q_out, want, 2.0 ** -19 * size + U * want.abs())
    new = {"k": exact(x[:, Hq:Hq + Hkv], kn)[0], "v": x[:, Hq + Hkv:]}
    touched = torch.zeros(s.n_pages, page // block, dtype=torch.bool, device="cuda")
    for b in range(len(kv)):
        n, first = int(s.q[b]), int(s.kv[b] - s.q[b])
        if n == 0:
            continue
        for blk in range(first // block, (int(s.kv[b]) - 1) // block + 1):
            lo, hi = max(first, blk * block), min(int(s.kv[b]), (blk + 1) * block)
            pg, slot = int(s.table[b, lo // page]), blk * block % page // block
            touched[pg, slot] = True
            r0 = int(s.start[b]) + lo - first
            for w, codes, scales in (("k", s.k, s.ks), ("v", s.v, s.vs)):
                y = new[w][r0:r0 + hi - lo].transpose(0, 1)  # [Hkv, rows, D]
                sc = y.abs().amax((1, 2)) / 127
                if lo > blk * block:
                    sc = torch.maximum(sc, was[w][pg, :, slot].double())
                got = scales[pg, :, slot].double()
                assert ((got - sc).abs() <= 2.0 ** -17 * sc).all()
                c = codes[pg, :, lo % page:lo % page + hi - lo].double()
                quotient = y / torch.where(sc > 0, sc, torch.ones_like(sc))[:, None, None]
                assert float((c - quotient).abs().max()) <= 0.5 + 0.001 + 2.0 ** -10
                # the older codes: exactly rint(c old / new) in f32
                old = codes_was[w][pg, :, blk * block % page:lo % page if lo % page else page]
                if lo > blk * block:
                    ratio = (was[w][pg, :, slot] / scales[pg, :, slot])[:, None, None]
                    again = torch.where(scales[pg, :, slot][:, None, None] > was[w][pg, :, slot][:, None, None],
                                        torch.round(old.float().double() * ratio.double()), old.double())
                    assert torch.equal(codes[pg, :, blk * block % page:blk * block % page + lo - blk * block].double(), again)
    # nothing else is written: codes of other positions, scales of other blocks, other layers
    pgs, off = i32(np.concatenate([s.table[b, own[s.start[b]:s.start[b + 1]] // page] for b in range(len(kv))] or [[]])).long(), i32(own % page).long()
    keep = torch.ones(s.n_pages, page, dtype=torch.bool, device="cuda")
    keep[pgs, off] = False
    for b in range(len(kv)):  # (the older positions of a block were looked at above)
        first = int(s.kv[b] - s.q[b])
        if s.q[b] and first % block:
            lo = first // block * block
            keep[int(s.table[b, lo // page]), lo % page:first % page if first % page else page] = False
    for now, old in zip(s.all[0], before[0]):
        assert torch.equal(now[:, layers - 1].transpose(1, 2)[keep], old[:, layers - 1].transpose(1, 2)[keep])
        assert torch.equal(now[:, :layers - 1], old[:, :layers - 1])
    for now, old in zip(s.all[1], before[1]):
        a, o = (t.contiguous().view(torch.int32) for t in (now, old))
        assert torch.equal(a[:, layers - 1].transpose(1, 2)[~touched], o[:, layers - 1].transpose(1, 2)[~touched])
        assert torch.equal(a[:, :layers - 1], o[:, :layers - 1])
    del older
    return s, q_out


@pytest.mark.parametrize("src", ["f32", "bf16"])
@pytest.mark.parametrize("kv,q,Hq,Hkv,D,page,block,rot,norm,axes", [
    ([1], [1], 1, 1, 128, 16, 16, 128, False, 0),
    ([5, 16, 17, 33], [1, 1, 1, 1], 16, 8, 128, 16, 16, 128, True, 0),
    ([40, 7, 0, 9, 200], [13, 7, 0, 1, 150], 8, 2, 128, 32, 16, 128, True, 3),
    ([40, 7, 9, 130, 64], [40, 0, 2, 3, 32], 5, 1, 64, 64, 64, 64, True, 3),
    ([300, 129, 128, 256, 255], [290, 1, 128, 255, 2], 4, 2, 128, 256, 128, 128, False, 3),
    ([77, 31], [60, 2], 3, 3, 64, 32, 32, 64, False, 1),
    ([12, 30], [3, 4], 4, 4, 128, 16, 16, 64, True, 1),     # rotated in part
    ([90, 3], [30, 2], 3, 1, 64, 128, 32, 12, False, 3),
    ([50, 20], [30, 20], 2, 1, 128, 64, 64, 0, True, 0),    # not at all
    ([20] * 700, [1] * 700, 4, 1, 64, 16, 16, 64, False, 0)])
def test_append(ctx, lq8_lib, src, kv, q, Hq, Hkv, D, page, block, rot, norm, axes):
    append_case(ctx, lq8_lib, src, kv, q, Hq, Hkv, D, page, block, rot, norm, axes)


def test_append_rows_at_odd_addresses(ctx, lq8_lib):
    append_case(ctx, lq8_lib, "bf16", [40, 7, 60], [13, 7, 1], 4, 2, 128, 32, 32, 128, True, 3, pad=3, offset=1)


def test_append_into_one_layer_of_many(ctx, lq8_lib):
    append_case(ctx, lq8_lib, "bf16", [40, 7, 9], [13, 7, 1], 8, 2, 128, 16, 16, 128, True, 3, layers=3)


def test_append_many_ragged_sequences(ctx, lq8_lib):
    rng = np.random.default_rng(3)
    q = rng.integers(0, 3, 600)
    q[100:300] = 0
    append_case(ctx, lq8_lib, "f32", q + rng.integers(0, 40, 600), q, 2, 1, 64, 32, 32, 64, False, 0)


@pytest.mark.parametrize("D,norm", [(128, True), (64, False)])
def test_append_quantises_what_the_f32_cache_holds(ctx, lq8_lib, D, norm):
    """Codes and scales from the values of an append into an f32 cache, bit for bit: a prompt, then rows of
    a few tokens, so that blocks begin, go on and are rounded again."""
    import torch
    Hq, Hkv, page, block, steps = 2, 3, 32, 32, [45, 1, 1, 7, 30, 1]
    f = lq8_lib.PagedKvCache.empty(ctx, 8, page, Hkv, D, torch.float32)
    c = lq8_lib.PagedKvCacheQ8.empty(ctx, 8, page, Hkv, D, block)
    table = i32([[5, 2, 7, 0]])
    rotary = lq8_lib.Rotary.build(D // 2, 200, 1e4)
    qn, kn = ((1 + 0.2 * randn(i, D)).to(torch.bfloat16) if norm else None for i in (1, 2))
    model = {w: (torch.zeros(Hkv, 128, D, dtype=torch.float64, device="cuda"), torch.zeros(Hkv, 4, device="cuda")) for w in "kv"}
    done = 0
    for i, n in enumerate(steps):
        qkv = randn(50 + i, n, (Hq + 2 * Hkv) * D, scale=1.0 + 0.3 * i)
        batch = lq8_lib.PagedBatch(table, i32([done + n]), q_start=i32([0, n]), max_q=n)
        qf = f.append(qkv, Hq, batch, rotary, q_norm=qn, k_norm=kn)
        qc = c.append(qkv, Hq, batch, rotary, q_norm=qn, k_norm=kn)
        assert torch.equal(qf.to(torch.bfloat16), qc)
        pos = np.arange(done, done + n)
        pg, off = table[0, i32(pos // page).long()].long(), i32(pos % page).long()
        for w, vals in (("k", f.k), ("v", f.v)):
            codes, scales = model[w]
            x = vals[pg, :, off].transpose(0, 1)
            for blk in range(done // block, (done + n - 1) // block + 1):
                lo, hi = max(done, blk * block), min(done + n, (blk + 1) * block)
                y = x[:, lo - done:hi - done]
                s = (y.abs().amax((1, 2)).double() / 127).float()  # (torch multiplies an f32 tensor by 1 / 127 instead)
                if lo > blk * block:
                    old = scales[:, blk]
                    s = torch.where(s > old, s, old)
                    again = torch.round(codes[:, blk * block:lo] * (old / s).double()[:, None, None])
                    codes[:, blk * block:lo] = torch.where((s > old)[:, None, None], again, codes[:, blk * block:lo])
                codes[:, lo:hi] = torch.round(y.double() * (1.0 / s).double()[:, None, None])
                scales[:, blk] = s
        done += n
        ids = table[0, :-(-done // page)].long()
        for w, got, sc in (("k", c.k, c.k_scale), ("v", c.v, c.v_scale)):
            codes, scales = model[w]
            assert torch.equal(got[ids].transpose(0, 1).reshape(Hkv, -1, D)[:, :done].double(), codes[:, :done])
            assert torch.equal(sc[ids].transpose(0, 1).reshape(Hkv, -1)[:, :-(-done // block)], scales[:, :-(-done // block)])
    ctx.device_status()


def test_append_zeros_tiny_and_non_finite_values(ctx, lq8_lib):
    import torch
    D, page = 64, 16
    c = lq8_lib.PagedKvCacheQ8.empty(ctx, 4, page, 1, D, 16)
    c.k_scale.fill_(7.0), c.v_scale.fill_(7.0)
    rotary = lq8_lib.Rotary.build(0, 1, 1e4)
    table = i32([[0], [1], [2], [3]])
    x = randn(9, 4, 3 * D)
    x[0, D:] = 0.0
    x[1, D:] = 1e-40
    x[2, D + 5] = float("nan")
    x[2, 2 * D + 7] = float("inf")
    batch = lq8_lib.PagedBatch(table, i32([1, 1, 1, 1]))
    c.append(x, 1, batch, rotary)
    k, v = c.read(batch, dtype=torch.float32)
    assert not k[:2].any() and not v[:2].any() and not c.k_scale[:2].any()
    assert k[2].isnan().all() and v[2].isnan().all()
    assert torch.isfinite(k[3]).all() and torch.isfinite(v[3]).all()
    # zeros behind a scale of zero, values behind zeros, finite values behind a NaN, a NaN behind values
    y = randn(10, 4, 3 * D)
    y[0] = 0.0
    y[3, D:] = float("nan")
    later = lq8_lib.PagedBatch(table, i32([2, 2, 2, 2]))
    c.append(y, 1, later, rotary)
    both = lq8_lib.PagedBatch(table, i32([2, 2, 2, 2]), q_start=i32([0, 2, 4, 6, 8]), max_q=2)
    k, v = c.read(both, rows=8, dtype=torch.float32)
    assert not k[:3].any() and float((k[3, 0] - y[1, D:2 * D]).abs().max()) <= float(y[1, D:2 * D].abs().max()) / 127 * 0.51
    assert k[4:].isnan().all() and v[4:].isnan().all()
    # the block's first position again
    c.append(randn(11, 4, 3 * D), 1, batch, rotary)
    k, v = c.read(batch, dtype=torch.float32)
    assert torch.isfinite(k).all() and torch.isfinite(v).all() and k.any(-1).all() and v.any(-1).all()
    ctx.device_status()


def test_append_padding_rows_and_reported_errors(ctx, lq8_lib):
    import torch
    rot = lq8_lib.Rotary.build(32, 100, 1e4)

    def setup():
        s = Cache(lq8_lib, ctx, [3, 5], [1, 2], 1, 64, 16, 16)
        s.all[0].zero_()
        s.all[1].zero_()
        return s

    qkv = randn(1, 6, 3 * 64)
    s = setup()  # three rows, then three of padding
    out = torch.full((6, 1, 64), 9.0, device="cuda", dtype=torch.bfloat16)
    s.cache.append(qkv, 1, s.batch, rot, q_out=out)
    ctx.device_status()
    assert (out[3:] == 9.0).all() and (out[:3] != 9.0).any(-1).all()
    for code, field, at, value in [(92, "page_table", 0, s.n_pages), (92, "page_table", 0, -1), (91, "kv_len", 0, 1000),
                                   (91, "kv_len", 0, 0), (91, "kv_len", 0, -2 ** 31)]:
        s = setup()
        getattr(s.batch, field).view(-1)[at] = value
        s.cache.append(qkv[:3].contiguous(), 1, s.batch, rot)
        with pytest.raises(lq8_lib.LQ8Error) as e:
            ctx.device_status()
        assert f"code {code}" in str(e.value)
        assert not s.k[s.table[0, 0]].any()     # the row without a slot is skipped,
        assert s.k[s.table[1, 0]].any()         # the others are not
    # a position outside the tables: that row's q and k are left out, its v is not
    s = setup()
    s.cache.append(qkv[:3].contiguous(), 1, s.batch, rot, pos=i32([1, 100, 2]))
    with pytest.raises(lq8_lib.LQ8Error) as e:
        ctx.device_status()
    assert "code 90" in str(e.value)
    k, v = s.k[s.table[1, 0], 0], s.v[s.table[1, 0], 0]
    assert not k[3].any() and k[4].any() and v[3].any() and v[4].any() and s.k[s.table[0, 0], 0, 2].any()
    assert int(k[4].abs().max()) == 127  # (the scale is that of the row that counts)
    # row starts that fall
    s = setup()
    s.batch.q_start[1] = 5
    s.cache.append(qkv, 1, s.batch, rot)
    ctx.synchronize()
    try:
        ctx.device_status()
    except lq8_lib.LQ8Error as e:
        assert "code 91" in str(e)


# ------------------------------------------------------------------------------------------
# reading back
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("kv,q,Hkv,D,page,block,layers", [
    ([1], [1], 1, 64, 16, 16, 1), ([33, 5, 64], [1, 1, 1], 8, 128, 32, 16, 1), ([70, 0, 16, 200], [70, 0, 3, 131], 3, 128, 64, 64, 2),
    ([300, 17], [300, 17], 4, 64, 256, 128, 1), ([40] * 90, [7] * 90, 2, 64, 16, 16, 1)])
def test_read(ctx, lq8_lib, dtype, kv, q, Hkv, D, page, block, layers):
    import torch
    dt = getattr(torch, dtype)
    s = Cache(lq8_lib, ctx, kv, q, Hkv, D, page, block, seed=3, layers=layers, layer=layers - 1).fill()
    buf = torch.full((2, s.rows + 2, Hkv * D + 16), 5.0, dtype=dt, device="cuda")  # two rows of padding, rows apart
    outs = [buf[i, :, :Hkv * D].unflatten(1, (Hkv, D)) for i in (0, 1)]
    k, v = s.cache.read(s.batch, *outs) if s.batch.q_start is not None else s.cache.read(s.batch, *(t[:s.rows] for t in outs))
    ctx.device_status()
    for got, w in ((k, "k"), (v, "v")):
        want = torch.cat([s.read(w, b)[:, int(s.kv[b] - s.q[b]):].transpose(0, 1) for b in range(len(kv))])
        assert torch.equal(got[:s.rows], want.float().to(dt))  # (the product of a code and a scale, rounded to f32)
    assert (buf[:, s.rows:] == 5.0).all() and (buf[:, :, Hkv * D:] == 5.0).all()
    k2, v2 = s.cache.read(s.batch, rows=s.rows, dtype=dt)
    assert torch.equal(k2, k[:s.rows]) and torch.equal(v2, v[:s.rows])


def test_read_reports_rows_without_a_slot(ctx, lq8_lib):
    import torch
    for code, field, value in [(92, "page_table", 10 ** 6), (91, "kv_len", 0), (91, "kv_len", 10 ** 6)]:
        s = Cache(lq8_lib, ctx, [20, 30], [1, 1], 2, 64, 16, 16).fill()
        getattr(s.batch, field).view(-1)[0 if field == "kv_len" else 1] = value
        out = torch.full((2, 2, 2, 64), 5.0, device="cuda")
        s.cache.read(s.batch, out[0], out[1])
        with pytest.raises(lq8_lib.LQ8Error) as e:
            ctx.device_status()
        assert f"code {code}" in str(e.value)
        assert (out[:, 0] == 5.0).all() and (out[:, 1] != 5.0).any(-1).all()


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------

def attention64(s, q, scale, dead=()):
    """(o, sum p |v|, d, w) of every row in f64, d and w as in the tolerances; rows that see nothing give
    zeros."""
    import torch
    Hkv, D = s.n_kv, s.D
    rows, Hq = q.shape[0], q.shape[1]
    G = Hq // Hkv
    o = torch.zeros(rows, Hq, D, dtype=torch.float64, device="cuda")
    a = torch.zeros_like(o)
    d = torch.zeros(rows, Hq, 1, dtype=torch.float64, device="cuda")
    w1 = torch.zeros_like(d)
    pk, pv = s.read("k"), s.read("v")
    for b in range(len(s.q)):
        r0, n = int(s.start[b]), int(s.q[b])
        if n == 0 or b in dead:
            continue
        k, v = torch.cat([pk, s.read("k", b)], 1), torch.cat([pv, s.read("v", b)], 1)
        x = q[r0:r0 + n].double().view(n, Hkv, G, D).permute(1, 2, 0, 3)
        sc = torch.einsum("hgnd,htd->hgnt", x, k) * scale
        t = torch.arange(k.shape[1], device="cuda")
        upto = s.prefix + (int(s.kv[b]) - n + torch.arange(n, device="cuda")).clamp_min(-1)
        hidden = t[None] > upto[:, None]
        sc.masked_fill_(hidden, -float("inf"))
        p = torch.nan_to_num(torch.softmax(sc, -1), nan=0.0)
        k1 = k.abs().sum(-1).amax(-1) if k.shape[1] else torch.zeros(Hkv, device="cuda", dtype=torch.float64)
        bound = x.abs().amax(-1) / 65024 * scale * k1[:, None, None]
        for dst, w in ((o, v), (a, v.abs())):
            dst[r0:r0 + n] = torch.einsum("hgnt,htd->hgnd", p, w).permute(2, 0, 1, 3).reshape(n, Hq, D)
        d[r0:r0 + n, :, 0] = bound.permute(2, 0, 1).reshape(n, Hq)
        for which, p1 in ((None, p[..., :s.prefix]), (b, p[..., s.prefix:])):
            pg, off = (i32(u).long() for u in s.slots(which))
            if len(pg):
                ps = p1 * s.vs[pg, :, off // s.block].double().T[:, None, None]
                ps = torch.nn.functional.pad(ps, (0, -ps.shape[-1] % 128)).unflatten(-1, (-1, 128)).amax(-1).sum(-1)
                w1[r0:r0 + n, :, 0] += 128 * 127 * ps.permute(2, 0, 1).reshape(n, Hq)
    return o, a, d, w1


def tolerance(want, streaming=True):
    import torch
    o, a, d, w = want
    if not streaming:
        return 2.0 ** -110 + U * o.abs() + (U + 2e-5) * a
    return 2.0 ** -110 + w / 65024 + U * o.abs() + (torch.expm1(2 * d) + 2e-5) * a


def attention_case(ctx, lq8_lib, kv, q, Hq, Hkv, D, page, block, prefix, seed=11, layers=1, qscale=1.0, quantized=False):
    import torch
    s = Cache(lq8_lib, ctx, kv, q, Hkv, D, page, block, prefix=prefix, seed=seed, layers=layers, layer=layers - 1).fill()
    x = randn(seed + 1, s.rows, Hq + 1, D, scale=qscale, dtype="bf16")[:, :Hq]
    out = torch.full((s.rows, Hq + 1, D), 7.0, device="cuda", dtype=torch.bfloat16)
    xq = None
    if quantized:
        xq = torch.empty(s.rows, Hq * D, dtype=torch.int8, device="cuda"), torch.empty(s.rows, Hq * D // 32, dtype=torch.int16, device="cuda")
    got = s.cache.attend(x, s.batch, out=out[:, :Hq], quantized=xq)
    ctx.device_status()
    assert (out[:, Hq:] == 7.0).all()
    want = attention64(s, x, D ** -0.5)
    # (which kernel ran: more than 32 stacked rows of one kv head take the tensor cores, where it exists)
    within(got, want[0], tolerance(want, streaming=False) + tolerance(want))
    again = s.cache.attend(x, s.batch)
    assert torch.equal(again, got)  # the same bits every time
    if quantized:  # Q8_0 of the rows before bf16: within half a step of the block and the rounding
        d = xq[1].view(torch.float16).double()
        back = (xq[0].double().view(s.rows, -1, 32) * d[..., None]).view(s.rows, Hq, D)
        step = d[..., None].expand(-1, -1, 32).reshape(s.rows, Hq, D)
        within(back, want[0], 0.5 * step * (1 + 2.0 ** -9) + 127 * step * 2.0 ** -11 + tolerance(want, streaming=False) + tolerance(want))
    return s, got


SHAPES = [
    ([1], [1], 1, 1, 128, 16, 16, 0),
    ([40, 1], [1, 1], 16, 8, 128, 16, 16, 100),
    ([5, 16, 17, 33, 700, 0, 1], [1, 1, 1, 1, 1, 0, 1], 16, 8, 128, 16, 16, 0),
    ([5, 16, 17, 33, 700, 2000], [1] * 6, 28, 4, 64, 32, 16, 0),
    ([513, 4000, 1024, 1025], [1] * 4, 64, 8, 128, 64, 64, 0),
    ([300, 600], [1, 1], 12, 4, 64, 128, 128, 0),
    ([1000, 255, 256, 257], [1] * 4, 16, 1, 128, 256, 128, 0),      # 16 rows
    ([90, 300, 7], [4, 2, 3], 8, 2, 128, 32, 32, 0),                # a few tokens a sequence
    ([90, 300, 7], [3, 1, 2], 5, 1, 64, 64, 32, 33),
    ([40, 7, 0, 9, 200], [13, 7, 0, 1, 150], 8, 2, 128, 32, 16, 65),
    ([300, 17, 200], [290, 17, 100], 4, 4, 64, 16, 16, 0),
    ([600, 129], [300, 129], 8, 1, 128, 128, 64, 513),
    ([3] * 300, [1] * 300, 8, 8, 128, 16, 16, 1000),
    ([20, 900] * 40, [1] * 80, 32, 8, 128, 64, 32, 2049),
    ([1, 0, 3], [2, 2, 3], 2, 1, 64, 16, 16, 0),                    # rows before their sequence's first position
    ([1, 0, 3], [2, 2, 3], 40, 1, 128, 16, 16, 5),
]


@pytest.mark.parametrize("kv,q,Hq,Hkv,D,page,block,prefix", SHAPES)
def test_attention(ctx, lq8_lib, kv, q, Hq, Hkv, D, page, block, prefix):
    attention_case(ctx, lq8_lib, kv, q, Hq, Hkv, D, page, block, prefix)


@pytest.mark.parametrize("kv,q,Hq,Hkv,D,prefix", [([77, 500], [1, 1], 8, 2, 128, 0), ([77, 500], [1, 1], 8, 2, 64, 0),
                                                  ([77, 500], [60, 1], 8, 2, 64, 40), ([200, 500], [99, 1], 8, 2, 128, 140)])
def test_attention_quantized_rows_and_layers(ctx, lq8_lib, kv, q, Hq, Hkv, D, prefix):
    attention_case(ctx, lq8_lib, kv, q, Hq, Hkv, D, 32, 32, prefix, layers=3, quantized=True)


@pytest.mark.parametrize("qscale", [1e-3, 30.0])
def test_attention_flat_and_peaked_weights(ctx, lq8_lib, qscale):
    attention_case(ctx, lq8_lib, [3000, 10, 400], [1, 1, 1], 8, 4, 128, 64, 32, 0, qscale=qscale)
    attention_case(ctx, lq8_lib, [700, 10, 400], [100, 3, 50], 8, 4, 128, 64, 32, 300, qscale=qscale)
