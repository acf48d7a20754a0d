"""GPU tests of the paged-serving operators against their definitions in 64 bits.

Tolerances, with u = 2^-8 the unit roundoff of a bf16 output (0 for f32):
- rotation: two products and a sum in f32, one rounding: 2^-22 (|x| + |x'|) + u |y| for a pair
  (x, x') (twice the first-order bound);
- append with norm weights: the f32 norm adds a tree sum of squares, a square root, a division and
  two products, under 32 roundings in all: 2^-19 (|x| + |x'|) + u |y| on the normalised pair;
- attention, bf16: each probability is rounded to bf16 once (u sum p |v| at most), the result once
  (u |o|), and f32 sums and exponentials stay within 2e-5 sum p |v| (scores of the size drawn
  here; the framework's tolerance for its f32 attention); f32: the last term alone.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {"bf16": 2.0 ** -8, "f32": 0.0}


def dtype_of(name):
    import torch
    return {"bf16": torch.bfloat16, "f32": torch.float32}[name]


def randn(seed, *shape, scale=1.0, dtype="f32"):
    import torch
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype_of(dtype))


def i32(a):
    import torch
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def turn64(x, cos, sin, pos, axis, sign=1.0):
    """The rotation's definition: x [rows, heads, D] f64, pos [axes, rows], tables f32."""
    import torch
    n = cos.shape[1]
    a = torch.as_tensor(np.zeros(n, np.int64) if axis is None else axis.astype(np.int64), device=x.device)
    at = pos.long()[a].T
    c = cos[at, torch.arange(n, device=x.device)].double()[:, None]
    s = sign * sin[at, torch.arange(n, device=x.device)].double()[:, None]
    p, q = x[..., :n], x[..., n:2 * n]
    return torch.cat([p * c - q * s, q * c + p * s, x[..., 2 * n:]], -1)


def pair_size(x, n):
    """|x| + |x'| of each dim's rotary pair (|x| alone past the rotated ones)."""
    import torch
    m = x[..., :n].abs() + x[..., n:2 * n].abs()
    return torch.cat([m, m, x[..., 2 * n:].abs()], -1)


def within(got, want, tol):
    import torch
    assert torch.isfinite(got).all()
    over = (got.double() - want).abs() - tol
    assert float(over.max()) <= 0, f"exceeds the tolerance by {float(over.max()):.3e}"


# ------------------------------------------------------------------------------------------
# rotary positions with several axes
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,heads,D,rot,kind", [
    (1, 1, 128, 128, "text"), (3, 5, 128, 128, "cyclic"), (257, 72, 128, 128, "blocks"), (7, 4, 64, 32, "cyclic"),
    (33, 9, 80, 80, "per_axis"), (5, 3, 72, 72, "per_axis"), (6, 2, 256, 256, "blocks"), (4, 7, 6, 2, "text"),
    (11, 300, 96, 96, "four"), (9, 3, 128, 0, "text")])
def test_mrope(ctx, lq8_lib, dtype, rows, heads, D, rot, kind):
    import torch
    n = rot // 2
    axis = {"text": None, "cyclic": lq8_lib.Rotary.cyclic([n - 2 * (n // 4), n // 4, n // 4]),
            "blocks": lq8_lib.Rotary.blocks([n - 2 * (n // 4), n // 4, n // 4]),
            "per_axis": lq8_lib.Rotary.blocks([n // 2, n - n // 2]),
            "four": lq8_lib.Rotary.blocks([n // 4, n // 4, n // 4, n - 3 * (n // 4)])}[kind]
    rot_t = lq8_lib.Rotary.build(n, 4000, 1e4, axis, per_axis=kind == "per_axis")
    pos = i32(np.random.default_rng(rows).integers(0, 4000, (4, rows)))
    x = randn(rows * 7 + D, rows, heads + 2, D, dtype=dtype)[:, 1:heads + 1]
    y = lq8_lib.mrope(ctx, x, rot_t, pos)
    want = turn64(x.double(), rot_t.cos, rot_t.sin, pos, axis)
    within(y, want, 2.0 ** -22 * pair_size(x.double(), n) + U[dtype] * want.abs())
    if rot < D:
        assert torch.equal(y[..., rot:], x[..., rot:])
    # the inverse, written over its input
    z = y.clone()
    assert lq8_lib.mrope(ctx, z, rot_t, pos, out=z, inverse=True) is z
    back = turn64(y.double(), rot_t.cos, rot_t.sin, pos, axis, -1.0)
    within(z, back, 2.0 ** -22 * pair_size(y.double(), n) + U[dtype] * back.abs())
    ctx.device_status()


def test_mrope_unaligned_rows_and_head_stride(ctx, lq8_lib):
    import torch
    rot = lq8_lib.Rotary.build(64, 100, 1e4)
    pos = i32(np.arange(5))
    buf = randn(3, 5, 4 * 131 + 1, dtype="bf16")
    x = torch.as_strided(buf, (5, 4, 128), (buf.stride(0), 131, 1), 1)  # odd address, odd strides
    y = lq8_lib.mrope(ctx, x, rot, pos)
    want = turn64(x.double(), rot.cos, rot.sin, pos[None], None)
    within(y, want, 2.0 ** -22 * pair_size(x.double(), 64) + U["bf16"] * want.abs())


def test_mrope_inverse_is_the_gradient(ctx, lq8_lib):
    """d/dx <g, R x> = R^T g: the inverse turn of g, against central differences."""
    import torch
    axis = lq8_lib.Rotary.cyclic([24, 20, 20])
    rot = lq8_lib.Rotary.build(64, 50, 1e4, axis)
    pos = i32([[3, 7], [1, 40], [9, 2]])
    x, g = randn(1, 2, 3, 128), randn(2, 2, 3, 128)
    grad = lq8_lib.mrope(ctx, g, rot, pos, inverse=True)
    for r, h, d in [(0, 0, 0), (1, 2, 63), (0, 1, 64), (1, 0, 127)]:
        e = torch.zeros_like(x)
        e[r, h, d] = 0.5
        up, dn = lq8_lib.mrope(ctx, x + e, rot, pos), lq8_lib.mrope(ctx, x - e, rot, pos)
        diff = float(((up.double() - dn.double()) * g.double()).sum())
        # the map is linear: the difference is exact but for f32 rounding of its values
        assert abs(diff - float(grad[r, h, d])) <= 2.0 ** -20 * float(g.abs().sum())


def test_mrope_position_outside_the_tables_is_reported(ctx, lq8_lib):
    import torch
    rot = lq8_lib.Rotary.build(64, 10, 1e4)
    x = randn(4, 3, 2, 128)
    out = torch.full_like(x, 7.0)
    lq8_lib.mrope(ctx, x, rot, i32([0, 10, -1]), out=out)
    with pytest.raises(lq8_lib.LQ8Error) as e:
        ctx.device_status()
    assert "code 90" in str(e.value)
    assert (out[1:] == 7.0).all() and (out[0] != 7.0).any()
    ctx.device_status()  # reported once


# ------------------------------------------------------------------------------------------
# a paged cache with sequences, for the append and the attention
# ------------------------------------------------------------------------------------------

class Setup:
    """Pages with garbage (NaN and infinities) everywhere but where a sequence or the prefix has a
    position; page ids in no order, three pages that nobody owns."""

    def __init__(self, lq8_lib, ctx, dtype, kv, q, n_kv, D, page, prefix=0, seed=0, layers=1, layer=0, garbage=True):
        import torch
        rng = np.random.default_rng(seed)
        self.kv, self.q = np.asarray(kv, np.int64), np.asarray(q, np.int64)
        self.page, self.prefix, self.D, self.n_kv, self.dtype = page, prefix, D, n_kv, dtype
        own, pp = -(-self.kv // page), -(-prefix // page)
        self.n_pages = int(own.sum()) + pp + 3
        ids = rng.permutation(self.n_pages)
        self.table = np.full((len(kv), max(1, int(own.max(initial=0)) + 1)), -7, np.int64)  # unused entries: no page
        at = pp
        for b in range(len(kv)):
            self.table[b, :own[b]] = ids[at:at + own[b]]
            at += own[b]
        self.ptable = ids[:pp]
        buf = torch.full((2, self.n_pages, layers, n_kv, page, D), float("nan"), dtype=dtype_of(dtype), device="cuda")
        if garbage:
            buf[0, ::2] = float("inf")
        else:
            buf.zero_()
        self.k, self.v = buf[0][:, layer], buf[1][:, layer]
        self.seed = seed
        self.start = np.concatenate([[0], np.cumsum(self.q)])
        self.rows = int(self.start[-1])
        self.cache = lq8_lib.PagedKvCache(ctx, self.k, self.v)
        one = bool((self.q == 1).all())
        self.batch = lq8_lib.PagedBatch(i32(self.table), i32(self.kv), q_start=None if one else i32(self.start),
                                        max_q=max(1, int(self.q.max(initial=0))), max_kv=int(self.kv.max(initial=0)),
                                        prefix_table=i32(self.ptable) if prefix else None, prefix_len=prefix)

    def slots(self, b=None):
        """(page, offset) of a sequence's own positions, or of the prefix."""
        n = self.prefix if b is None else int(self.kv[b])
        p = np.arange(n)
        t = self.ptable if b is None else self.table[b]
        return t[p // self.page], p % self.page

    def fill(self):
        """Values for every position of the prefix and of the sequences."""
        for x in (self.k, self.v):
            self.seed += 1000
            for b in [None, *range(len(self.kv))]:
                pg, off = self.slots(b)
                if len(pg):
                    self.seed += 1
                    x[i32(pg).long(), :, i32(off).long()] = randn(self.seed, len(pg), self.n_kv, self.D, dtype=self.dtype)
        return self

    def read(self, x, b=None):
        """[n_kv, positions, D] in f64."""
        pg, off = self.slots(b)
        return x[i32(pg).long(), :, i32(off).long()].double().transpose(0, 1)


# ------------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------------

def append_case(ctx, lq8_lib, src, dtype, kv, q, Hq, Hkv, D, page, rot, norm, axes, seed=5, layers=1, bf16_rule=False):
    import torch
    s = Setup(lq8_lib, ctx, dtype, kv, q, Hkv, D, page, seed=seed, layers=layers, layer=layers - 1)
    n = rot // 2
    axis = None if axes <= 1 else lq8_lib.Rotary.cyclic([n - 2 * (n // 4), n // 4, n // 4])
    rotary = lq8_lib.Rotary.build(n, 5000, 1e4, axis)
    rows = s.rows
    qkv = randn(seed, rows, (Hq + 2 * Hkv) * D + 4, scale=2.0, dtype=src)[:, :(Hq + 2 * Hkv) * D]
    own = np.concatenate([np.arange(a - b, a) for a, b in zip(s.kv, s.q)] or [[]]).astype(np.int64)
    pos = i32(np.random.default_rng(seed).integers(0, 5000, (3, rows))) if axes else None
    qn, kn = ((1 + 0.2 * randn(seed + i, D)).to(torch.bfloat16) if norm else None for i in (1, 2))
    before = s.k.clone(), s.v.clone()
    q_out = s.cache.append(qkv, Hq, s.batch, rotary, pos=pos, q_norm=qn, k_norm=kn, eps=1e-6, norm_bf16=bf16_rule)
    ctx.device_status()
    x = qkv.double().view(rows, Hq + 2 * Hkv, D)
    at = pos if axes else i32(own[None])

    def expect(y, w):
        if w is not None:
            y = y / (y.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        want = turn64(y, rotary.cos, rotary.sin, at, axis)
        return want, 2.0 ** -19 * pair_size(y, n) + U[dtype] * want.abs()

    within(q_out, *expect(x[:, :Hq], qn))
    b = np.repeat(np.arange(len(s.q)), s.q)
    pg, off = i32(s.table[b, own // page]).long(), i32(own % page).long()
    within(s.k[pg, :, off], *expect(x[:, Hq:Hq + Hkv], kn))
    assert torch.equal(s.v[pg, :, off], qkv.view(rows, Hq + 2 * Hkv, D)[:, Hq + Hkv:].to(s.v.dtype)) if rows else True
    # nothing else is written
    for x, old in ((s.k, before[0]), (s.v, before[1])):
        keep = torch.ones(s.n_pages, page, dtype=torch.bool, device="cuda")
        keep[pg, off] = False
        bits = torch.int16 if dtype == "bf16" else torch.int32
        now, was = (t.transpose(1, 2)[keep].contiguous().view(bits) for t in (x, old))
        assert torch.equal(now, was)


@pytest.mark.parametrize("src,dtype", [("f32", "bf16"), ("bf16", "bf16"), ("f32", "f32"), ("bf16", "f32")])
@pytest.mark.parametrize("kv,q,Hq,Hkv,D,page,rot,norm,axes", [
    ([1], [1], 1, 1, 128, 8, 128, False, 0),
    ([5, 16, 17, 33], [1, 1, 1, 1], 16, 8, 128, 16, 128, True, 0),
    ([40, 7, 0, 9, 200], [13, 7, 0, 1, 150], 8, 2, 128, 32, 128, True, 3),
    ([40, 7, 9], [40, 0, 2], 5, 1, 64, 64, 64, True, 3),
    ([12, 300], [12, 290], 4, 2, 256, 128, 256, False, 3),
    ([12, 30], [3, 4], 6, 3, 80, 16, 80, True, 0),      # a head dimension of the general kernel
    ([12, 30], [3, 4], 4, 4, 128, 16, 64, True, 1),     # rotated in part
    ([9, 3], [3, 2], 3, 1, 34, 8, 12, False, 3),
    ([2] * 1500, [1] * 1500, 4, 1, 64, 8, 64, False, 0)])
def test_append(ctx, lq8_lib, src, dtype, kv, q, Hq, Hkv, D, page, rot, norm, axes):
    append_case(ctx, lq8_lib, src, dtype, kv, q, Hq, Hkv, D, page, rot, norm, axes)


def test_append_many_ragged_sequences(ctx, lq8_lib):
    """Rows find their sequence among thousands, with runs of sequences that bring none."""
    rng = np.random.default_rng(3)
    q = rng.integers(0, 3, 3000)
    q[100:1400] = 0
    append_case(ctx, lq8_lib, "f32", "bf16", q + rng.integers(0, 20, 3000), q, 2, 1, 64, 8, 64, False, 0)


def test_append_into_one_layer_of_many(ctx, lq8_lib):
    append_case(ctx, lq8_lib, "bf16", "bf16", [40, 7, 9], [13, 7, 1], 8, 2, 128, 16, 128, True, 3, layers=3)


def test_append_equals_qk_norm_rope_kv_bit_for_bit(ctx, lq8_lib):
    """With the reference's rounding points, the f32 cache gets what the contiguous cache gets."""
    import torch
    B, Hq, Hkv, D, T = 3, 16, 8, 128, 60
    ct = torch.empty((T, 64), device="cuda")
    st = torch.empty_like(ct)
    ctx.call("lq_rope_tables", D, T, 1e6, ct.data_ptr(), st.data_ptr())
    qkv = randn(8, B, (Hq + 2 * Hkv) * D, scale=3.0)
    qn, kn = ((1 + 0.1 * randn(i, D)).to(torch.bfloat16) for i in (1, 2))
    q0 = torch.zeros(B, Hq, 1, D, device="cuda")
    kc, vc = torch.zeros(B, Hkv, T, D, device="cuda"), torch.zeros(B, Hkv, T, D, device="cuda")
    ctx.call("lq_qk_norm_rope_kv", qkv.data_ptr(), B, 1, Hq, Hkv, D, qn.data_ptr(), kn.data_ptr(), 1e-6, ct.data_ptr(),
             st.data_ptr(), 41, None, q0.data_ptr(), kc.data_ptr(), vc.data_ptr(), T)
    s = Setup(lq8_lib, ctx, "f32", [42] * B, [1] * B, Hkv, D, 16)
    q1 = s.cache.append(qkv, Hq, s.batch, lq8_lib.Rotary(ct, st), q_norm=qn, k_norm=kn, eps=1e-6, norm_bf16=True)
    assert torch.equal(q1, q0[:, :, 0])
    for b in range(B):
        assert torch.equal(s.read(s.k, b)[:, 41], kc[b, :, 41].double())
        assert torch.equal(s.read(s.v, b)[:, 41], vc[b, :, 41].double())


def test_append_padding_rows_and_reported_errors(ctx, lq8_lib):
    import torch
    rot = lq8_lib.Rotary.build(32, 100, 1e4)

    def setup():
        return Setup(lq8_lib, ctx, "f32", [3, 5], [1, 2], 1, 64, 8, garbage=False)

    qkv = randn(1, 6, 3 * 64)
    s = setup()  # three rows, then three of padding
    out = torch.full((6, 1, 64), 9.0, device="cuda")
    s.cache.append(qkv, 1, s.batch, rot, q_out=out)
    ctx.device_status()
    assert (out[3:] == 9.0).all() and (out[:3] != 9.0).any(-1).all()
    for code, field, value in [(92, "page_table", s.n_pages), (92, "page_table", -1), (91, "kv_len", 1000), (91, "kv_len", 0)]:
        s = setup()
        getattr(s.batch, field).view(-1)[0] = value
        s.cache.append(qkv[:3].contiguous(), 1, s.batch, rot)
        with pytest.raises(lq8_lib.LQ8Error) as e:
            ctx.device_status()
        assert f"code {code}" in str(e.value)
        assert not s.k[s.table[0, 0]].any()     # the row without a slot is skipped,
        assert s.k[s.table[1, 0]].any()         # the others are not


# ------------------------------------------------------------------------------------------
# attention
# ------------------------------------------------------------------------------------------

def attention64(s, q, scale):
    """(o, sum p |v|) of every row in f64; rows that see nothing give zeros."""
    import torch
    Hkv, D = s.n_kv, s.D
    rows, Hq = q.shape[0], q.shape[1]
    G = Hq // Hkv
    o = torch.zeros(rows, Hq, D, dtype=torch.float64, device="cuda")
    a = torch.zeros_like(o)
    pk, pv = s.read(s.k), s.read(s.v)
    for b in range(len(s.q)):
        r0, n = int(s.start[b]), int(s.q[b])
        if n == 0:
            continue
        k, v = torch.cat([pk, s.read(s.k, b)], 1), torch.cat([pv, s.read(s.v, b)], 1)
        x = q[r0:r0 + n].double().view(n, Hkv, G, D).permute(1, 2, 0, 3)
        sc = torch.einsum("hgnd,htd->hgnt", x, k) * scale
        t = torch.arange(k.shape[1], device="cuda")
        last = s.prefix + int(s.kv[b]) - n + torch.arange(n, device="cuda")
        sees = (t[None] <= last[:, None]) | (t[None] < s.prefix)
        sc = sc.masked_fill(~sees, float("-inf"))
        p = torch.nan_to_num(torch.softmax(sc, -1)) if k.shape[1] else sc
        o[r0:r0 + n] = torch.einsum("hgnt,htd->nhgd", p, v).reshape(n, Hq, D)
        a[r0:r0 + n] = torch.einsum("hgnt,htd->nhgd", p, v.abs()).reshape(n, Hq, D)
    return o, a


def attention_case(ctx, lq8_lib, dtype, kv, q, Hq, Hkv, D, page, prefix, qscale=1.5, seed=11, layers=1, scale=None):
    s = Setup(lq8_lib, ctx, dtype, kv, q, Hkv, D, page, prefix, seed=seed, layers=layers, layer=layers - 1).fill()
    x = randn(seed, s.rows, Hq, D, scale=qscale, dtype=dtype)
    out = s.cache.attend(x, s.batch, scale=scale)
    ctx.device_status()
    want, mass = attention64(s, x, D ** -0.5 if scale is None else scale)
    if s.rows:
        within(out, want, (U[dtype] + 2e-5) * mass + U[dtype] * want.abs())
    return s, x, out


SHAPES = [
    # kv, q, prefix
    ([1], [1], 0),                                              # one position
    ([0, 3], [1, 1], 0),                                        # a row that sees nothing
    ([0, 0, 0], [1, 1, 1], 5),                                  # nothing but the prefix
    ([1, 7, 8, 9, 127, 128, 129, 300], [1] * 8, 0),             # around page and tile ends
    ([1, 40, 128, 257], [1] * 4, 1),
    ([5, 64, 200, 0, 33], [1] * 5, 127),
    ([5, 64, 200, 1, 33], [1] * 5, 128),
    ([17] * 40, [1] * 40, 129),                                 # more than one tile of stacked rows
    ([30, 2, 0, 90, 140], [3, 2, 0, 90, 1], 300),               # ragged new rows
    ([400, 129], [400, 129], 0),                                # prompts, causal
    ([260, 515, 1], [130, 257, 1], 77),
    ([4, 2], [6, 2], 9),                                        # more rows than own positions
    ([4, 2], [6, 2], 0),                                        # ... some see nothing at all
    ([1030], [1], 2500),
]


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Hq,Hkv,D,page", [(8, 2, 128, 16), (8, 1, 64, 8), (3, 3, 128, 128), (5, 1, 128, 32),
                                           (28, 4, 64, 64), (64, 8, 128, 256), (96, 1, 128, 16)])
@pytest.mark.parametrize("kv,q,prefix", SHAPES)
def test_attention(ctx, lq8_lib, dtype, Hq, Hkv, D, page, kv, q, prefix):
    attention_case(ctx, lq8_lib, dtype, kv, q, Hq, Hkv, D, page, prefix)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv,q,Hq,Hkv,D,page,prefix", [
    ([600 + 37 * b for b in range(20)], [1] * 20, 64, 8, 128, 16, 9000),   # long prefix, split over the SMs
    ([3 + 40 * (b % 7) for b in range(200)], [1] * 200, 32, 8, 128, 32, 1000),
    ([9000, 20], [1, 1], 8, 2, 128, 64, 0),
    ([5000, 700], [1500, 700], 16, 8, 128, 64, 3000),
    ([2] * 1500, [1] * 1500, 4, 1, 64, 8, 100),                            # more sequences than threads
])
def test_attention_long(ctx, lq8_lib, dtype, kv, q, Hq, Hkv, D, page, prefix):
    attention_case(ctx, lq8_lib, dtype, kv, q, Hq, Hkv, D, page, prefix)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("kv,q,Hq,Hkv,D,page,prefix", [
    # a chunk next to many decode rows: the prefix keeps blocks over all sequences
    ([200] + [3] * 39, [200] + [1] * 39, 32, 8, 128, 16, 2000),
    ([70, 1, 300, 0, 50] * 6, [70, 1, 40, 2, 1] * 6, 28, 4, 64, 32, 1500),
    # chunks of whole blocks: each takes the prefix and its own positions in one go
    ([600, 300], [600, 300], 16, 2, 128, 256, 129),
    ([700, 64, 900], [513, 64, 200], 32, 4, 64, 256, 640),
    ([0, 513, 40], [300, 513, 100], 8, 1, 128, 8, 255),      # rows before their first own position
    ([2000], [256], 64, 8, 128, 64, 4097),
    ([33], [33], 96, 1, 128, 128, 1),
])
def test_attention_chunks_behind_a_prefix(ctx, lq8_lib, dtype, kv, q, Hq, Hkv, D, page, prefix):
    attention_case(ctx, lq8_lib, dtype, kv, q, Hq, Hkv, D, page, prefix)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("qscale", [0.0, 40.0])
def test_attention_flat_and_sharp(ctx, lq8_lib, dtype, qscale):
    """Equal probabilities, and scores in the hundreds whose maximum moves from tile to tile
    (their own f32 rounding is 2^-24 of the score: an extra 2^-23 |score| sum p |v|)."""
    s = Setup(lq8_lib, ctx, dtype, [700, 90], [1, 40], 2, 128, 16, 1000, seed=4).fill()
    x = randn(4, s.rows, 8, 128, scale=qscale, dtype=dtype)
    out = s.cache.attend(x, s.batch)
    want, mass = attention64(s, x, 128 ** -0.5)
    top = qscale * 128 ** 0.5 * 6  # |score| stays below: |q||k|/sqrt(128), six deviations
    within(out, want, (U[dtype] + 2e-5 + 128 * 2.0 ** -24 * top) * mass + U[dtype] * want.abs())


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_scale_layer_view_and_strided_rows(ctx, lq8_lib, dtype):
    import torch
    s, x, out = attention_case(ctx, lq8_lib, dtype, [30, 200], [4, 1], 8, 2, 128, 16, 50, layers=3, scale=0.03)
    wide = torch.full((s.rows, 11, 128), 5.0, dtype=x.dtype, device="cuda")
    wide[:, :8] = x
    into = torch.full((s.rows, 10, 128), 6.0, dtype=x.dtype, device="cuda")
    s.cache.attend(wide[:, :8], s.batch, scale=0.03, out=into[:, :8])
    assert torch.equal(into[:, :8], out) and (into[:, 8:] == 6.0).all()


def test_attention_offsets_past_32_bits(ctx, lq8_lib):
    """Pages so far apart that element offsets leave 32 bits."""
    import torch
    n, Hkv, page, D, stride = 5, 2, 16, 128, 1 << 29
    buf = torch.empty(4 * stride + Hkv * page * D * 2, dtype=torch.bfloat16, device="cuda")
    k = torch.as_strided(buf, (n, Hkv, page, D), (stride, page * D, D, 1), 0)
    v = torch.as_strided(buf, (n, Hkv, page, D), (stride, page * D, D, 1), Hkv * page * D)
    cache = lq8_lib.PagedKvCache(ctx, k, v)
    rot = lq8_lib.Rotary.build(64, 100, 1e4)
    qkv = randn(1, 40, (4 + 2 * Hkv) * D)
    batch = lq8_lib.PagedBatch(i32([[4, 0, 3]]), i32([40]), q_start=i32([0, 40]), max_q=40)
    q = cache.append(qkv, 4, batch, rot)
    out = cache.attend(q, batch)
    ctx.device_status()
    small = lq8_lib.PagedKvCache.empty(ctx, n, page, Hkv, D, torch.bfloat16)
    small.append(qkv, 4, batch, rot)
    assert torch.equal(small.k[4], k[4]) and torch.equal(small.v[3, :, :8], v[3, :, :8])
    assert torch.equal(small.attend(q, batch), out)
    del buf, k, v, cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_q8_rows(ctx, lq8_lib, oracle, dtype):
    """The Q8_0 rows: for an f32 cache the quantization of the f32 output, bit for bit; for bf16 of
    the value before its rounding, so within a step (d) and the rounding of the output."""
    import torch
    s = Setup(lq8_lib, ctx, dtype, [30, 200, 0], [4, 1, 1], 2, 128, 16, 300, seed=9).fill()
    x = randn(9, s.rows, 8, 128, dtype=dtype)
    xq = torch.empty(s.rows, 8 * 128, dtype=torch.int8, device="cuda")
    xd = torch.empty(s.rows, 32, dtype=torch.int16, device="cuda")
    out = s.cache.attend(x, s.batch, quantized=(xq, xd)).float().view(s.rows, -1)
    only = torch.empty_like(xq)
    lens = s.batch
    ctx.call("lq_prefix_attention", x.data_ptr(), s.cache.dtype, 0, s.rows, 8, 2, 128, 128 ** -0.5, *s.cache._pages,
             s.n_pages, 16, 0, lens.prefix_table.data_ptr(), 300, *lens._seqs, 4, 200, None, 0, only.data_ptr(),
             xd.data_ptr())
    ctx.device_status()
    assert torch.equal(only, xq)
    d = xd.view(torch.float16).float()
    if dtype == "f32":
        oq, od = oracle.q8_0_quantize(out.cpu().numpy())
        assert np.array_equal(xq.cpu().numpy(), oq) and np.array_equal(xd.cpu().numpy().view(np.uint16), od)
    else:
        back = xq.float().view(s.rows, 32, 32) * d[..., None]
        err = (back - out.view(s.rows, 32, 32)).abs()
        amax = out.view(s.rows, 32, 32).abs().amax(-1, keepdim=True)
        assert (err <= amax / 127 * 0.51 + amax * 2.0 ** -8 + amax * 2.0 ** -10).all()


def test_attention_is_deterministic_and_free_of_the_batch_order(ctx, lq8_lib):
    """The same call twice gives the same bits, between other calls too."""
    import torch
    for dtype in ("bf16", "f32"):
        s, x, out = attention_case(ctx, lq8_lib, dtype, [600, 90, 33, 0] * 8, [1] * 32, 16, 4, 128, 16, 2000)
        attention_case(ctx, lq8_lib, dtype, [60, 9], [60, 1], 8, 8, 64, 16, 20)
        for _ in range(3):
            assert torch.equal(s.cache.attend(x, s.batch), out)


def test_append_then_attend_in_a_graph_with_growing_lengths(ctx, lq8_lib):
    """A captured step (append, attend) replayed while kv_len advances on the device equals the
    same steps called one by one."""
    import torch
    Hq, Hkv, D, page, prefix, B, steps = 8, 2, 128, 16, 200, 3, 20
    rot = lq8_lib.Rotary.build(64, 1000, 1e4)
    rows = randn(5, steps, B, (Hq + 2 * Hkv) * D)

    def world():
        s = Setup(lq8_lib, ctx, "bf16", [10 + steps, 3 + steps, steps], [1] * B, Hkv, D, page, prefix, seed=2).fill()
        s.batch.kv_len.copy_(i32([10, 3, 0]))
        return s

    a = world()
    want = []
    for t in range(steps):
        a.batch.kv_len.add_(1)
        want.append(a.cache.attend(a.cache.append(rows[t], Hq, a.batch, rot), a.batch).clone())
    b = world()
    qkv, q, out = rows[0].clone(), torch.empty(B, Hq, D, dtype=torch.bfloat16, device="cuda"), None
    out = torch.empty_like(q)
    b.cache.attend(q.zero_(), b.batch, out=out)  # the workspace exists before the capture
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=ctx._torch_stream):
        b.batch.kv_len.add_(1)
        b.cache.append(qkv, Hq, b.batch, rot, q_out=q)
        b.cache.attend(q, b.batch, out=out)
    for t in range(steps):
        qkv.copy_(rows[t])
        g.replay()
        assert torch.equal(out, want[t])
    ctx.device_status()


def test_attention_on_another_stream(ctx, lq8_lib):
    """The context moved to another stream, back and forth without waiting in between."""
    import torch
    s, x, out = attention_case(ctx, lq8_lib, "bf16", [600, 90, 33, 0] * 8, [1] * 32, 16, 4, 128, 16, 2000)
    t, y, out2 = attention_case(ctx, lq8_lib, "bf16", [60, 900], [60, 1], 8, 8, 64, 16, 20)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    home = ctx.stream
    got = [torch.empty_like(out) for _ in range(6)] + [torch.empty_like(out2) for _ in range(6)]
    torch.cuda.synchronize()
    try:
        for i in range(6):
            ctx.check(ctx.lib.lq_set_stream(ctx.h, other.cuda_stream))
            s.cache.attend(x, s.batch, out=got[i])
            ctx.check(ctx.lib.lq_set_stream(ctx.h, home))
            t.cache.attend(y, t.batch, out=got[6 + i])
    finally:
        ctx.check(ctx.lib.lq_set_stream(ctx.h, home))
    torch.cuda.synchronize()
    assert all(torch.equal(g, out) for g in got[:6]) and all(torch.equal(g, out2) for g in got[6:])


def test_attention_reports_bad_lengths_and_pages(ctx, lq8_lib):
    import torch

    def setup():
        return Setup(lq8_lib, ctx, "bf16", [30, 50], [1, 1], 2, 128, 16, 40, seed=6, garbage=False).fill()

    x = randn(1, 2, 4, 128, dtype="bf16")
    good = setup()
    ref = good.cache.attend(x, good.batch)
    for code, field, at, value in [(92, "page_table", 0, 10 ** 6), (92, "page_table", 0, -5), (91, "kv_len", 0, 51),
                                   (91, "kv_len", 0, -1), (92, "prefix_table", 1, 10 ** 6)]:
        s = setup()
        getattr(s.batch, field).view(-1)[at] = value
        got = s.cache.attend(x, s.batch)
        with pytest.raises(lq8_lib.LQ8Error) as e:
            ctx.device_status()
        assert f"code {code}" in str(e.value)
        if field != "prefix_table":
            assert torch.equal(got[1], ref[1])  # the other sequence is unharmed
    s = Setup(lq8_lib, ctx, "bf16", [30, 50], [2, 1], 2, 128, 16, 40, seed=6, garbage=False).fill()
    s.batch.max_q = 1
    s.cache.attend(randn(1, 3, 4, 128, dtype="bf16"), s.batch)
    with pytest.raises(lq8_lib.LQ8Error) as e:
        ctx.device_status()
    assert "code 93" in str(e.value)


# ------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------

def test_refusals(ctx, lq8_lib):
    import torch
    L = lq8_lib
    rot = L.Rotary.build(64, 100, 1e4)
    x = randn(0, 4, 2, 128)
    pos = i32(np.arange(4))

    def bad(fn, *what):
        with pytest.raises((ValueError, L.LQ8Error)) as e:
            fn()
        for w in what:
            assert w in str(e.value), str(e.value)

    bad(lambda: L.mrope(ctx, x.half(), rot, pos), "neither float32 nor bfloat16")
    bad(lambda: L.mrope(ctx, x[..., ::2], rot, pos), "contiguous dims")
    bad(lambda: L.mrope(ctx, x, rot, pos[:3]), "expected")
    bad(lambda: L.mrope(ctx, x, rot, pos.long()), "int32")
    bad(lambda: L.mrope(ctx, x[..., :100], rot, pos), "rot_dim")
    bad(lambda: L.mrope(ctx, x, rot, pos, out=torch.empty_like(x)[:, :1].expand(4, 2, 128)), "overlap")
    bad(lambda: L.Rotary(rot.cos, rot.sin, np.zeros(63)), "one axis a pair")
    bad(lambda: L.mrope(ctx, x, L.Rotary(rot.cos, rot.sin, np.full(64, 2)), pos), "expected")
    bad(lambda: L.mrope(ctx, x, L.Rotary(rot.cos, rot.sin, np.full(64, 4)), i32(np.zeros((5, 4)))), "n_axes")
    assert L.mrope(ctx, x[:0], rot, pos[:0]).shape == (0, 2, 128)

    k = torch.zeros(4, 2, 16, 128, device="cuda")
    bad(lambda: L.PagedKvCache(ctx, k.half(), k.half()), "neither")
    bad(lambda: L.PagedKvCache(ctx, k, k.bfloat16()), "one type")
    bad(lambda: L.PagedKvCache(ctx, k.transpose(1, 2), k.transpose(1, 2)), "dense inside")
    bad(lambda: L.PagedKvCache(ctx, k[:1].expand(4, 2, 16, 128), k[:1].expand(4, 2, 16, 128)), "apart")
    cache = L.PagedKvCache(ctx, k, torch.zeros_like(k))
    table, lens = i32([[0, 1], [2, 3]]), i32([3, 4])
    batch = L.PagedBatch(table, lens)
    bad(lambda: L.PagedBatch(table, lens[:1]), "one row a sequence")
    bad(lambda: L.PagedBatch(table, lens, q_start=i32([0, 1])), "n_seqs + 1")
    bad(lambda: L.PagedBatch(table, lens, prefix_len=3), "page table")
    bad(lambda: L.PagedBatch(table.long(), lens), "int32")
    bad(lambda: L.PagedBatch(i32(np.zeros((2, 4)))[:, :2], lens), "contiguous")
    qkv = randn(0, 2, 8 * 128)
    bad(lambda: cache.append(qkv, 3, batch, rot), "contiguous values")
    bad(lambda: cache.append(qkv[:1].expand(2, 1024), 4, batch, rot), "contiguous values")
    bad(lambda: cache.append(qkv.double(), 4, batch, rot), "neither")
    bad(lambda: cache.append(qkv, 4, batch, rot, q_norm=torch.ones(128, device="cuda")), "norm weights")
    bad(lambda: cache.append(randn(0, 3, 8 * 128), 4, batch, rot), "one row")
    bad(lambda: cache.append(qkv, 4, batch, L.Rotary(rot.cos, rot.sin, np.arange(64) % 3)), "several axes")
    bad(lambda: cache.append(qkv, 4, batch, rot, q_out=torch.empty(2, 4, 128, device="cuda").bfloat16()), "cache's type")
    q = randn(0, 2, 4, 128)
    bad(lambda: cache.attend(q.bfloat16(), batch), "cache's type")
    bad(lambda: cache.attend(randn(0, 2, 3, 128), batch), "head counts")
    bad(lambda: cache.attend(randn(0, 2, 4, 256)[..., ::2], batch), "cache's type")
    bad(lambda: cache.attend(q, L.PagedBatch(table, lens, max_q=0)), "max_q")
    bad(lambda: cache.attend(randn(0, 3, 4, 128), batch), "one row")
    odd = torch.zeros(4 * 2 * 16 * 128 + 1, device="cuda")[1:].view(4, 2, 16, 128)
    bad(lambda: L.PagedKvCache(ctx, odd, odd).attend(q, batch), "16 bytes")
    k96 = torch.zeros(4, 2, 16, 96, device="cuda")
    bad(lambda: L.PagedKvCache(ctx, k96, k96).attend(randn(0, 2, 4, 96), batch), "64 or 128")
    k12 = torch.zeros(4, 2, 12, 128, device="cuda")
    bad(lambda: L.PagedKvCache(ctx, k12, k12).attend(q, batch), "page_size")
    assert cache.attend(q[:0], batch).shape == (0, 4, 128)
    ctx.device_status()


def test_injected_faults(ctx, lq8_lib, monkeypatch):
    for name in ("lq_mrope", "lq_paged_append", "lq_prefix_attention", "lq_device_status"):
        monkeypatch.setenv("LQ_FAULT", name)
        n = len(lq8_lib.SIGNATURES[name][1]) - 1
        zeros = [0.0 if t.__name__ == "c_float" else 0 for t in lq8_lib.SIGNATURES[name][1][1:]]
        assert getattr(ctx.lib, name)(ctx.h, *zeros[:n]) == -5
        monkeypatch.delenv("LQ_FAULT")
