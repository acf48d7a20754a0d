"""GPU tests of the attention over 8-bit caches, each kernel held to its own roundings (the definition and the streaming
kernel's bound are those of test_gpu_paged_q8.py).

Which kernel has a row follows from the bounds of the call: up to 32 stacked rows (max_q times the group; behind a prefix
all of the call's rows times the group) the streaming one, else the one for tiles of 128 rows. Behind a prefix with many
rows in all and few a sequence the prefix is the latter's and the own positions are the former's, and the errors
add up.

The kernel for tiles has q and codes exact, weights p (times V's scale s) in fp16: each is off by half a step,
2^-11 of itself, or, below fp16's normal numbers, by 2^-25 where a row's largest is 2^7 or more: 2^-32 of the largest
p s, times codes of up to 127, for each of T positions. With w = sum over tiles of 128 127 max(p s), T 127 max(p s) is
at most w times the number of tiles. f32 sums and exponentials stay within 2e-5 sum p |v|, the result is rounded once:
u |o|, u = 2^-8."""
import pytest

from test_gpu_paged import randn, within
from test_gpu_paged_q8 import SHAPES, U, Cache, attention64, tolerance

pytestmark = pytest.mark.gpu

MANY = [
    ([100] * 40, [1] * 40, 8, 2, 128, 16, 16, 300),        # the prefix apart
    ([700, 40, 900], [1, 8, 3], 8, 2, 64, 64, 32, 2000),
    ([4000, 100], [1, 1], 33, 1, 128, 32, 16, 0),          # 33 rows: tiles; 32 of them: streaming
    ([4000, 100], [1, 1], 32, 1, 128, 32, 16, 0),
    ([4000, 100], [1, 1], 16, 1, 64, 32, 16, 900),         # 32 rows in all
    ([900, 100], [9, 4], 4, 1, 128, 32, 16, 0),
    ([900, 1300], [400, 200], 4, 1, 64, 32, 32, 129),
]


@pytest.mark.parametrize("kv,q,Hq,Hkv,D,page,block,prefix", SHAPES + MANY)
def test_each_kernel_within_its_own_bound(ctx, lq8_lib, kv, q, Hq, Hkv, D, page, block, prefix):
    s = Cache(lq8_lib, ctx, kv, q, Hkv, D, page, block, prefix=prefix, seed=51).fill()
    x = randn(52, s.rows, Hq, D, dtype="bf16")
    want = o, a, _, w = attention64(s, x, D ** -0.5)
    got = s.cache.attend(x, s.batch)
    ctx.device_status()
    G = Hq // Hkv
    own_streams = max(1, int(s.q.max())) * G <= 32
    prefix_streams = s.rows * G <= 32 if prefix else own_streams
    tiles = -(-prefix // 128) + max(-(-int(k) // 128) for k in s.kv)
    of_tiles = 2.0 ** -110 + U * o.abs() + (2.0 ** -11 + 2e-5) * a + w * tiles * 2.0 ** -32
    if own_streams and prefix_streams:
        tol = tolerance(want)
    elif not own_streams:
        tol = of_tiles
    else:  # (the result is rounded once)
        tol = of_tiles + tolerance(want) - U * o.abs()
    within(got, o, tol)


@pytest.mark.parametrize("image", [True, False])
def test_the_serving_example_stays_near_the_f32_cache(ctx, lq8_lib, image):
    """Two layers with an 8-bit cache against the contiguous f32 path. A value of a block is off by at most half a step, 1/254 of the
    block's largest, and evenly so: 1/254/sqrt(3) of it in the mean square, about 2^-8.8 of a largest value of about 3.5
    deviations, 0.8 % of a deviation, where bf16 values are off by 2^-9/sqrt(3) of themselves, 0.11 %. Errors of
    128 dims and of the positions are independent, so that scores and outputs are off by about 0.8 % of a
    deviation for each of K and V and layer: 0.8 % sqrt(4) = 1.6 % of the hidden state's part that attention gives, and less
    of the sum with what it is added to. The largest of 21000 logits is 4 deviations and an error of 4.5 of its own
    deviations may be among as many: 1.6 % 4.5 / 4 = 1.8 %. Twice that."""
    import os
    import sys

    import torch
    sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))
    import shared_prefix_serving as ex
    got, want, _ = ex.serve(torch.int8, image, ctx=ctx)
    assert got.shape == want.shape == (7, 3, 1000) and torch.isfinite(got).all()
    assert float((got - want).abs().max()) <= 3.6e-2 * float(want.abs().max())


# ------------------------------------------------------------------------------------------
# row starts that fall
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("prefix,starts,q", [(0, [0, 1, 0, 2], [1, 1, 1]), (40, [0, 30, 2, 33], [1, 1, 31]), (0, [0, 60, 20, 61], [50, 1, 1])])
def test_row_starts_that_fall_are_reported_and_give_nothing(ctx, lq8_lib, prefix, starts, q):
    """Code 93 (a sequence of less than no rows); nothing of the batch is computed: rows keep what they held, or are zero, and
    the next call is right."""
    import torch
    from test_gpu_paged import i32
    s = Cache(lq8_lib, ctx, [70, 200, 64], q, 2, 128, 32, 16, prefix=prefix, seed=2).fill()
    x = randn(2, 70, 4, 128, dtype="bf16")
    y = x[:s.rows].contiguous()
    want = s.cache.attend(y, s.batch)
    b = lq8_lib.PagedBatch(s.batch.page_table, s.batch.kv_len, q_start=i32(starts), max_q=max(b - a for a, b in zip(starts, starts[1:])), max_kv=200, prefix_table=s.batch.prefix_table,
                           prefix_len=prefix)
    for _ in range(3):
        out = torch.full_like(x, 9.0)
        s.cache.attend(x, b, out=out)
        with pytest.raises(lq8_lib.LQ8Error) as e:
            ctx.device_status()
        assert "code 93" in str(e.value)
        assert (out[starts[-1]:] == 9.0).all()  # (rows behind the last sequence's)
        if not prefix:
            assert ((out == 9.0) | (out == 0.0)).all()
        assert torch.equal(s.cache.attend(y, s.batch), want)
        ctx.device_status()


@pytest.mark.parametrize("rot", [64, 32])  # (whole heads, and in part: two kernels)
def test_append_whose_row_starts_fall_stays_in_its_own_pages(ctx, lq8_lib, rot):
    """The sequences' own pages may hold anything afterwards; no other page changes, nor what lies behind the rows."""
    import torch
    from test_gpu_paged import i32
    D = 64
    rotary = lq8_lib.Rotary.build(rot // 2, 400, 1e4)
    for starts in ([0, 5, 3, 6], [0, 2, 0, 1], [0, 40, 1, 2], [0, -3, 4, 6], [0, 3, 2, -5]):
        s = Cache(lq8_lib, ctx, [30, 5, 70], [1, 2, 3], 1, D, 16, 16, seed=4).fill()
        before = [t.clone() for t in s.all]
        out = torch.full((9, 1, D), 9.0, device="cuda", dtype=torch.bfloat16)
        b = lq8_lib.PagedBatch(s.batch.page_table, s.batch.kv_len, q_start=i32(starts), max_q=40, max_kv=100)
        s.cache.append(randn(1, 6, 3 * D), 1, b, rotary, q_out=out[:6])
        try:  # (a row may be found a place that it has not, or none: whatever was met first is reported)
            ctx.device_status()
        except lq8_lib.LQ8Error as e:
            assert any(f"code {c}" in str(e) for c in (91, 92, 93)), str(e)
        ctx.device_status()
        owned = torch.zeros(s.n_pages, dtype=torch.bool, device="cuda")
        for i, kv in enumerate(s.kv):
            owned[i32(s.table[i, :-(-int(kv) // 16)]).long()] = True
        for now, old in zip(s.all, before):
            bits = (lambda t: t.contiguous().view(torch.int32)) if now.dtype == torch.float32 else (lambda t: t)
            assert torch.equal(bits(now[:, ~owned]), bits(old[:, ~owned]))
        assert (out[6:] == 9.0).all()
