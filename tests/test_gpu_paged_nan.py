"""GPU tests of NaN, infinities and scales that are no normal numbers in paged caches. In the attention they reach the rows that see them, whichever
kernel has a row and whether or not its parts go through the merge, and no others. Definitions and
tolerances of the other rows are those of test_gpu_paged.py and test_gpu_paged_q8.py."""
import pytest

import test_gpu_paged as wide
import test_gpu_paged_q8 as q8
from test_gpu_paged import randn, within

pytestmark = pytest.mark.gpu


def check(got, want, tol, bad):
    """NaN in every dim of the rows `bad` (rows, heads), the definition's values in the others."""
    import torch
    assert got[bad].isnan().all()
    within(got[~bad], want[~bad], tol.expand_as(want)[~bad])
    assert bool(torch.isfinite(got[~bad]).all())


# ------------------------------------------------------------------------------------------
# rows of which every score is NaN, behind a prefix: their partials have nothing but the NaN in the sum
# ------------------------------------------------------------------------------------------

KV = [100, 90, 80, 300, 64, 7]


@pytest.mark.parametrize("prefix", [1, 100, 4000])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("rows", [[1] * 6, [1] * 40, [50] + [1] * 5])  # streaming; prefix apart; tiles of 128 rows
def test_rows_that_are_nan_behind_a_prefix(ctx, lq8_lib, rows, D, prefix):
    import torch
    s = q8.Cache(lq8_lib, ctx, KV + [40] * (len(rows) - 6), rows, 2, D, 16, 16, prefix=prefix, seed=31).fill()
    x = randn(32, s.rows, 4, D, dtype="bf16")
    want = q8.attention64(s, x, D ** -0.5)
    at = [int(i) for i in s.start]
    y = x.clone()
    y[at[1], 1, 5] = float("nan")
    y[at[2], 2, 9] = float("inf")
    s.vs[int(s.table[5, 0]), 0] = float("nan")                                  # all that sequence 5 has, kv head 0
    s.ks[torch.as_tensor(s.table[4, :4], device="cuda"), 1] = float("nan")      # all of sequence 4, kv head 1
    got = s.cache.attend(y, s.batch)
    ctx.device_status()
    bad = torch.zeros(s.rows, 4, dtype=torch.bool, device="cuda")
    bad[at[1], 1] = bad[at[2], 2] = True
    bad[at[5], :2] = bad[at[4], 2:] = True
    check(got, want[0], q8.tolerance(want, streaming=False) + q8.tolerance(want), bad)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 1, 100, 4000])
@pytest.mark.parametrize("rows", [[1] * 6, [50] + [1] * 5])
def test_rows_that_are_nan_in_wider_caches(ctx, lq8_lib, dtype, rows, prefix):
    import torch
    s = wide.Setup(lq8_lib, ctx, dtype, KV, rows, 2, 128, 16, prefix, seed=33).fill()
    x = randn(34, s.rows, 4, 128, dtype=dtype)
    want, mass = wide.attention64(s, x, 128 ** -0.5)
    at = [int(i) for i in s.start]
    y = x.clone()
    y[at[1], 1, 5] = float("nan")
    y[at[2], 2, 9] = float("inf")
    s.k[int(s.table[5, 0]), 0, :7] = float("nan")  # all that sequence 5 has, kv head 0
    got = s.cache.attend(y, s.batch)
    ctx.device_status()
    bad = torch.zeros(s.rows, 4, dtype=torch.bool, device="cuda")
    bad[at[1], 1] = bad[at[2], 2] = True
    bad[at[5], :2] = True
    check(got, want, (wide.U[dtype] + 2e-5) * mass + wide.U[dtype] * want.abs(), bad)


# ------------------------------------------------------------------------------------------
# scales that are NaN, in blocks that only the later rows of a sequence see
# ------------------------------------------------------------------------------------------

def spoil(s, places, heads):
    """Scales of (K or V, sequence, kv head, block of positions) become NaN; the rows (rows, heads) that see them."""
    import torch
    bad = torch.zeros(s.rows, heads, dtype=torch.bool, device="cuda")
    G, per = heads // s.n_kv, s.page // s.block
    for which, b, kh, blk in places:
        (s.ks if which == "k" else s.vs)[int(s.table[b, blk // per]), kh, blk % per] = float("nan")
        for j in range(int(s.q[b])):
            if int(s.kv[b] - s.q[b]) + j >= blk * s.block:
                bad[int(s.start[b]) + j, kh * G:(kh + 1) * G] = True
    return bad


def hidden_case(ctx, lq8_lib, kv, q, Hq, Hkv, D, page, block, prefix, places, streaming):
    s = q8.Cache(lq8_lib, ctx, kv, q, Hkv, D, page, block, prefix=prefix, seed=35).fill()
    x = randn(36, s.rows, Hq, D, dtype="bf16")
    want = q8.attention64(s, x, D ** -0.5)
    bad = spoil(s, places, Hq)
    assert bool(bad.any()) and not bool(bad.all())
    got = s.cache.attend(x, s.batch)
    ctx.device_status()
    check(got, want[0], q8.tolerance(want) if streaming else q8.tolerance(want, streaming=False) + q8.tolerance(want), bad)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix", [0, 100])
def test_nan_scales_that_few_rows_see(ctx, lq8_lib, prefix, D):
    """Up to 32 stacked rows: the last rows of a sequence begin a block (of 16, of 64) that the first ones do not see."""
    hidden_case(ctx, lq8_lib, [34, 131, 257, 18], [4, 3, 2, 4], 4, 2, D, 16, 16, prefix,
                [("v", 0, 0, 2), ("k", 0, 1, 2), ("k", 1, 0, 8), ("v", 1, 1, 8), ("v", 2, 0, 16), ("v", 3, 1, 1)], True)
    hidden_case(ctx, lq8_lib, [66, 130], [4, 3], 4, 2, D, 64, 64, prefix, [("v", 0, 0, 1), ("k", 1, 1, 2), ("v", 1, 0, 2)], True)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("prefix", [0, 100, 3000])
@pytest.mark.parametrize("q", [[150, 3, 20, 60], [300, 3, 20, 300], [20, 3, 17, 2]])
def test_nan_scales_that_later_rows_of_a_chunk_see(ctx, lq8_lib, q, prefix, D):
    """More rows: tiles of 128 of them, of up to 64 and of up to 8."""
    import torch
    kv = [q[0] + 7, 33 + 128, q[2] + 40, q[3] + 300]
    places = [("v", 0, 0, (kv[0] - 1) // 16), ("k", 0, 1, (q[0] // 2 + 7) // 16), ("v", 1, 0, 10), ("k", 1, 1, 10),
              ("k", 2, 0, (kv[2] - 1) // 16), ("v", 2, 1, (kv[2] - 9) // 16), ("v", 3, 0, (kv[3] - 1) // 16), ("k", 3, 1, 18)]
    hidden_case(ctx, lq8_lib, kv, q, 6, 2, D, 32, 16, prefix, places, False)
    if prefix:  # a block of the prefix: every row of its kv head, and of no other
        s = q8.Cache(lq8_lib, ctx, kv, q, 2, D, 32, 16, prefix=prefix, seed=37).fill()
        x = randn(38, s.rows, 6, D, dtype="bf16")
        want = q8.attention64(s, x, D ** -0.5)
        s.vs[int(s.ptable[1]), 1, 0] = float("nan")
        bad = torch.zeros(s.rows, 6, dtype=torch.bool, device="cuda")
        bad[:, 3:] = True
        check(s.cache.attend(x, s.batch), want[0], q8.tolerance(want, streaming=False) + q8.tolerance(want), bad)
        ctx.device_status()


# ------------------------------------------------------------------------------------------
# scales below the normal numbers
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("tiny", [2.0 ** -130, 2.0 ** -149, 1.1e-38, 0.0])
@pytest.mark.parametrize("block", [16, 128])
def test_append_behind_a_scale_below_the_normal_numbers(ctx, lq8_lib, tiny, block):
    """A cache that its owner filled: such a scale counts as zero, as one that an append works out does."""
    import torch
    from test_gpu_paged import i32
    D = 64
    c = lq8_lib.PagedKvCacheQ8.empty(ctx, 3, 128, 1, D, block)
    for t in (c.k, c.v):
        t.fill_(5)
    for t in (c.k_scale, c.v_scale):
        t.fill_(tiny)
    rotary, table = lq8_lib.Rotary.build(0, 1, 1e4), i32([[0], [1], [2]])
    x = randn(3, 3, 3 * D)
    x[0, D:] = 0.0
    x[1, D:] = 1e-40
    c.append(x, 1, lq8_lib.PagedBatch(table, i32([2, 2, 2])), rotary)
    ctx.device_status()
    both = lq8_lib.PagedBatch(table, i32([2, 2, 2]), q_start=i32([0, 2, 4, 6]), max_q=2)
    for w, (codes, scale, got) in enumerate(zip((c.k, c.v), (c.k_scale, c.v_scale), c.read(both, rows=6, dtype=torch.float32))):
        assert not codes[:2, 0, 1].any() and not scale[:2, 0, 0].any() and not got[:4].any()
        want = x[2, (w + 1) * D:(w + 2) * D]
        assert not codes[2, 0, 0].any() and int(codes[2, 0, 1].abs().max()) == 127 and not got[4].any()
        assert float((got[5, 0] - want).abs().max()) <= float(want.abs().max()) / 127 * 0.51
