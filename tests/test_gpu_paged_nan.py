"""GPU tests of NaN and infinities in the attention over paged caches: they reach the rows that see them, whichever
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
