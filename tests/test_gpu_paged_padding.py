"""GPU tests of attention calls whose rows are all padding, next to ordinary ones on one stream."""
import pytest

import test_gpu_paged as wide
import test_gpu_paged_q8 as q8
from test_gpu_paged import i32, randn

pytestmark = pytest.mark.gpu


def cache_of(lq8_lib, ctx, dtype, kv, prefix, seed):
    if dtype == "q8":
        return q8.Cache(lq8_lib, ctx, kv, [1] * len(kv), 2, 128, 16, 16, prefix=prefix, seed=seed).fill()
    return wide.Setup(lq8_lib, ctx, dtype, kv, [1] * len(kv), 2, 128, 16, prefix, seed=seed).fill()


@pytest.mark.parametrize("dtype", ["q8", "bf16", "f32"])
@pytest.mark.parametrize("seqs,pad", [(6, 6), (60, 200), (60, 3000)])  # few rows in all; the prefix apart; a long call
def test_a_call_of_padding_alone_ends_before_the_next_one_begins(ctx, lq8_lib, dtype, seqs, pad):
    """The padding's call computes on the prefix for nothing, in the workspace that the next call uses."""
    import torch
    s = cache_of(lq8_lib, ctx, dtype, [40 + 13 * b for b in range(seqs)], 4000, 41)
    x = randn(42, seqs, 8, 128, dtype="f32" if dtype == "f32" else "bf16")
    want = s.cache.attend(x, s.batch).clone()
    b = s.batch
    none = lq8_lib.PagedBatch(b.page_table, b.kv_len, q_start=i32([0] * (seqs + 1)), max_q=1, max_kv=b.max_kv, prefix_table=b.prefix_table,
                              prefix_len=b.prefix_len)
    y = randn(43, pad, 8, 128, dtype="f32" if dtype == "f32" else "bf16")
    idle = torch.full_like(y, 5.0)
    outs = [torch.empty_like(x) for _ in range(30)]
    torch.cuda.synchronize()
    for out in outs:
        s.cache.attend(y, none, out=idle)
        s.cache.attend(x, b, out=out)
    ctx.device_status()
    assert all(torch.equal(o, want) for o in outs) and bool((idle == 5.0).all())
