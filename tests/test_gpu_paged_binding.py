"""GPU tests of what the binding of the paged caches refuses."""
import pytest

from test_gpu_paged import i32, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,block", [(64, 24), (64, 48), (128, 100), (32, 64), (64, 8), (256, 256), (64, 0), (64, -16)])
def test_blocks_that_an_8_bit_cache_cannot_have(ctx, lq8_lib, page, block):
    """Rounded to the next one that divides a page they would be other blocks than those asked for."""
    import torch
    with pytest.raises(ValueError):
        lq8_lib.PagedKvCacheQ8.empty(ctx, 3, page, 2, 64, block)
    if block > 0 and page % block == 0:
        codes, scales = (torch.zeros(3, 2, page, 64, dtype=torch.int8, device="cuda") for _ in range(2)), (
            torch.zeros(3, 2, page // block, device="cuda") for _ in range(2))
        with pytest.raises(ValueError):
            lq8_lib.PagedKvCacheQ8(ctx, *codes, *scales)
    assert lq8_lib.PagedKvCacheQ8.empty(ctx, 3, 64, 2, 64, 64).block == 64


class Elsewhere:
    """A context on a device that the tensors are not on."""

    def __init__(self, ctx):
        self.lib, self.h, self.device = ctx.lib, ctx.h, 1


@pytest.mark.parametrize("kind", ["q8", "f32", "bf16"])
def test_tensors_on_another_device_than_the_context(ctx, lq8_lib, kind):
    """Their addresses would be read on a device that they do not belong to."""
    import torch
    if kind == "q8":
        c = lq8_lib.PagedKvCacheQ8.empty(ctx, 4, 16, 1, 64)
        parts, make = (c.k, c.v, c.k_scale, c.v_scale), lq8_lib.PagedKvCacheQ8
    else:
        c = lq8_lib.PagedKvCache.empty(ctx, 4, 16, 1, 64, {"f32": torch.float32, "bf16": torch.bfloat16}[kind])
        parts, make = (c.k, c.v), lq8_lib.PagedKvCache
    make(ctx, *parts)
    with pytest.raises(ValueError):
        make(Elsewhere(ctx), *parts)
    batch, rotary = lq8_lib.PagedBatch(i32([[0], [1]]), i32([3, 4])), lq8_lib.Rotary.build(32, 50, 1e4)
    qkv = randn(1, 2, 3 * 64, dtype="bf16")
    q = c.append(qkv, 1, batch, rotary)
    c.attend(q, batch)
    ctx.device_status()
    away = lq8_lib.PagedBatch(i32([[0], [1]]), i32([3, 4]))
    away.device = 1
    turned = lq8_lib.Rotary.build(32, 50, 1e4)
    turned.device = 1
    ones = torch.ones(64, dtype=torch.bfloat16)
    calls = [lambda: c.append(qkv, 1, away, rotary), lambda: c.append(qkv, 1, batch, turned), lambda: c.append(qkv.cpu(), 1, batch, rotary),
             lambda: c.append(qkv, 1, batch, rotary, q_norm=ones), lambda: c.append(qkv, 1, batch, rotary, pos=torch.zeros(2, dtype=torch.int32)),
             lambda: c.append(qkv, 1, batch, rotary, q_out=torch.empty(2, 1, 64, dtype=c.type)), lambda: c.attend(q, away), lambda: c.attend(q.cpu(), batch),
             lambda: c.attend(q, batch, out=torch.empty(2, 1, 64, dtype=c.type)),
             lambda: lq8_lib.mrope(Elsewhere(ctx), q, rotary, i32([[1, 2]])), lambda: lq8_lib.mrope(ctx, q, turned, i32([[1, 2]])),
             lambda: lq8_lib.PagedBatch(i32([[0], [1]]).cpu(), i32([3, 4])), lambda: lq8_lib.PagedBatch(i32([[0], [1]]), i32([3, 4]).cpu())]
    if kind == "q8":
        calls.append(lambda: c.read(away))
    for i, call in enumerate(calls):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {i}")
    ctx.device_status()
