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
