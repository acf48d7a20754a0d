"""GPU tests of the paged-serving operators in a server's conditions: large ragged batches, captured
graphs and streams next to other calls, padding, and calls that are refused. Definitions and
tolerances are those of test_gpu_paged.py."""
import numpy as np
import pytest

from test_gpu_paged import attention_case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,prefix", [
    ([4000 * (512 - i) // 512 or 1 for i in range(512)], 0),
    ([32768] * 16 + [100] * 25, 0),
    ([8192] * 64 + [100] * 40, 300),
])
def test_attention_of_ragged_decode_batches(ctx, lq8_lib, kv, prefix):
    """Batches whose CTAs have flows of very unequal length (their schedules end by the CPU's model,
    test_prefix_schedule.py)."""
    attention_case(ctx, lq8_lib, "bf16", kv, [1] * len(kv), 8, 8, 64, 128, prefix)
