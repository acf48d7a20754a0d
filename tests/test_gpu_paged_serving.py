"""GPU tests of the paged-serving operators in a server's conditions: large ragged batches, captured
graphs and streams next to other calls, padding, and calls that are refused. Definitions and
tolerances are those of test_gpu_paged.py."""
import numpy as np
import pytest

from test_gpu_paged import Setup, attention_case, randn

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


@pytest.mark.parametrize("kv,q,prefix,page", [
    ([40 + 7 * (b % 90) for b in range(300)], [1] * 300, 0, 16),    # few rows a segment, flows apart
    ([40 + 7 * (b % 90) for b in range(300)], [1] * 300, 2000, 64),
    ([300, 500, 40] * 6, [200, 300, 3] * 6, 1000, 32),              # prompt chunks
])
def test_attention_whose_waits_run_out(ctx, lq8_lib, monkeypatch, kv, q, prefix, page):
    """LQ_FAULT=prefix_attn_wait: every CTA stops handing out work after 0 to 7 batches, so that the
    waits of its other warps run out. The call ends, the error is reported, and the next call is
    right."""
    import torch
    s = Setup(lq8_lib, ctx, "bf16", kv, q, 2, 128, page, prefix, seed=3, garbage=False).fill()
    x = randn(3, s.rows, 8, 128, dtype="bf16")
    want = s.cache.attend(x, s.batch)
    ctx.device_status()
    for _ in range(3):
        monkeypatch.setenv("LQ_FAULT", "prefix_attn_wait")
        s.cache.attend(x, s.batch)
        monkeypatch.delenv("LQ_FAULT")
        with pytest.raises(lq8_lib.LQ8Error, match="code 94"):
            ctx.device_status()
        assert torch.equal(s.cache.attend(x, s.batch), want)
        ctx.device_status()


def test_f32_attention_whose_waits_run_out(ctx, lq8_lib, monkeypatch):
    """The same for an f32 cache: every wait for a copy gives up at once, with the copies in flight."""
    import torch
    s = Setup(lq8_lib, ctx, "f32", [40 + 7 * (b % 90) for b in range(300)], [1] * 300, 2, 128, 16, 500, seed=3, garbage=False).fill()
    x = randn(3, s.rows, 8, 128)
    want = s.cache.attend(x, s.batch)
    ctx.device_status()
    for _ in range(3):
        monkeypatch.setenv("LQ_FAULT", "prefix_attn_wait")
        s.cache.attend(x, s.batch)
        monkeypatch.delenv("LQ_FAULT")
        with pytest.raises(lq8_lib.LQ8Error, match="code 95"):
            ctx.device_status()
        assert torch.equal(s.cache.attend(x, s.batch), want)
        ctx.device_status()
