"""The shared-prompt serving example against the contiguous path and the model runner.

Tolerances: with an f32 cache and the runner's rounding points both paths do the same arithmetic up
to the order of f32 sums, which can move a Q8_0 activation by one step (1/127 of a block's
largest): 1e-2 of the largest logit over two layers and seven steps. A bf16 cache rounds k, v, q
and the probabilities by up to 2^-8 each (and leaves out the f32 path's rounding of the norm to
bf16, the same size): 2e-2 for each of the two layers."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("image", [True, False])
@pytest.mark.parametrize("dtype,tol", [("float32", 1e-2), ("bfloat16", 4e-2)])
def test_shared_prompt_serving(ctx, lq8_lib, dtype, tol, image):
    import torch
    import shared_prefix_serving as ex
    got, want, runner = ex.serve(getattr(torch, dtype), image, ctx=ctx)
    assert got.shape == want.shape == (7, 3, 1000) and torch.isfinite(got).all()
    assert float((got - want).abs().max()) <= tol * float(want.abs().max())
    if runner is not None:
        assert float((got - runner).abs().max()) <= tol * float(runner.abs().max())
