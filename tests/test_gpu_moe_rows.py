"""GPU tests of the expert layer's bits: a row's result depends neither on the rows next to it nor on the call.
Every output adds its blocks in ascending order, whatever the pass that a token falls into, so that large batches,
small ones and single rows give the same bits, every time."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


def tensors(gen, n, k):
    import torch
    q = torch.randint(-127, 128, (n, k), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)
    d = (torch.rand(n, k // 32, generator=gen, device="cuda") * 0.01 + 0.005).to(torch.float16).view(torch.int16)
    return q, d


# (experts' weights larger than L2; batches with one and with many passes an expert)
@pytest.mark.parametrize("rows,hidden,E,top_k,inter,calls", [(64, 2048, 32, 8, 768, 600), (512, 2048, 128, 8, 768, 40), (1500, 2048, 32, 4, 768, 20),
                                                             (9, 2048, 128, 8, 768, 200), (200, 512, 64, 8, 256, 100)])
def test_rows_are_independent_and_calls_repeat(ctx, lq8_lib, rows, hidden, E, top_k, inter, calls):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(rows)
    R, GU, DN, X = tensors(gen, E, hidden), tensors(gen, E * 2 * inter, hidden), tensors(gen, E * hidden, inter), tensors(gen, rows, hidden)
    view = lambda t: lq8_lib.Q8Tensor(t[0].shape[0], t[0].shape[1], t[0].data_ptr(), t[1].data_ptr())  # noqa: E731
    router, experts = view(R), lq8_lib.MoeExperts(E, inter, hidden, view(GU), view(DN))

    def call(lo, hi):
        out = torch.empty(hi - lo, hidden, device="cuda")
        ctx.call("lq_moe_forward", C.byref(router), C.byref(experts), X[0][lo:hi].data_ptr(), X[1][lo:hi].data_ptr(), hi - lo, top_k, 1,
                 out.data_ptr(), None, None, None)
        return out

    want = call(0, rows)
    assert torch.isfinite(want).all() and want.any(1).all()
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for _ in range(calls):
        wrong += (call(0, rows) != want).any()
    for n in (64, 7, 1):  # (16 tokens a pass, 8, one row)
        for lo in range(0, rows if n > 1 else min(rows, 40), n):
            hi = min(rows, lo + n)
            wrong += (call(lo, hi) != want[lo:hi]).any()
    ctx.device_status()
    assert int(wrong) == 0
