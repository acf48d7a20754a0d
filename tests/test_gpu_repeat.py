"""GPU tests that a call gives the same bits every time, while another stream keeps memory and the SMs' load paths busy
with gathers of rows: stages of weights are copied in by the copy engine while others are read."""
import ctypes as C

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


class Busy:
    """Gathers on another stream, a few ahead of the calls under test."""

    def __init__(self):
        import torch
        self.stream = torch.cuda.Stream()
        with torch.cuda.stream(self.stream):
            self.rows = torch.zeros(1 << 16, 512, device="cuda")
            self.at = torch.randint(0, 1 << 16, (4096,), device="cuda")
            self.out = torch.empty(4096, 512, device="cuda")

    def go(self):
        import torch
        with torch.cuda.stream(self.stream):
            torch.index_select(self.rows, 0, self.at, out=self.out)


@pytest.mark.parametrize("n,k", [(25600, 5120), (5120, 25600), (4096, 4096)])
@pytest.mark.parametrize("m", [1, 4, 8, 16, 32, 64])
def test_matmul_repeats(ctx, lq8_lib, n, k, m):
    import torch
    gen = torch.Generator(device="cuda")
    gen.manual_seed(m)
    q = lambda r: torch.randint(-127, 128, (r, k), generator=gen, device="cuda", dtype=torch.int32).to(torch.int8)  # noqa: E731
    d = lambda r: (torch.rand(r, k // 32, generator=gen, device="cuda") * 0.01 + 0.005).to(torch.float16).view(torch.int16)  # noqa: E731
    wq, wd, xq, xd = q(n), d(n), q(m), d(m)
    w = lq8_lib.Q8Tensor(n, k, wq.data_ptr(), wd.data_ptr())

    def call():
        y = torch.empty(m, n, device="cuda")
        ctx.call("lq_q8_0_matmul", C.byref(w), xq.data_ptr(), xd.data_ptr(), m, y.data_ptr(), None, 0)
        return y

    want, busy = call(), Busy()
    torch.cuda.synchronize()
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(150):
        if i % 4 == 0:
            busy.go()
        wrong += (call() != want).any()
    torch.cuda.synchronize()
    ctx.device_status()
    assert int(wrong) == 0


@pytest.mark.parametrize("B", [1, 4, 8])
def test_decode_steps_repeat(ctx, lq8_lib, B):
    import torch
    cfg = lq8_lib.make_config(hidden=2048, layers=3, n_heads=16, n_kv_heads=8, head_dim=128, inter=6144, vocab=151936, max_pos=40960,
                              tied=0, eps=1e-6, theta=1e6, init_std=0.02, norm_std=0.0)
    m = lq8_lib.Qwen3ForCausalLM(ctx, cfg, 7, max_batch=B, ctx_max=160)
    prompts = np.random.default_rng(1).integers(0, 151936, (B, 70)).astype(np.int32)
    busy, want = Busy(), None
    for _ in range(8):
        m.clear_kv_cache()
        m.set_batch(B)
        tok, got = m.prefill(prompts), []
        for _ in range(12):
            for _ in range(3):
                busy.go()
            tok, logits = m.decode_step(tok, want_logits=True)
            got.append(logits)
        if want is None:
            want = got
        assert all(np.array_equal(a, b) for a, b in zip(got, want))
    torch.cuda.synchronize()
    m.close()


@pytest.mark.parametrize("kind", ["f32", "bf16", "q8"])
@pytest.mark.parametrize("seqs,new,prefix", [(12, 1, 1000), (70, 1, 5000), (48, 1, 0), (6, 90, 700)])
def test_paged_attention_repeats(ctx, lq8_lib, kind, seqs, new, prefix):
    import torch
    import test_gpu_paged as wide
    import test_gpu_paged_q8 as q8
    kv, q = [new + 37 * (b % 60) for b in range(seqs)], [new] * seqs
    if kind == "q8":
        s = q8.Cache(lq8_lib, ctx, kv, q, 4, 128, 16, 16, prefix=prefix, seed=61).fill()
    else:
        s = wide.Setup(lq8_lib, ctx, kind, kv, q, 4, 128, 16, prefix, seed=61).fill()
    x = wide.randn(62, s.rows, 16, 128, dtype="f32" if kind == "f32" else "bf16")
    want, busy = s.cache.attend(x, s.batch), Busy()
    torch.cuda.synchronize()
    wrong = torch.zeros((), dtype=torch.int64, device="cuda")
    for i in range(100):
        if i % 4 == 0:
            busy.go()
        wrong += (s.cache.attend(x, s.batch) != want).any()
    torch.cuda.synchronize()
    ctx.device_status()
    assert int(wrong) == 0
