"""GPU tests of the paged-serving operators in a server's conditions: large ragged batches, captured
graphs and streams next to other calls, padding, and calls that are refused. Definitions and
tolerances are those of test_gpu_paged.py."""
import numpy as np
import pytest

from test_gpu_paged import U, Setup, attention64, attention_case, i32, randn, within

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


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attention_in_another_batch_order(ctx, lq8_lib, dtype):
    """The same sequences in another order: each result within the tolerance, whatever shares its
    tiles (the bits may differ)."""
    import torch
    kv, n = [600, 90, 33, 1, 250] * 8, 40
    s = Setup(lq8_lib, ctx, dtype, kv, [1] * n, 4, 128, 16, 2000, seed=12).fill()
    x = randn(12, n, 16, 128, scale=1.5, dtype=dtype)
    want, mass = attention64(s, x, 128 ** -0.5)
    for seed in range(3):
        order = np.random.default_rng(seed).permutation(n)
        at = i32(order).long()
        b = lq8_lib.PagedBatch(s.batch.page_table[at].contiguous(), s.batch.kv_len[at], max_kv=600, prefix_table=s.batch.prefix_table,
                               prefix_len=2000)
        out = torch.empty_like(x)
        out[at] = s.cache.attend(x[at], b)
        within(out, want, (U[dtype] + 2e-5) * mass + U[dtype] * want.abs())
    ctx.device_status()


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


# ------------------------------------------------------------------------------------------
# graphs and streams
# ------------------------------------------------------------------------------------------

def decode(ctx, lq8_lib, seqs, prefix, seed):
    """A decode batch: setup, q and the result of a plain call."""
    s = Setup(lq8_lib, ctx, "bf16", [40 + 13 * b for b in range(seqs)], [1] * seqs, 2, 128, 16, prefix, seed=seed, garbage=False).fill()
    x = randn(seed, seqs, 8, 128, dtype="bf16")
    return s, x, s.cache.attend(x, s.batch).clone()


def capture(ctx, s, x):
    import torch
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=ctx._torch_stream):
        s.cache.attend(x, s.batch, out=out)
    return g, out


def test_a_graph_outlives_a_larger_call(ctx, lq8_lib):
    """A captured decode step, then eager calls and captures that need more workspace and memory
    that takes what was freed; the replays give the same bits and write nothing else."""
    import torch
    c = lq8_lib.Context(0)
    s, x, want = decode(c, lq8_lib, 5, 300, 1)
    g, out = capture(c, s, x)
    big, y, _ = decode(c, lq8_lib, 200, 3000, 2)
    taken = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(64)]
    g2, out2 = capture(c, big, y)
    for _ in range(3):
        out.zero_(), out2.zero_()
        g.replay()
        g2.replay()
        assert torch.equal(out, want) and torch.equal(out2, big.cache.attend(y, big.batch))
    assert all(bool((t == 7).all()) for t in taken)
    c.device_status()
    del g, g2
    c.close()


@pytest.mark.parametrize("name,m", [("lq_q8_0_linear", 3), ("lq_q8_0_linear", 16), ("lq_q8_0_matmul", 16), ("lq_q8_0_matmul_prefill", 128)])
def test_a_graph_of_a_linear_outlives_a_larger_call(ctx, lq8_lib, name, m):
    """The layers' buffers next to those of the paged attention: quantized rows, K-split partials, fp16
    operands."""
    import ctypes as C
    import torch
    c = lq8_lib.Context(0)

    def call(n, k, rows, seed):
        t = lq8_lib.QTensor.quantize(c, randn(seed, n, k, scale=0.02))
        w = t.struct()
        x, y = randn(seed + 1, rows, k), torch.zeros(rows, n, device="cuda")
        rows8 = lq8_lib.QTensor.quantize(c, x)
        if name == "lq_q8_0_linear":
            args = (C.byref(w), x.data_ptr(), lq8_lib.DTYPE_F32, rows, y.data_ptr())
        else:
            args = (C.byref(w), rows8.qs.data_ptr(), rows8.d.data_ptr(), rows, y.data_ptr(), None, n)
        return (lambda: c.call(name, *args)), y, (t, w, x, rows8)

    run, y, keep = call(256, 4096, m, 1)
    run()
    want = y.clone()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=c._torch_stream):
        run()
    larger, y2, keep2 = call(1024, 16384, 4 * m, 3)
    larger()
    taken = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(64)]
    y.zero_()
    g.replay()
    assert torch.equal(y, want) and all(bool((t == 7).all()) for t in taken)
    del g
    c.close()


def test_a_capture_may_be_the_first_call(ctx, lq8_lib):
    """No warm-up: the workspace is made while the graph is captured."""
    import torch
    s, x, want = decode(ctx, lq8_lib, 70, 900, 3)
    c = lq8_lib.Context(0)
    cache = lq8_lib.PagedKvCache(c, s.k, s.v)
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=c._torch_stream):
        cache.attend(x, s.batch, out=out)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    del g
    c.close()


def test_replays_next_to_eager_calls_on_another_stream(ctx, lq8_lib):
    import torch
    s, x, want = decode(ctx, lq8_lib, 60, 4000, 4)
    t, y, want2 = decode(ctx, lq8_lib, 90, 3000, 5)
    g, out = capture(ctx, s, x)
    other = torch.cuda.Stream()
    got, got2 = [torch.empty_like(out) for _ in range(20)], [torch.empty_like(y) for _ in range(20)]
    torch.cuda.synchronize()
    for i in range(20):
        with torch.cuda.stream(other):
            g.replay()
            got[i].copy_(out)
        t.cache.attend(y, t.batch, out=got2[i])
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in got) and all(torch.equal(o, want2) for o in got2)


def test_the_stream_that_the_context_leaves_may_be_gone(ctx, lq8_lib):
    import ctypes as C
    import torch
    s, x, want = decode(ctx, lq8_lib, 60, 4000, 6)
    home, rt = ctx.stream, torch.cuda.cudart()
    got = [torch.empty_like(want) for _ in range(8)]
    torch.cuda.synchronize()
    try:
        for i in range(0, 8, 2):
            h = C.c_void_p()
            assert int(rt.cudaStreamCreate(C.addressof(h))) == 0
            ctx.check(ctx.lib.lq_set_stream(ctx.h, h))
            s.cache.attend(x, s.batch, out=got[i])
            torch.cuda.synchronize()
            assert int(rt.cudaStreamDestroy(h.value)) == 0
            ctx.check(ctx.lib.lq_set_stream(ctx.h, home))
            s.cache.attend(x, s.batch, out=got[i + 1])
    finally:
        ctx.check(ctx.lib.lq_set_stream(ctx.h, home))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def test_more_streams_than_workspaces(ctx, lq8_lib):
    """Calls of two sizes in turn on seven streams, with no wait in between."""
    import torch
    a, b = decode(ctx, lq8_lib, 60, 4000, 7), decode(ctx, lq8_lib, 150, 5000, 8)
    streams, home = [torch.cuda.Stream() for _ in range(7)], ctx.stream
    assert len({t.cuda_stream for t in streams}) == 7
    got = [(torch.empty_like(a[2]), torch.empty_like(b[2])) for _ in range(21)]
    torch.cuda.synchronize()
    try:
        for i, (ga, gb) in enumerate(got):
            ctx.check(ctx.lib.lq_set_stream(ctx.h, streams[i * 3 % 7].cuda_stream))
            for (s, x, _), g in ((a, ga), (b, gb)) if i % 2 else ((b, gb), (a, ga)):
                s.cache.attend(x, s.batch, out=g)
    finally:
        ctx.check(ctx.lib.lq_set_stream(ctx.h, home))
    torch.cuda.synchronize()
    assert all(torch.equal(ga, a[2]) and torch.equal(gb, b[2]) for ga, gb in got)


# ------------------------------------------------------------------------------------------
# padding
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D,rot", [(64, 64), (128, 128), (256, 256), (128, 64), (80, 80)])
@pytest.mark.parametrize("axes", [1, 3])
def test_positions_of_padding_rows_are_not_looked_at(ctx, lq8_lib, D, rot, axes):
    """A batch of fixed size: what stands in the padding's positions is no error; a live row's is."""
    import torch
    n = rot // 2
    rotary = lq8_lib.Rotary.build(n, 100, 1e4, lq8_lib.Rotary.cyclic([n - 2 * (n // 4), n // 4, n // 4]) if axes == 3 else None)
    qkv = randn(1, 9, 3 * D)

    def run(pos):
        s = Setup(lq8_lib, ctx, "f32", [3, 5], [1, 2], 1, D, 8, garbage=False)
        out = torch.full((9, 1, D), 9.0, device="cuda")
        s.cache.append(qkv, 1, s.batch, rotary, pos=i32(pos), q_out=out)
        return s, out

    pos = np.random.default_rng(1).integers(0, 100, (axes, 9))
    want, out = run(pos)
    ctx.device_status()
    pos[:, 3:] = [100, -1, 2 ** 31 - 1, -2 ** 31, 12345, 7]
    got, out2 = run(pos)
    ctx.device_status()
    assert torch.equal(out, out2) and (out2[3:] == 9.0).all() and torch.equal(want.k, got.k) and torch.equal(want.v, got.v)
    pos[axes - 1, 1] = 100
    run(pos)
    with pytest.raises(lq8_lib.LQ8Error, match="code 90, value 100"):
        ctx.device_status()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("q,pad,prefix", [([1, 2, 1], 1, 1000), ([1] * 40, 200, 3000), ([1, 3, 0, 60], 500, 500), ([300, 200], 70, 900),
                                          ([200] + [1] * 30, 300, 2000)])
def test_what_padding_rows_hold_has_no_effect(ctx, lq8_lib, dtype, q, pad, prefix):
    """Finite values, NaN or infinities in the padding: the other rows' bits are the same, and its own
    outputs are left alone."""
    import torch
    s = Setup(lq8_lib, ctx, dtype, [n + 20 + 3 * (b % 50) for b, n in enumerate(q)], q, 2, 128, 16, prefix, seed=5).fill()
    s.batch = lq8_lib.PagedBatch(s.batch.page_table, s.batch.kv_len, q_start=i32(s.start), max_q=max(q), max_kv=int(s.kv.max()),
                                 prefix_table=s.batch.prefix_table, prefix_len=prefix)
    x = torch.cat([randn(5, s.rows, 8, 128, dtype=dtype), randn(6, pad, 8, 128, dtype=dtype, scale=30.0)])
    outs = []
    for fill in (None, 0.0, float("nan"), float("inf")):
        if fill is not None:
            x[s.rows:] = fill
        out = torch.full_like(x, 9.0)
        s.cache.attend(x, s.batch, out=out)
        ctx.device_status()
        assert (out[s.rows:] == 9.0).all() and torch.isfinite(out).all()
        outs.append(out)
    assert all(torch.equal(o, outs[0]) for o in outs)


# ------------------------------------------------------------------------------------------
# refusals
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_q8_rows_that_are_not_aligned_are_refused(ctx, lq8_lib, dtype):
    import torch
    s = Setup(lq8_lib, ctx, dtype, [30, 2], [1, 1], 2, 64, 16, 0, garbage=False).fill()
    x = randn(1, 2, 4, 64, dtype=dtype)
    q, d = torch.zeros(2 * 256 + 8, dtype=torch.int8, device="cuda"), torch.zeros(2 * 8, dtype=torch.int16, device="cuda")
    with pytest.raises(lq8_lib.LQ8Error, match="multiples of 16 bytes"):
        s.cache.attend(x, s.batch, quantized=(q[8:].view(2, 256), d.view(2, 8)))
    with pytest.raises(lq8_lib.LQ8Error, match="multiples of 16 bytes"):
        ctx.call("lq_prefix_attention", x.data_ptr(), s.cache.dtype, 0, 2, 4, 2, 64, 0.125, *s.cache._pages, s.n_pages, 16, 0,
                 None, 0, *s.batch._seqs, 1, 30, None, 0, q.data_ptr(), d.data_ptr() + 1)
    ctx.device_status()


def test_q8_rows_on_the_host_are_refused(ctx, lq8_lib):
    import torch
    s = Setup(lq8_lib, ctx, "bf16", [30, 2], [1, 1], 2, 64, 16, 0, garbage=False).fill()
    x = randn(1, 2, 4, 64, dtype="bf16")
    q, d = torch.zeros(2, 256, dtype=torch.int8), torch.zeros(2, 8, dtype=torch.int16)
    for pair in ((q, d), (q.cuda(), d), (q, d.cuda())):
        with pytest.raises(ValueError, match="on the GPU"):
            s.cache.attend(x, s.batch, quantized=pair)


def test_a_prefix_longer_than_its_page_table_is_refused(ctx, lq8_lib):
    import torch
    s = Setup(lq8_lib, ctx, "bf16", [30, 2], [1, 1], 2, 64, 16, 33, garbage=False).fill()
    x = randn(1, 2, 4, 64, dtype="bf16")
    want = s.cache.attend(x, s.batch)
    part = dict(prefix_table=s.batch.prefix_table[:2])
    bad = lq8_lib.PagedBatch(s.batch.page_table, s.batch.kv_len, prefix_len=33, **part)
    with pytest.raises(ValueError, match="33 prefix positions"):
        s.cache.attend(x, bad)
    good = lq8_lib.PagedBatch(s.batch.page_table, s.batch.kv_len, prefix_len=32, **part)
    assert not torch.equal(s.cache.attend(x, good), want)
    good.prefix_len = 48
    with pytest.raises(ValueError, match="48 prefix positions"):
        s.cache.attend(x, good)
    ctx.device_status()


def test_pointers_that_are_not_aligned_to_their_elements_are_refused(ctx, lq8_lib):
    """Every device pointer of the three entries, one byte past where it belongs."""
    import torch
    z = torch.zeros(1 << 16, device="cuda")
    p = z.data_ptr()

    def refused(name, args, pointers):
        for i in pointers:
            bad = list(args)
            bad[i] = p + 1
            with pytest.raises(lq8_lib.LQ8Error, match="aligned|multiples of 16 bytes"):
                ctx.call(name, *bad)

    # x, dtype, rows, heads, dim, strides, out, strides, rot, cos, sin, len, axes of pairs, axes, pos, stride, inverse
    refused("lq_mrope", (p, 1, 2, 2, 64, 128, 64, p, 128, 64, 64, p, p, 4, None, 1, p, 2, 0), (0, 7, 11, 12, 16))
    # qkv, dtype, stride, rows, heads, kv heads, dim, norms, eps, bf16, rot, cos, sin, len, axes of pairs, axes, pos, stride, base,
    # sequences, starts, lengths, pages, ld, k, v, dtype, pages, size, stride, q out, stride
    refused("lq_paged_append", (p, 1, 0, 2, 2, 1, 64, p, p, 1e-6, 0, 64, p, p, 4, None, 1, p, 2, 0, 2, p, p, p, 1, p, p, 1, 4, 8, 0, p, 0),
            (0, 7, 8, 12, 13, 17, 21, 22, 23, 25, 26, 31))
    # q, dtype, stride, rows, heads, kv heads, dim, scale, k, v, pages, size, stride, prefix, length, sequences, starts, lengths,
    # pages, ld, most rows, most positions, out, stride, xq, xd
    refused("lq_prefix_attention", (p, 1, 0, 2, 2, 1, 64, 1.0, p, p, 4, 8, 0, p, 8, 2, p, p, p, 1, 1, 8, p, 0, p, p),
            (0, 8, 9, 13, 16, 17, 18, 22, 24, 25))
    ctx.device_status()


def test_mrope_refuses_rows_and_heads_of_the_output_that_overlap(ctx, lq8_lib):
    import torch
    rot = lq8_lib.Rotary.build(32, 100, 1e4)
    x, pos = randn(1, 5, 3, 64), i32(np.arange(5))
    want = lq8_lib.mrope(ctx, x, rot, pos)
    buf = torch.full((8192,), 9.0, device="cuda")
    for row, head in [(64, 64), (64, 128), (128, 64), (191, 64), (64, 319), (0, 64), (64, 0), (32, 1000), (1000, 32)]:
        with pytest.raises(lq8_lib.LQ8Error, match="overlap"):
            lq8_lib.mrope(ctx, x, rot, pos, out=torch.as_strided(buf, (5, 3, 64), (row, head, 1)))
    assert (buf == 9.0).all()
    for row, head in [(192, 64), (64, 320), (200, 64), (65, 330), (256, 66), (400, 130)]:
        assert torch.equal(lq8_lib.mrope(ctx, x, rot, pos, out=torch.as_strided(buf, (5, 3, 64), (row, head, 1))), want)
    one = torch.as_strided(buf, (1, 3, 64), (0, 64, 1))
    assert torch.equal(lq8_lib.mrope(ctx, x[:1], rot, pos[:1], out=one), want[:1])
    one = torch.as_strided(buf, (5, 1, 64), (64, 0, 1))
    assert torch.equal(lq8_lib.mrope(ctx, x[:, :1], rot, pos, out=one), want[:, :1])
    ctx.device_status()


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("prefix", [0, 300])
@pytest.mark.parametrize("starts", [[0, 4, 2, 6], [0, 6, 0, 6], [0, 3, 6, 5]])
def test_row_starts_that_fall_are_reported(ctx, lq8_lib, dtype, prefix, starts):
    """Such a batch names rows several times, and with many sequences more work than a launch can
    number: nothing of it is computed."""
    import torch
    s = Setup(lq8_lib, ctx, dtype, [30, 50, 70], [2, 2, 2], 2, 128, 16, prefix, seed=6, garbage=False).fill()
    s.batch.max_q = 6  # (the bounds of a call shape its sums: the same ones throughout)
    x = randn(1, 6, 8, 128, dtype=dtype)
    want = s.cache.attend(x, s.batch).clone()
    s.batch.q_start.copy_(i32(starts))
    s.cache.attend(x, s.batch)
    with pytest.raises(lq8_lib.LQ8Error, match="code 93"):
        ctx.device_status()
    s.batch.q_start.copy_(i32([0, 2, 4, 6]))
    assert torch.equal(s.cache.attend(x, s.batch), want)
    ctx.device_status()
