"""GPU tests of the operators on a paged cache in 8 bits in a server's conditions: a run of them together,
captured graphs and streams next to other calls, waits that run out, padding, large caches, and calls
that are refused. Definitions and tolerances are those of test_gpu_paged_q8.py."""
import os
import sys

import numpy as np
import pytest

from test_gpu_paged import i32, randn, within
from test_gpu_paged_q8 import Cache, attention64, attention_case, tolerance

pytestmark = pytest.mark.gpu

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


# ------------------------------------------------------------------------------------------
# together
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D,block,Hq,Hkv", [(128, 32, 8, 2), (64, 16, 5, 1)])
def test_prompts_then_decode_steps(ctx, lq8_lib, D, block, Hq, Hkv):
    """A shared prompt, ragged questions behind it, then decode steps of a growing batch: each call's
    attention against the definition on what `read` gives of the cache at that time."""
    import torch
    page, prefix = 32, 75
    c = lq8_lib.PagedKvCacheQ8.empty(ctx, 40, page, Hkv, D, block)
    rotary = lq8_lib.Rotary.build(D // 2, 400, 1e4)
    qn, kn = ((1 + 0.2 * randn(i, D)).to(torch.bfloat16) for i in (1, 2))
    ids = np.random.default_rng(1).permutation(40)
    ptable, table = i32(ids[:3]), i32(ids[3:3 + 3 * 5].reshape(3, 5))
    rows = lambda n, seed: randn(seed, n, (Hq + 2 * Hkv) * D, scale=1.5, dtype="bf16")  # noqa: E731
    first = lq8_lib.PagedBatch(ptable[None].contiguous(), i32([prefix]), q_start=i32([0, prefix]), max_q=prefix, max_kv=prefix)
    c.append(rows(prefix, 3), Hq, first, rotary, q_norm=qn, k_norm=kn)
    pk, pv = c.read(first, rows=prefix, dtype=torch.float32)
    kv = np.array([0, 0, 0])
    for step, q in enumerate([[40, 1, 17], [1, 1, 1], [1, 1, 1], [3, 0, 2], [1, 1, 1]] + [[1, 1, 1]] * 12):
        q = np.array(q)
        kv = kv + q
        start, n = np.concatenate([[0], np.cumsum(q)]), int(q.sum())
        b = lq8_lib.PagedBatch(table, i32(kv), q_start=i32(start) if step != 1 else None, max_q=int(q.max()), max_kv=150,
                               prefix_table=ptable, prefix_len=prefix)
        x = c.append(rows(n, 10 + step), Hq, b, rotary, q_norm=qn, k_norm=kn)
        got = c.attend(x, b)
        whole = lq8_lib.PagedBatch(table, i32(kv), q_start=i32(np.concatenate([[0], np.cumsum(kv)])), max_q=int(kv.max()))
        k, v = c.read(whole, rows=int(kv.sum()), dtype=torch.float32)
        ctx.device_status()
        G, at = Hq // Hkv, np.concatenate([[0], np.cumsum(kv)])
        for s in range(3):
            if not q[s]:
                continue
            keys, vals = (torch.cat([p, o[at[s]:at[s + 1]]]).double().transpose(0, 1) for p, o in ((pk, k), (pv, v)))
            y = x[start[s]:start[s + 1]].double().view(-1, Hkv, G, D).permute(1, 2, 0, 3)
            score = torch.einsum("hgnd,htd->hgnt", y, keys) * D ** -0.5
            t = torch.arange(keys.shape[1], device="cuda")
            score.masked_fill_(t[None] > prefix + int(kv[s] - q[s]) + torch.arange(int(q[s]), device="cuda")[:, None], -float("inf"))
            p = torch.softmax(score, -1)
            o, a = (torch.einsum("hgnt,htd->nhgd", p, w).reshape(int(q[s]), Hq, D) for w in (vals, vals.abs()))
            # the streaming kernel's bounds hold with w <= 128 127 max |v| / 127 a tile, three tiles at most; the other's too
            d = (y.abs().amax(-1) / 65024 * D ** -0.5 * keys.abs().sum(-1).amax(-1)[:, None, None]).permute(2, 0, 1).reshape(int(q[s]), Hq, 1)
            tol = 2.0 ** -8 * o.abs() + (torch.expm1(2 * d) + 2.0 ** -8 + 2e-5) * a + 3 * 128 * float(vals.abs().max()) / 65024
            within(got[start[s]:start[s + 1]], o, tol)


@pytest.mark.parametrize("image", [True, False])
def test_shared_prompt_serving(ctx, lq8_lib, image):
    """The serving example on an 8-bit cache. k and v are off by up to 1/254 of their block's largest
    value, which is about four times a typical one: where a bf16 cache is held to 2e-2 for each of the
    two layers (2^-8 of each value), four times that."""
    import torch
    import shared_prefix_serving as ex
    got, want, _ = ex.serve(torch.int8, image, ctx=ctx)
    assert got.shape == want.shape == (7, 3, 1000) and torch.isfinite(got).all()
    assert float((got - want).abs().max()) <= 1.6e-1 * float(want.abs().max())


# ------------------------------------------------------------------------------------------
# batches
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv,Hq,Hkv,D,prefix", [
    ([4000 * (512 - i) // 512 or 1 for i in range(512)], 8, 8, 64, 0),
    ([32768] * 5 + [100] * 25, 16, 2, 128, 0),
    ([1] * 1500, 4, 1, 64, 0),
    ([8192] * 20 + [100] * 40, 8, 2, 128, 300)])
def test_attention_of_ragged_decode_batches(ctx, lq8_lib, kv, Hq, Hkv, D, prefix):
    attention_case(ctx, lq8_lib, kv, [1] * len(kv), Hq, Hkv, D, 128, 64, prefix)


def test_attention_of_prompts_next_to_decode_rows(ctx, lq8_lib):
    attention_case(ctx, lq8_lib, [700, 40, 900, 3, 1200, 64], [300, 1, 1, 3, 1, 64], 8, 2, 128, 64, 32, 0)
    attention_case(ctx, lq8_lib, [700, 40, 900, 3, 1200, 64], [300, 1, 1, 3, 1, 64], 8, 2, 64, 64, 32, 500)


def test_a_cache_past_32_bits(ctx, lq8_lib):
    """Codes and scales more than 2^31 elements apart: pages at both ends of 2.4 billion codes."""
    import torch
    Hkv, page, D, block = 8, 256, 128, 16
    n_pages = (2400 << 20) // (Hkv * page * D)
    c = lq8_lib.PagedKvCacheQ8.empty(ctx, n_pages, page, Hkv, D, block)
    table = i32([[n_pages - 1, 0, n_pages // 2], [n_pages - 2, 1, n_pages - 3]])
    kv, rows = [700, 520], 1220
    b = lq8_lib.PagedBatch(table, i32(kv), q_start=i32([0, 700, 1220]), max_q=700, max_kv=700)
    rotary = lq8_lib.Rotary.build(D // 2, 800, 1e4)
    qkv = randn(5, rows, (16 + 2 * Hkv) * D, dtype="bf16")
    q = c.append(qkv, 16, b, rotary)
    k, v = c.read(b, rows=rows, dtype=torch.float32)
    small = lq8_lib.PagedKvCacheQ8.empty(ctx, 6, page, Hkv, D, block)
    b2 = lq8_lib.PagedBatch(i32([[3, 0, 5], [1, 4, 2]]), i32(kv), q_start=i32([0, 700, 1220]), max_q=700, max_kv=700)
    assert torch.equal(small.append(qkv, 16, b2, rotary), q)
    k2, v2 = small.read(b2, rows=rows, dtype=torch.float32)
    assert torch.equal(k, k2) and torch.equal(v, v2)
    for lo, hi, max_q in ((0, 1220, 700), (699, 701, 1)):
        n = hi - lo
        starts = [0, 700, 1220] if n > 2 else [0, 1, 2]
        lengths = kv if n > 2 else [700, 1]
        args = dict(q_start=i32(starts), max_q=max_q, max_kv=700)
        x = q[lo:hi].contiguous()
        assert torch.equal(c.attend(x, lq8_lib.PagedBatch(table, i32(lengths), **args)),
                           small.attend(x, lq8_lib.PagedBatch(i32([[3, 0, 5], [1, 4, 2]]), i32(lengths), **args)))
    ctx.device_status()


# ------------------------------------------------------------------------------------------
# waits that run out
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("kv,q,prefix,page,D,codes", [
    ([40 + 7 * (b % 90) for b in range(300)], [1] * 300, 0, 16, 128, (97,)),       # streaming alone
    ([40 + 7 * (b % 90) for b in range(300)], [1] * 300, 0, 16, 64, (97,)),
    ([40 + 7 * (b % 90) for b in range(300)], [1] * 300, 2000, 64, 128, (94, 97)),  # the prefix apart
    ([300, 500, 40] * 6, [200, 300, 3] * 6, 1000, 32, 128, (94,)),                 # prompt chunks
])
def test_attention_whose_waits_run_out(ctx, lq8_lib, monkeypatch, kv, q, prefix, page, D, codes):
    """LQ_FAULT=prefix_attn_wait: the waits inside the kernels give up early. The call ends, the error is
    reported, and the next call is right."""
    import torch
    s = Cache(lq8_lib, ctx, kv, q, 2, D, page, 16, prefix=prefix, seed=3).fill()
    x = randn(3, s.rows, 8, D, dtype="bf16")
    want = s.cache.attend(x, s.batch)
    ctx.device_status()
    for _ in range(3):
        monkeypatch.setenv("LQ_FAULT", "prefix_attn_wait")
        s.cache.attend(x, s.batch)
        monkeypatch.delenv("LQ_FAULT")
        with pytest.raises(lq8_lib.LQ8Error) as e:
            ctx.device_status()
        assert any(f"code {c}" in str(e.value) for c in codes)
        assert torch.equal(s.cache.attend(x, s.batch), want)
        ctx.device_status()


# ------------------------------------------------------------------------------------------
# graphs and streams
# ------------------------------------------------------------------------------------------

def decode(ctx, lq8_lib, seqs, prefix, seed):
    """A decode batch: cache, q and the result of a plain call."""
    s = Cache(lq8_lib, ctx, [40 + 13 * b for b in range(seqs)], [1] * seqs, 2, 128, 16, 16, prefix=prefix, seed=seed).fill()
    x = randn(seed, seqs, 8, 128, dtype="bf16")
    return s, x, s.cache.attend(x, s.batch).clone()


def test_a_captured_step_advances_on_the_device(ctx, lq8_lib):
    """Append and attention captured once and replayed while the lengths grow, against eager calls."""
    import torch
    Hq, Hkv, D, B, steps = 4, 2, 128, 5, 40
    rotary = lq8_lib.Rotary.build(D // 2, 200, 1e4)
    qkv = randn(7, steps, B, (Hq + 2 * Hkv) * D)
    table = i32(np.random.default_rng(2).permutation(B * 4).reshape(B, 4))

    def make():
        return lq8_lib.PagedKvCacheQ8.empty(ctx, B * 4, 16, Hkv, D), i32(np.zeros(B))

    want = []
    c, kv = make()
    batch = lq8_lib.PagedBatch(table, kv, max_kv=64)
    for i in range(steps):
        kv.add_(1)
        torch.cuda.synchronize()
        want.append(c.attend(c.append(qkv[i], Hq, batch, rotary), batch).clone())
    torch.cuda.synchronize()
    c, kv = make()
    batch = lq8_lib.PagedBatch(table, kv, max_kv=64)
    x, q, out = torch.empty_like(qkv[0]), torch.empty(B, Hq, D, dtype=torch.bfloat16, device="cuda"), torch.empty(B, Hq, D, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=ctx._torch_stream):
        kv.add_(1)
        c.append(x, Hq, batch, rotary, q_out=q)
        c.attend(q, batch, out=out)
    for i in range(steps):
        x.copy_(qkv[i])
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    ctx.device_status()
    del g


@pytest.mark.parametrize("prefix", [0, 900])
def test_a_capture_may_be_the_first_call_and_outlives_larger_ones(ctx, lq8_lib, prefix):
    import torch
    s, x, want = decode(ctx, lq8_lib, 70, prefix, 3)
    c = lq8_lib.Context(0)
    cache = lq8_lib.PagedKvCacheQ8(c, s.k, s.v, s.ks, s.vs)
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=c._torch_stream):
        cache.attend(x, s.batch, out=out)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    big, y, _ = decode(c, lq8_lib, 300, 3000, 4)  # more workspace, by eager calls
    taken = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(64)]
    for _ in range(3):
        out.zero_()
        g.replay()
        big.cache.attend(y, big.batch)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    assert all(bool((t == 7).all()) for t in taken)
    del g
    c.close()


def test_replays_next_to_eager_calls_on_another_stream(ctx, lq8_lib):
    import torch
    s, x, want = decode(ctx, lq8_lib, 60, 4000, 4)
    t, y, want2 = decode(ctx, lq8_lib, 90, 0, 5)
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=ctx._torch_stream):
        s.cache.attend(x, s.batch, out=out)
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
    del g


def test_calls_of_all_caches_in_turn_on_several_streams(ctx, lq8_lib):
    """8-bit and bf16 calls of several sizes share a stream's workspace; seven streams, no wait in between."""
    import torch
    from test_gpu_paged_serving import decode as decode_bf16
    jobs = [decode(ctx, lq8_lib, 60, 4000, 7), decode_bf16(ctx, lq8_lib, 150, 5000, 8), decode(ctx, lq8_lib, 150, 0, 9), decode(ctx, lq8_lib, 7, 20, 10)]
    streams, home = [torch.cuda.Stream() for _ in range(7)], ctx.stream
    got = [[torch.empty_like(w) for _, _, w in jobs] for _ in range(21)]
    torch.cuda.synchronize()
    try:
        for i, outs in enumerate(got):
            ctx.check(ctx.lib.lq_set_stream(ctx.h, streams[i * 3 % 7].cuda_stream))
            for k in np.random.default_rng(i).permutation(len(jobs)):
                s, x, _ = jobs[k]
                s.cache.attend(x, s.batch, out=outs[k])
    finally:
        ctx.check(ctx.lib.lq_set_stream(ctx.h, home))
    torch.cuda.synchronize()
    for outs in got:
        assert all(torch.equal(o, w) for o, (_, _, w) in zip(outs, jobs))


# ------------------------------------------------------------------------------------------
# padding, bad inputs, refusals
# ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D,rot", [(64, 64), (128, 128), (128, 64)])
@pytest.mark.parametrize("axes", [1, 3])
def test_positions_of_padding_rows_are_not_looked_at(ctx, lq8_lib, D, rot, axes):
    import torch
    n = rot // 2
    rotary = lq8_lib.Rotary.build(n, 100, 1e4, lq8_lib.Rotary.cyclic([n - 2 * (n // 4), n // 4, n // 4]) if axes == 3 else None)
    qkv = randn(1, 9, 3 * D)

    def run(pos):
        s = Cache(lq8_lib, ctx, [3, 5], [1, 2], 1, D, 16, 16)
        out = torch.full((9, 1, D), 9.0, device="cuda", dtype=torch.bfloat16)
        s.cache.append(qkv, 1, s.batch, rotary, pos=i32(pos), q_out=out)
        return s, out

    pos = np.random.default_rng(1).integers(0, 100, (axes, 9))
    want, out = run(pos)
    ctx.device_status()
    bad = pos.copy()
    bad[:, 3:] = [[-5, 100, 2 ** 31 - 1, -2 ** 31, 7, 101]] * axes
    got, out2 = run(bad)
    ctx.device_status()
    assert torch.equal(out, out2) and (out[3:] == 9.0).all()
    assert torch.equal(want.k, got.k) and torch.equal(want.v, got.v)


@pytest.mark.parametrize("q,pad,prefix", [([1] * 40, 0, 0), ([3, 60, 0, 1], 200, 0), ([3, 60, 0, 1], 200, 130), ([1, 2, 1], 90, 70)])
def test_what_padding_rows_hold_has_no_effect(ctx, lq8_lib, q, pad, prefix):
    import torch
    s = Cache(lq8_lib, ctx, [70 + 9 * b for b in range(len(q))], q, 2, 128, 16, 16, prefix=prefix, seed=5).fill()
    if pad and s.batch.q_start is None:
        pytest.skip("no padding without row starts")
    n = s.rows + pad
    x = randn(6, n, 8, 128, dtype="bf16")
    outs = []
    for fill in (0.0, float("nan"), float("inf")):
        y = x.clone()
        y[s.rows:] = fill
        out = torch.full_like(y, 3.0)
        s.cache.attend(y, s.batch, out=out)
        outs.append(out)
        assert (out[s.rows:] == 3.0).all()
    ctx.device_status()
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_nan_and_infinity_in_q_and_scales_reach_their_rows_alone(ctx, lq8_lib):
    import torch
    for rows in ([1] * 6, [50, 1, 1, 1, 1, 1]):
        s = Cache(lq8_lib, ctx, [100, 90, 80, 300, 64, 33], rows, 2, 128, 16, 16, seed=8).fill()
        x = randn(9, s.rows, 4, 128, dtype="bf16")
        want = s.cache.attend(x, s.batch)
        y = x.clone()
        at = int(s.start[1])
        y[at, 1, 5] = float("nan")
        y[at, 2] = 0.0
        s.ks[int(s.table[3, 2]), 1, 0] = float("nan")   # positions 32 to 47 of sequence 3, kv head 1: heads 2 and 3
        s.vs[int(s.table[4, 1]), 0, 0] = float("nan")   # positions 16 to 31 of sequence 4, kv head 0: heads 0 and 1
        got = s.cache.attend(y, s.batch)
        ctx.device_status()
        bad = torch.zeros(s.rows, 4, dtype=torch.bool, device="cuda")
        bad[at, 1] = bad[int(s.start[3]), 2:] = bad[int(s.start[4]), :2] = True
        assert got[bad].isnan().all() and torch.isfinite(got[~bad]).all()
        bad[at, 2] = True
        assert torch.equal(got[~bad], want[~bad])


@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("D", [64, 128])
def test_zero_scales(ctx, lq8_lib, rows, D):
    """Blocks whose values are all zero: their positions count with a score of zero, and give nothing. Codes
    that are not zero under a scale of zero: V's scale counts as 2^-80, and a mean of codes is at most 128."""
    import torch
    s = Cache(lq8_lib, ctx, [200, 90], [rows, 1], 1, D, 16, 16, seed=21).fill()
    for b, page in ((0, 1), (0, 12), (1, 0), (1, 5)):
        s.ks[int(s.table[b, page])] = 0.0
        s.vs[int(s.table[b, page])] = 0.0
        s.k[int(s.table[b, page])] = 0
        s.v[int(s.table[b, page])] = 0
    x = randn(22, s.rows, 4, D, scale=1.5, dtype="bf16")
    want = attention64(s, x, D ** -0.5)
    within(s.cache.attend(x, s.batch), want[0], tolerance(want, streaming=False) + tolerance(want))
    s.ks.zero_(), s.vs.zero_()
    assert float(s.cache.attend(x, s.batch).abs().max()) <= 128 * 2.0 ** -80
    s.k.zero_(), s.v.zero_()
    assert not s.cache.attend(x, s.batch).any()
    ctx.device_status()


@pytest.mark.parametrize("rows", [1, 70])
@pytest.mark.parametrize("lo,hi", [(-75, -68), (-126, -80), (10, 18), (-80, 18)])
def test_scales_of_v_of_any_size(ctx, lq8_lib, rows, lo, hi):
    """Scales from 2^lo to 2^hi. Below 2^-80 they count as that, by definition: then the result is within 128
    2^-80 of the one with the scales as they are (a mean of codes times a difference below 2^-80), and
    the roundings are those of the values that count, which is why the definition is evaluated with these (with the
    scales as they are and 127 2^-80 for all else, the rounding of a value of 127 2^-80 has no room)."""
    s = Cache(lq8_lib, ctx, [900, 90], [rows, 1], 1, 128, 32, 16, prefix=100, seed=23).fill()
    s.vs.copy_(2.0 ** (lo + (hi - lo) * abs(randn(24, *s.vs.shape).sin())))
    x = randn(25, s.rows, 8, 128, dtype="bf16")
    got = s.cache.attend(x, s.batch)
    plain = attention64(s, x, 128 ** -0.5)[0]
    s.vs.clamp_(min=2.0 ** -80)
    want = attention64(s, x, 128 ** -0.5)
    assert float((want[0] - plain).abs().max()) <= 128 * 2.0 ** -80
    within(got, want[0], tolerance(want, streaming=False) + tolerance(want))
    ctx.device_status()


@pytest.mark.parametrize("rows", [1, 60])
@pytest.mark.parametrize("prefix", [0, 100])
def test_bad_lengths_and_pages_are_reported(ctx, lq8_lib, rows, prefix):
    import torch
    for code, field, at, value in [(92, "page_table", 1, 10 ** 6), (92, "page_table", 0, -1), (91, "kv_len", 0, 5000), (91, "kv_len", 0, -3),
                                   (92, "prefix_table", 1, 10 ** 6), (93, "q_start", 2, 1000)]:
        s = Cache(lq8_lib, ctx, [70, 200], [rows, 2], 2, 128, 32, 16, prefix=prefix, seed=2).fill()
        if getattr(s.batch, field) is None:
            continue
        x = randn(2, s.rows, 4, 128, dtype="bf16")
        getattr(s.batch, field).view(-1)[at] = value
        s.cache.attend(x, s.batch)
        with pytest.raises(lq8_lib.LQ8Error) as e:
            ctx.device_status()
        assert f"code {code}" in str(e.value)
        ctx.device_status()


@pytest.mark.parametrize("prefix,starts", [(0, [0, 1, 0, 2]), (40, [0, 30, 2, 33])])
def test_row_starts_that_fall_compute_nothing(ctx, lq8_lib, prefix, starts):
    import torch
    s = Cache(lq8_lib, ctx, [70, 200, 64], [1, 1, 31] if prefix else [1, 1, 1], 2, 128, 32, 16, prefix=prefix, seed=2).fill()
    b = lq8_lib.PagedBatch(s.batch.page_table, s.batch.kv_len, q_start=i32(starts), max_q=40, max_kv=200, prefix_table=s.batch.prefix_table,
                           prefix_len=prefix)
    x = randn(2, 40, 4, 128, dtype="bf16")
    s.cache.attend(x, b)
    with pytest.raises(lq8_lib.LQ8Error):
        ctx.device_status()
    ctx.device_status()


def test_refusals(ctx, lq8_lib):
    import torch
    Q = lq8_lib.PagedKvCacheQ8
    c = Q.empty(ctx, 4, 32, 2, 64, 16)
    codes = lambda *shape: torch.zeros(shape, dtype=torch.int8, device="cuda")  # noqa: E731
    scales = lambda *shape: torch.zeros(shape, device="cuda")  # noqa: E731
    ok = (codes(4, 2, 32, 64), codes(4, 2, 32, 64), scales(4, 2, 2), scales(4, 2, 2))
    Q(ctx, *ok)
    for i, bad in [(0, codes(4, 2, 32, 128)), (0, ok[0].float()), (0, ok[0].cpu()), (1, ok[1].transpose(1, 2).contiguous().transpose(1, 2)),
                   (2, scales(4, 2, 3)), (2, scales(4, 1, 2)), (2, scales(4, 2, 0)), (2, ok[2].double()), (3, scales(8, 2, 2)[::2]), (3, ok[3].cpu())]:
        with pytest.raises(ValueError):
            Q(ctx, *(bad if j == i else t for j, t in enumerate(ok)))
    table, kv = i32([[0, 1], [2, 3]]), i32([40, 20])
    b = lq8_lib.PagedBatch(table, kv)
    rot = lq8_lib.Rotary.build(32, 100, 1e4)
    qkv, q = randn(1, 2, 6 * 64, dtype="bf16"), randn(2, 2, 2, 64, dtype="bf16")
    for call in (lambda: c.append(qkv[:, :-64], 2, b, rot), lambda: c.append(qkv.to(torch.float16), 2, b, rot),
                 lambda: c.append(qkv, 2, b, rot, q_out=torch.empty(2, 2, 64, device="cuda")),
                 lambda: c.attend(q.float(), b), lambda: c.attend(q, b, out=torch.empty(2, 2, 64, device="cuda")), lambda: c.attend(q[:, :, :32], b),
                 lambda: c.read(b, torch.empty(2, 2, 64, device="cuda")), lambda: c.read(b, torch.empty(2, 2, 32, device="cuda"), torch.empty(2, 2, 32, device="cuda")),
                 lambda: c.read(lq8_lib.PagedBatch(table, kv, q_start=i32([0, 1, 2]))), lambda: c.read(b, dtype=torch.float16),
                 lambda: c.read(b, q[:, :2], q[:, :2], rows=3)):
        with pytest.raises(ValueError):
            call()
    # the C boundary: block, page size, head dimension, alignment, strides, rows without starts, NULL
    lib, h, I = ctx.lib, ctx.h, lq8_lib
    k, v, ks, vs = (t.data_ptr() for t in ok)
    out = torch.zeros(4, 2, 64, device="cuda")

    def read(k=k, ks=ks, heads=2, D=64, n_pages=4, page=32, stride=0, block=16, sstride=0, rows=2, o=out.data_ptr(), dt=I.DTYPE_F32, ostride=0):
        return lib.lq_paged_read_q8(h, k, v, ks, vs, heads, D, n_pages, page, stride, block, sstride, 2, None, kv.data_ptr(), table.data_ptr(), 2,
                                    rows, o, o, dt, ostride)

    assert read() == 0 and read(rows=0, k=None, ks=None) == 0
    for bad in (dict(block=8), dict(block=24), dict(block=64), dict(page=8, block=16), dict(page=48), dict(D=80), dict(D=32), dict(k=k + 8), dict(ks=ks + 2),
                dict(stride=32 * 64), dict(stride=2 * 32 * 64 + 8), dict(sstride=1), dict(k=None), dict(ks=None), dict(rows=3), dict(o=out.data_ptr() + 4),
                dict(o=None), dict(dt=I.DTYPE_F16), dict(ostride=64), dict(ostride=130), dict(heads=0), dict(n_pages=0)):
        assert read(**bad) == -1, bad
    x, y = randn(3, 2, 4, 64, dtype="bf16"), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")

    def attend(q=x.data_ptr(), heads=4, kvh=2, D=64, scale=0.1, block=16, k=k, max_q=1, max_kv=64, o=y.data_ptr(), qs=0, xq=None, xd=None, prefix=0):
        return lib.lq_prefix_attention_q8(h, q, qs, 2, heads, kvh, D, scale, k, v, ks, vs, 4, 32, 0, block, 0, None, prefix, 2, None, kv.data_ptr(),
                                          table.data_ptr(), 2, max_q, max_kv, o, 0, xq, xd)

    assert attend() == 0
    for bad in (dict(heads=3), dict(heads=0), dict(D=128 + 64), dict(scale=0.0), dict(scale=float("nan")), dict(block=33), dict(k=k + 4), dict(k=None),
                dict(max_q=0), dict(max_kv=-1), dict(o=None), dict(q=None), dict(q=x.data_ptr() + 2), dict(qs=100), dict(xq=y.data_ptr()), dict(prefix=5),
                dict(heads=512, kvh=2)):
        assert attend(**bad) == -1, bad
    ctx.device_status()
    assert lib.lq_prefix_attention_q8(None, *([0] * 4), 1, 64, 0.1, *([None] * 4), *([0] * 5), None, 0, 0, None, None, None, 0, 1, 0, None, 0, None, None) == -1
