"""Serving a batch that shares a prompt, on the paged operators.

A Qwen3 model's weights (lq8.Qwen3ForCausalLM) drive a decoder whose K/V cache is paged: the shared
prompt is computed once and kept in pages of its own, every sequence brings a question (a ragged
chunk of new rows) and then decodes, one row a sequence and step. Positions may have three axes
(time, height, width), for an image inside the prompt.

`contiguous_logits` runs the same tokens the other way, one sequence at a time on a contiguous
cache: the norm by lq_qk_norm_rope_kv without a rotation, the rotation by lq_mrope, attention by
lq_attention. Text-only prompts can also be held against the model runner itself.

    python examples/shared_prefix_serving.py            # a small random model, checks and timings
"""
import ctypes as C
import os
import sys
import time

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen-omni-inference-rs_b200"))
import lq8  # noqa: E402

PAGE = 16


def i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


class Weights:
    """The layer ops of a Qwen3 model over its own Q8_0 weights."""

    def __init__(self, ctx, model):
        self.ctx, self.model, self.cfg = ctx, model, model.cfg
        c = model.cfg
        self.qkv, self.o, self.gate_up, self.down = ([model.linear(i, k) for i in range(c.layers)]
                                                     for k in ("qkv", "o", "gate_up", "down"))
        self.lm_head = model.linear(-1, "lm_head")
        norm = lambda layer, kind: lq8.wrap_device(*[(p, (n,), "<i2") for p, n in [model.tensor(layer, kind)]][0])  # noqa: E731
        self.in_norm, self.post_norm, self.q_norm, self.k_norm = ([norm(i, k) for i in range(c.layers)]
                                                                  for k in ("in_norm", "post_norm", "q_norm", "k_norm"))
        self.final_norm, self.embed = norm(-1, "final_norm"), model.tensor(-1, "embed")[0]

    def embedding(self, ids):
        out = torch.empty((ids.numel(), self.cfg.hidden), device="cuda")
        self.ctx.call("lq_embedding", self.embed, self.cfg.vocab, self.cfg.hidden, ids.data_ptr(), ids.numel(), out.data_ptr())
        return out

    def norm(self, x, w):
        """RMSNorm to Q8_0 rows."""
        q = torch.empty(x.shape, dtype=torch.int8, device="cuda")
        d = torch.empty((x.shape[0], x.shape[1] // 32), dtype=torch.int16, device="cuda")
        self.ctx.call("lq_rmsnorm", x.data_ptr(), lq8.DTYPE_F32, x.shape[0], x.shape[1], w.data_ptr(), self.cfg.eps, None,
                      q.data_ptr(), d.data_ptr())
        return q, d

    def matmul(self, w, rows, residual=None):
        q, d = rows
        y = torch.empty((q.shape[0], w.n), device="cuda") if residual is None else residual
        self.ctx.call("lq_q8_0_matmul", C.byref(w), q.data_ptr(), d.data_ptr(), q.shape[0], y.data_ptr(),
                      None if residual is None else residual.data_ptr(), w.n)
        return y

    def mlp(self, x, layer):
        gu = self.matmul(self.gate_up[layer], self.norm(x, self.post_norm[layer]))
        m, inter = x.shape[0], self.cfg.inter
        q = torch.empty((m, inter), dtype=torch.int8, device="cuda")
        d = torch.empty((m, inter // 32), dtype=torch.int16, device="cuda")
        self.ctx.call("lq_silu_mul", gu.data_ptr(), m, inter, None, q.data_ptr(), d.data_ptr())
        self.matmul(self.down[layer], (q, d), x)

    def logits(self, x):
        return self.matmul(self.lm_head, self.norm(x, self.final_norm))

    def argmax(self, logits):
        out = torch.empty(logits.shape[0], dtype=torch.int32, device="cuda")
        self.ctx.call("lq_argmax", logits.data_ptr(), logits.shape[0], logits.shape[1], out.data_ptr())
        return out


class PagedDecoder:
    """A batch behind a shared prompt. cache_dtype float32 keeps the model runner's numerics
    (norm_bf16: its rounding points); bfloat16 halves the cache, int8 (codes, a scale for each page and kv
    head) halves it again."""

    def __init__(self, weights, rotary, n_pages, cache_dtype=torch.float32):
        self.w, self.rotary = weights, rotary
        c = weights.cfg
        # every layer's pages in one allocation, page by page: [2, pages, layers, kv heads, page, dim]
        buf = torch.zeros((2, n_pages, c.layers, c.n_kv_heads, PAGE, c.head_dim), dtype=cache_dtype, device="cuda")
        if cache_dtype == torch.int8:
            scales = torch.zeros((2, n_pages, c.layers, c.n_kv_heads, 1), device="cuda")
            self.caches = [lq8.PagedKvCacheQ8(weights.ctx, *(t[j][:, i] for t in (buf, scales) for j in (0, 1))) for i in range(c.layers)]
        else:
            self.caches = [lq8.PagedKvCache(weights.ctx, buf[0][:, i], buf[1][:, i]) for i in range(c.layers)]
        self.free = list(range(n_pages))[::-1]
        self.prefix_table, self.prefix_len = None, 0

    def rows(self, ids, batch, pos=None):
        """Runs new rows through the layers; hidden states [rows, hidden]."""
        w, c = self.w, self.w.cfg
        x = w.embedding(ids)
        m = x.shape[0]
        att = (torch.empty((m, c.n_heads * c.head_dim), dtype=torch.int8, device="cuda"),
               torch.empty((m, c.n_heads * c.head_dim // 32), dtype=torch.int16, device="cuda"))
        for i, cache in enumerate(self.caches):
            qkv = w.matmul(w.qkv[i], w.norm(x, w.in_norm[i]))
            q = cache.append(qkv, c.n_heads, batch, self.rotary, pos=pos, q_norm=w.q_norm[i], k_norm=w.k_norm[i],
                             eps=c.eps, norm_bf16=cache.k.dtype == torch.float32)
            cache.attend(q, batch, quantized=att)
            w.matmul(w.o[i], att, x)
            w.mlp(x, i)
        return x

    def share(self, ids, pos=None):
        """Computes the shared prompt once; its pages stay."""
        n = len(ids)
        pages = [self.free.pop() for _ in range(-(-n // PAGE))]
        batch = lq8.PagedBatch(i32([pages]), i32([n]), q_start=i32([0, n]), max_q=n, max_kv=n)
        self.rows(i32(ids), batch, pos)
        self.prefix_table, self.prefix_len = i32(pages), n

    def start(self, questions, max_new, pos=None):
        """Every sequence's own rows, ragged; logits of each one's last row."""
        lens = [len(q) for q in questions]
        own = [-(-(n + max_new) // PAGE) for n in lens]
        table = np.zeros((len(lens), max(own)), np.int32)
        for b, n in enumerate(own):
            table[b, :n] = [self.free.pop() for _ in range(n)]
        start = np.concatenate([[0], np.cumsum(lens)])
        self.table, self.kv_len = i32(table), i32(lens)
        shared = dict(prefix_table=self.prefix_table, prefix_len=self.prefix_len)
        first = lq8.PagedBatch(self.table, self.kv_len, q_start=i32(start), max_q=max(lens), max_kv=max(lens), **shared)
        self.batch = lq8.PagedBatch(self.table, self.kv_len, max_kv=max(lens) + max_new, **shared)  # one row a sequence
        x = self.rows(i32(np.concatenate(questions)), first, pos)
        return self.w.logits(x[torch.from_numpy(start[1:] - 1).cuda()].contiguous())

    def step(self, ids, pos=None):
        """One decode step; lengths advance on the device."""
        self.kv_len.add_(1)
        return self.w.logits(self.rows(ids, self.batch, pos))


def contiguous_logits(weights, rotary, ids, pos):
    """Logits of every row of one sequence on a contiguous f32 cache; pos [axes, rows]."""
    w, c, ctx = weights, weights.cfg, weights.ctx
    L, D, Hq, Hkv = len(ids), c.head_dim, c.n_heads, c.n_kv_heads
    one, zero = torch.ones((L, D // 2), device="cuda"), torch.zeros((L, D // 2), device="cuda")
    x = w.embedding(i32(ids))
    q, k, v = (torch.zeros((h, L, D), device="cuda") for h in (Hq, Hkv, Hkv))
    att = (torch.empty((L, Hq * D), dtype=torch.int8, device="cuda"), torch.empty((L, Hq * D // 32), dtype=torch.int16, device="cuda"))
    for i in range(c.layers):
        qkv = w.matmul(w.qkv[i], w.norm(x, w.in_norm[i]))
        ctx.call("lq_qk_norm_rope_kv", qkv.data_ptr(), 1, L, Hq, Hkv, D, w.q_norm[i].data_ptr(), w.k_norm[i].data_ptr(), c.eps,
                 one.data_ptr(), zero.data_ptr(), 0, None, q.data_ptr(), k.data_ptr(), v.data_ptr(), L)
        for t in (q, k):  # [heads, rows, dim], turned in place
            lq8.mrope(ctx, t.transpose(0, 1), rotary, pos, out=t.transpose(0, 1))
        ctx.call("lq_attention", q.data_ptr(), k.data_ptr(), v.data_ptr(), 1, Hq, Hkv, L, 0, None, L, D, None,
                 att[0].data_ptr(), att[1].data_ptr())
        w.matmul(w.o[i], att, x)
        w.mlp(x, i)
    return w.logits(x)


def grid_positions(n_text, rows, cols):
    """[3, n]: text (equal axes), then a rows x cols image, ending where the next text begins."""
    text = np.arange(n_text)
    r, q = np.divmod(np.arange(rows * cols), cols)
    pos = np.concatenate([np.stack([text] * 3), n_text + np.stack([0 * r, r, q])], axis=1)
    return pos, n_text + max(rows, cols)


def serve(cache_dtype=torch.float32, image=True, steps=6, seed=7, ctx=None):
    """Serves three questions behind one prompt, forcing the tokens that the first path chose.
    Returns (paged logits, contiguous logits, the model runner's where it can take the prompt):
    [steps + 1, 3, vocab] each."""
    ctx = ctx or lq8.Context(0)
    cfg = lq8.make_config(hidden=256, layers=2, n_heads=4, n_kv_heads=2, head_dim=128, inter=512, vocab=1000, tied=1, norm_std=0.1)
    model = lq8.Qwen3ForCausalLM(ctx, cfg, 1234, max_batch=1, ctx_max=256)
    w = Weights(ctx, model)
    if image:
        rotary = lq8.Rotary.build(64, 512, 1e6, lq8.Rotary.blocks([16, 24, 24]))
    else:  # the model runner's own tables
        ct = torch.empty((512, 64), device="cuda")
        st = torch.empty_like(ct)
        ctx.call("lq_rope_tables", 128, 512, 1e6, ct.data_ptr(), st.data_ptr())
        rotary = lq8.Rotary(ct, st)
    rng = np.random.default_rng(seed)
    prompt_pos, after = grid_positions(23, 4, 9) if image else (np.stack([np.arange(59)] * 3), 59)
    prompt = rng.integers(0, cfg.vocab, prompt_pos.shape[1])
    questions = [rng.integers(0, cfg.vocab, n) for n in (5, 1, 21)]
    text = [np.stack([after + np.arange(len(q) + steps)] * 3) for q in questions]
    dec = PagedDecoder(w, rotary, 64, cache_dtype)
    dec.share(prompt, i32(prompt_pos))
    lens = [len(q) for q in questions]
    got = [dec.start(questions, steps, i32(np.concatenate([t[:, :n] for t, n in zip(text, lens)], axis=1)))]
    tokens = []
    for s in range(steps):
        tokens.append(w.argmax(got[-1]))
        got.append(dec.step(tokens[-1], i32(np.stack([t[:, n + s] for t, n in zip(text, lens)], axis=1))))
    ctx.device_status()
    tokens = torch.stack(tokens).cpu().numpy()
    want = []
    for b, q in enumerate(questions):
        ids = np.concatenate([prompt, q, tokens[:, b]])
        lg = contiguous_logits(w, rotary, ids, i32(np.concatenate([prompt_pos, text[b]], axis=1)))
        want.append(lg[len(prompt) + len(q) - 1:])
    runner = None
    if not image:  # the runner, one sequence at a time, on the same tokens
        runner = []
        for b, q in enumerate(questions):
            model.clear_kv_cache()
            lg = [model.prefill(np.concatenate([prompt, q]), want_logits=True)[1][0]]
            for s in range(steps):
                lg.append(model.decode_step(tokens[s, b:b + 1], want_logits=True)[1][0])
            runner.append(np.stack(lg))
        runner = torch.from_numpy(np.stack(runner, axis=1)).cuda()
    model.close()
    return torch.stack(got), torch.stack(want, dim=1), runner


def main():
    for dtype in (torch.float32, torch.bfloat16, torch.int8):
        for image in (True, False):
            t0 = time.time()
            got, want, runner = serve(dtype, image)
            far = lambda a, b: float((a - b).abs().max() / b.abs().max())  # noqa: E731
            print(f"{str(dtype):16s} {'image in the prompt' if image else 'text only':20s} largest logit difference / largest logit: "
                  f"contiguous path {far(got, want):.2e}" + (f", model runner {far(got, runner):.2e}" if runner is not None else "") +
                  f"  ({time.time() - t0:.1f} s)")


if __name__ == "__main__":
    main()
