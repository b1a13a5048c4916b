"""The serving-step operators together, as a program uses them: rotate and append, attend, sample -- over several steps of a ragged batch whose sequences
join and grow, eagerly, on another stream, and captured once and replayed with new lengths."""
import numpy as np
import pytest

import serving_reference as ref
from gpu_util import bridge, ctx, synth  # noqa: F401

pytestmark = pytest.mark.gpu
nH, nKV, HD, PAGE, VOCAB = 8, 2, 64, 16, 300


class Program:
    """One layer's worth of a server: a paged cache, a page table that hands out pages, and the four calls."""

    def __init__(self, ctx, n_seq, rows, dtype="f32", pages=40, wide=12):
        self.ctx, self.dtype, self.n_seq, self.rows = ctx, dtype, n_seq, rows
        zero = np.zeros((pages, PAGE, nKV, HD), np.float32)
        self.cache = bridge.PagedCache(ctx.array(zero, dtype), ctx.array(zero, dtype))
        self.cfg = bridge.RopeConfig.make(HD, 32, layout="half", scaling="linear", factor=2.0)
        self.freqs = ctx.rope_frequencies(self.cfg)
        self.q_start, self.kv_len, self.table = ctx.array(np.zeros(n_seq + 1, np.int32), "i32"), ctx.array(np.zeros(n_seq, np.int32), "i32"), ctx.array(np.zeros((n_seq, wide), np.int32), "i32")
        self.batch = bridge.PagedBatch(self.q_start, self.kv_len, self.table, rows, rows)
        self.q, self.k, self.v = (ctx.empty((rows, h, HD), dtype) for h in (nH, nKV, nKV))
        self.q_rot, self.o = ctx.empty((rows, nH, HD), dtype), ctx.empty((rows, nH, HD), dtype).zero()
        self.lse = ctx.empty((rows, nH))
        self.ws = ctx.empty((ctx.paged_attn_workspace(self.cache, self.batch, nH) // 4,))
        w = synth.normal(3, "w", (nH * HD, VOCAB)) * np.float32(0.2)
        self.w_host, self.w = (synth.bf16_round(w) if dtype == "bf16" else w), ctx.array(w, dtype)
        self.logits, self.u = ctx.empty((rows, VOCAB), dtype), ctx.empty((rows,))
        self.out = (ctx.empty((rows,), "i32"), ctx.empty((rows,), "i32"), ctx.empty((rows,)))
        self.free, self.tab, self.lens = list(range(pages))[::-1], np.full((n_seq, wide), -1, np.int32), np.zeros(n_seq, np.int64)
        self.keys, self.values = [[] for _ in range(n_seq)], [[] for _ in range(n_seq)]

    def set(self, counts, seed):
        """New rows for each sequence: pages, lengths and inputs to the device."""
        for s, n in enumerate(counts):
            for p in range(-(-int(self.lens[s]) // PAGE), -(-int(self.lens[s] + n) // PAGE)):
                self.tab[s, p] = self.free.pop()
            self.lens[s] += n
        self.counts = counts
        rnd = synth.bf16_round if self.dtype == "bf16" else (lambda x: x)
        self.h = [rnd(synth.normal(seed, n, (self.rows, h, HD))) for n, h in (("q", nH), ("k", nKV), ("v", nKV))]
        self.u_host = (synth.token_ids(seed, "u", (self.rows,), 1 << 24) / (1 << 24)).astype(np.float32)
        for d, x in zip((self.q, self.k, self.v, self.u), self.h + [self.u_host]):
            d.upload(x)
        self.q_start.upload(np.concatenate(([0], np.cumsum(counts))))
        self.kv_len.upload(self.lens)
        self.table.upload(self.tab)

    def step(self):
        c = self.ctx
        c.paged_append(self.cache, self.batch, self.k, self.v, rope=self.cfg, freqs=self.freqs, q=self.q, q_out=self.q_rot)
        c.paged_attn(self.cache, self.batch, self.q_rot, out=self.o, lse=self.lse, workspace=self.ws)
        c._check(c.lib.b200_gemm(c.h, self.o.ptr, self.w.ptr, self.logits.ptr, self.rows, VOCAB, nH * HD, 0, 0, 0, self.o.code, self.o.code))
        c.sample_given(self.logits, self.u, out=self.out)

    def check(self):
        """Attention from the history of all rows so far; the sampled ids from the logits that the device itself computed."""
        f, row, eps = ref.frequencies(self.cfg), 0, 2.0 ** -8 if self.dtype == "bf16" else 2.0 ** -24
        got = self.o.download()
        for s, n in enumerate(self.counts):
            pos = self.lens[s] - n + np.arange(n)
            k, _ = ref.rope(self.h[1][row:row + n], pos, f, 32, "half")
            q, _ = ref.rope(self.h[0][row:row + n], pos, f, 32, "half")
            self.keys[s].extend(k); self.values[s].extend(self.h[2][row:row + n].astype(np.float64))
            K, V = np.array(self.keys[s]), np.array(self.values[s])
            for i in range(n):
                m = int(pos[i]) + 1
                for h in range(nH):
                    g = h // (nH // nKV)
                    sc = K[:m, g] @ q[i, h] / np.sqrt(HD)
                    p = np.exp(sc - sc.max())
                    p /= p.sum()
                    want, A = p @ V[:m, g], p @ np.abs(V[:m, g])
                    # a half step for the result and one for the probabilities, and what the half steps of q and k do to a score: eps x sum |q k|
                    # scaled, twice, to first order on both sides of the quotient
                    noise = 2 * 2 * eps * (np.abs(K[:m, g]) @ np.abs(q[i, h])).max() / np.sqrt(HD)
                    assert (np.abs(got[row + i, h] - want) <= 1.1 * A * (2 * eps + noise) + 1e-5 * A).all(), (s, i, h)
            row += n
        logits, tok = self.logits.download(), self.out[0].download()
        for r in range(row):
            assert int(tok[r]) == ref.sample(logits[r], float(self.u_host[r]))[0]


STEPS = [[7, 1, 20], [1, 1, 1], [1, 16, 0], [1, 1, 1]]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_steps_of_a_growing_batch(ctx, dtype):
    p = Program(ctx, 3, 28, dtype)
    for i, counts in enumerate(STEPS):
        p.set(counts, 10 + i)
        p.step()
        ctx.sync()
        p.check()


def test_two_programs_in_turn_and_another_stream(ctx):
    """Two servers share the context; the second half of the work is enqueued on another library's stream."""
    import torch
    a, b = Program(ctx, 3, 28, "bf16"), Program(ctx, 3, 28, "bf16")
    stream = torch.cuda.Stream()
    try:
        for i, counts in enumerate(STEPS):
            if i == 2:
                ctx.sync()
                ctx.use_stream(stream.cuda_stream)
            a.set(counts, 20 + i)
            b.set(counts, 40 + i)
            a.step()
            b.step()
            ctx.sync()
            a.check()
            b.check()
    finally:
        ctx.own_stream()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_step_replays_with_new_lengths(ctx, dtype):
    """One capture, replayed as sequences grow: lengths and tables are read on the device.  Two captures with workspaces of their own, replayed in turn."""
    import torch
    stream = torch.cuda.Stream()
    ps = [Program(ctx, 3, 28, dtype), Program(ctx, 3, 28, dtype)]
    ctx.use_stream(stream.cuda_stream)
    graphs = []
    try:
        for i, p in enumerate(ps):                           # an eager step first: kernel attributes and workspaces are set up outside the capture
            p.set(STEPS[0], 60 + i)
            p.step()
            ctx.sync()
            p.check()
        for p in ps:
            g = torch.cuda.CUDAGraph()
            stream.wait_stream(torch.cuda.current_stream())
            with torch.cuda.graph(g, stream=stream):
                p.step()
            graphs.append(g)
        for i, counts in enumerate(STEPS[1:]):
            for j, p in enumerate(ps):
                p.set(counts, 70 + 10 * j + i)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                for g in graphs:
                    g.replay()
            torch.cuda.synchronize()
            for p in ps:
                p.check()
    finally:
        ctx.own_stream()
    del graphs


def test_bad_batches_are_reported_and_the_context_goes_on(ctx):
    """Page ids and lengths out of range (shown on the CPU to stay inside the arrays): b200_sync names them, the next call is right."""
    for dtype in ("f32", "bf16"):
        p = Program(ctx, 3, 28, dtype)
        p.set(STEPS[0], 90)
        good = p.tab.copy()
        for table, lens in ((np.where(good >= 0, 10 ** 6, good), p.lens), (good, p.lens + 1000), (np.full_like(good, -7), p.lens)):
            p.table.upload(table)
            p.kv_len.upload(lens)
            p.step()
            with pytest.raises(bridge.B200Error, match="paged batch"):
                ctx.sync()
        p.table.upload(good)
        p.kv_len.upload(p.lens)
        p.step()
        ctx.sync()
        p.check()


def test_long_cache_offsets_beyond_32_bits(ctx):
    """A pool of pages whose last page lies more than 2^32 bytes and 2^31 elements from its first: append to it and attend over it."""
    import torch
    pages, page, kv, hd = 66000, 64, 4, 128                       # 2.16e9 elements each
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of free device memory")
    cache = bridge.PagedCache(ctx.empty((pages, page, kv, hd), "bf16"), ctx.empty((pages, page, kv, hd), "bf16"))
    table = np.array([[pages - 1, 0, pages - 2], [pages - 3, 1, -1]], np.int32)
    kv_lens, q_lens, rows = [150, 100], [150, 100], 250
    k, v, q = (synth.bf16_round(synth.normal(5, n, (rows, h, hd))) for n, h in (("k", kv), ("v", kv), ("q", 8)))
    batch = bridge.PagedBatch(ctx.array(np.array([0, 150, 250], np.int32), "i32"), ctx.array(np.array(kv_lens, np.int32), "i32"), ctx.array(table, "i32"), rows)
    ctx.paged_append(cache, batch, ctx.array(k, "bf16"), ctx.array(v, "bf16"))
    one = bridge.PagedBatch(ctx.array(np.array([0, 1, 2], np.int32), "i32"), batch.arrays[1], batch.arrays[2], 2)
    lone_q = np.stack([q[149], q[249]])
    full = ctx.paged_attn(cache, batch, ctx.array(q, "bf16"))
    lone = ctx.paged_attn(cache, one, ctx.array(lone_q, "bf16"))
    ctx.sync()
    dense = np.zeros((2, 3, page, kv, hd), np.float32), np.zeros((2, 3, page, kv, hd), np.float32)
    at = 0
    for s, n in enumerate(q_lens):
        for d, x in zip(dense, (k, v)):
            d[s].reshape(-1, kv, hd)[:n] = x[at:at + n]
        at += n
    t2 = np.array([[0, 1, 2], [3, 4, 5]], np.int32)
    kp, vp = (d.reshape(6, page, kv, hd) for d in dense)
    o, _, A, s = ref.attention(q, kp, vp, q_lens, kv_lens, t2)
    bound = 1.02 * (2.0 ** -8 * np.abs(o) + A * 2.0 ** -8) + A * (2 * hd * 2.0 ** -24 * s[..., None] + 2e-5)
    assert (np.abs(full.download() - o) <= bound).all()
    assert (np.abs(lone.download() - o[[149, 249]]) <= bound[[149, 249]]).all()
    for x in (cache.k, cache.v):
        x.free()
