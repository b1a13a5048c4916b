"""Attention of a ragged batch over a paged cache against a 64-bit form.

Tolerance of an output element: with A = sum p |v| and s = the largest scale * sum |q k| of the row,
  half a step of the type (bf16 2^-8, fp32 2^-24) of the value;  A x (2 e + r + (keys + 16) 2^-24 + 2^-21), where
  e = hd 2^-24 s, the rounding of a score's sum; r = 2^-8 for bf16 (probabilities are rounded to it before the product with V), else 0; the
  sums over the keys; and 2^-21 for the base-2 exponential and its argument (both within 2^-22 at |argument| < 2^2 near the maximum).
The log-sum-exp is a 32-bit number of either type: e + (keys + 16) 2^-24 + 2^-21 (1 + |lse|)."""
import numpy as np
import pytest

import serving_reference as ref
from gpu_util import bridge, ctx, synth  # noqa: F401

pytestmark = pytest.mark.gpu
STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


class Made:
    def __init__(self, ctx, q_lens, kv_lens, nH, nKV, hd, page, dtype, seed=1, spare=2, head_major=False, sharp=1.5):
        rnd = synth.bf16_round if dtype == "bf16" else (lambda x: x)
        need = [max(1, -(-m // page)) for m in kv_lens]
        n_pages, wide = sum(need) + 2, max(need) + 1
        order = np.random.RandomState(seed).permutation(n_pages)
        self.table, at = np.full((len(q_lens), wide), -1, np.int32), 0
        self.kp, self.vp = (rnd(synth.normal(seed, n, (n_pages, page, nKV, hd))) for n in ("kp", "vp"))
        dirty_k, dirty_v = np.full_like(self.kp, np.nan), np.full_like(self.vp, np.inf)     # slots never written hold anything
        for s, n in enumerate(need):
            ids = order[at:at + n]
            at += n
            self.table[s, :n] = ids
            for j, p in enumerate(ids):
                m = min(page, max(0, kv_lens[s] - j * page))
                dirty_k[p, :m], dirty_v[p, :m] = self.kp[p, :m], self.vp[p, :m]
        self.dirty = dirty_k, dirty_v
        rows = sum(q_lens) + spare
        self.q_lens, self.kv_lens, self.rows, self.spare, self.dtype, self.hd = q_lens, kv_lens, rows, spare, dtype, hd
        self.q = rnd(synth.normal(seed, "q", (rows, nH, hd)) * np.float32(sharp))
        self.q_start = np.concatenate(([0], np.cumsum(q_lens))).astype(np.int32)
        if head_major:                                                   # pages [n, kv heads, page, hd]
            arr = [ctx.array(np.ascontiguousarray(x.transpose(0, 2, 1, 3)), dtype) for x in self.dirty]
            view = [ctx.wrap(x.ptr, self.kp.shape, dtype) for x in arr]
            self.cache = bridge.PagedCache(*view, page_stride=page * nKV * hd, token_stride=hd, head_stride=page * hd)
        else:
            self.cache = bridge.PagedCache(*(ctx.array(x, dtype) for x in self.dirty))
        self.batch = bridge.PagedBatch(ctx.array(self.q_start, "i32"), ctx.array(np.array(kv_lens, np.int32), "i32"), ctx.array(self.table, "i32"), rows, max(max(q_lens), 1))
        self.d_q = ctx.array(self.q, dtype)
        self.out, self.lse = ctx.array(np.full(self.q.shape, 7.0, np.float32), dtype), ctx.array(np.full((rows, nH), 7.0, np.float32))

    def check(self, got=None, lse=None, scale=None):
        got, lse = (self.out.download() if got is None else got), (self.lse.download() if lse is None else lse)
        o, l, A, s = ref.attention(self.q, self.kp, self.vp, self.q_lens, self.kv_lens, self.table, scale)
        n = max(self.kv_lens) if self.kv_lens else 0
        e = (self.hd * 2.0 ** -24 * s)
        sums = (n + 16) * 2.0 ** -24
        bound = STEP[self.dtype] * np.abs(o) * 1.01 + A * (2 * e[..., None] + (2.0 ** -8 if self.dtype == "bf16" else 0) * 1.01 + sums + 2.0 ** -21)
        live = self.rows - self.spare
        bad = ~(np.abs(got - o)[:live] <= bound[:live])
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:3].tolist(), float(np.nanmax(np.abs(got - o)[:live])))
        empty = ~np.isfinite(l[:live])
        assert (lse[:live][empty] == -np.inf).all() and (got[:live][empty] == 0).all()
        le, got_l, err = l[:live][~empty], lse[:live][~empty], e[:live][~empty]
        bad = ~(np.abs(got_l - le) <= err + sums + 2.0 ** -21 * (1 + np.abs(le)))
        assert not bad.any(), int(bad.sum())
        assert (got[live:] == 7.0).all() and (lse[live:] == 7.0).all()     # rows behind the last sequence


def run(ctx, m, **kw):
    ctx.paged_attn(m.cache, m.batch, m.d_q, out=m.out, lse=m.lse, **kw)
    ctx.sync()


LENS = {
    "one token": ([1], [1]),
    "single tokens": ([1, 1, 1, 1], [1, 16, 17, 300]),
    "with idle and empty sequences": ([1, 0, 2, 1], [40, 9, 0, 64]),
    "drafts": ([2, 5, 1, 8], [2, 100, 257, 1000]),
    "padding rows first": ([6, 3], [4, 3]),
    "chunks": ([40, 129], [40, 500]),
    "long padding": ([100, 40, 3], [60, 0, 0]),
    "chunks and tokens": ([1, 150, 1, 1, 33], [700, 150, 5, 1200, 90]),
}
HEADS = [(4, 1, 128), (8, 2, 64), (3, 3, 128), (5, 1, 64), (16, 2, 128), (6, 2, 80), (2, 1, 256), (3, 1, 20)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nH,nKV,hd", HEADS)
@pytest.mark.parametrize("lens", list(LENS))
def test_ragged_batches(ctx, lens, nH, nKV, hd, dtype):
    m = Made(ctx, *LENS[lens], nH, nKV, hd, 16, dtype)
    run(ctx, m)
    m.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("page", [1, 5, 8, 24, 64, 128, 256, 1000])
def test_page_sizes(ctx, page, dtype):
    m = Made(ctx, [1, 70, 3], [301, 200, 129], 4, 2, 64, page, dtype, seed=page)
    run(ctx, m)
    m.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_pages_by_head(ctx, dtype):
    m = Made(ctx, [1, 60, 3], [301, 200, 129], 8, 2, 128, 16, dtype, head_major=True)
    run(ctx, m)
    m.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("nH,nKV,hd,q,kv", [(4, 1, 128, 1, 9000), (1, 1, 64, 3, 4097), (64, 1, 64, 2, 700), (32, 8, 128, 1, 2500), (40, 1, 128, 30, 800), (200, 1, 64, 3, 300)])
def test_long_caches_and_wide_groups(ctx, nH, nKV, hd, q, kv, dtype):
    m = Made(ctx, [q], [kv], nH, nKV, hd, 32, dtype)
    run(ctx, m)
    m.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_sequences(ctx, dtype):
    """More sequences than threads in a CTA, chunks among single tokens."""
    rng = np.random.RandomState(3)
    kv = rng.randint(1, 60, 700).tolist()
    q = [min(m, 1 if i % 9 else int(rng.randint(1, 40))) for i, m in enumerate(kv)]
    m = Made(ctx, q, kv, 2, 1, 64, 8, dtype)
    run(ctx, m)
    m.check()


def test_scale_and_peaked_scores(ctx):
    """A scale of its own; scores so far apart that all but one probability vanish."""
    m = Made(ctx, [1, 80], [333, 400], 4, 2, 128, 16, "bf16", sharp=8.0)
    run(ctx, m, scale=0.5)
    m.check(scale=0.5)


@pytest.mark.parametrize("dtype,hd", [("bf16", 128), ("f32", 80)])
def test_strided_queries_and_outputs(ctx, dtype, hd):
    m = Made(ctx, [1, 90, 2], [500, 90, 33], 4, 2, hd, 16, dtype)
    width = 4 * hd
    for ld, off in ((width + 2 * hd, hd), (width + 3, 1)):
        big = np.zeros((m.rows + 1, ld), np.float32)
        flat = big.reshape(-1)
        for r in range(m.rows):
            flat[off + r * ld:off + r * ld + width] = m.q[r].ravel()
        d_q, d_o = ctx.array(big, dtype), ctx.array(np.full_like(big, 7.0), dtype)
        ws = ctx.empty((ctx.paged_attn_workspace(m.cache, m.batch, 4) // 4,))
        ctx._check(ctx.lib.b200_paged_attn(ctx.h, m.cache.ref, m.batch.ref, d_q.at(off), ld, d_o.at(off), ld, m.lse.ptr, 4, 0.0, ws.ptr, ws.nbytes))
        ctx.sync()
        back = d_o.download().reshape(-1)
        got = np.stack([back[off + r * ld:off + r * ld + width].reshape(4, hd) for r in range(m.rows)])
        m.check(got)
        keep = np.ones(back.size, bool)
        for r in range(m.rows):
            keep[off + r * ld:off + r * ld + width] = False
        assert (back[keep] == 7.0).all()                       # nothing written between the rows


def test_the_same_call_gives_the_same_bits(ctx):
    m = Made(ctx, [1, 300, 5], [3000, 900, 77], 8, 2, 128, 16, "bf16")
    run(ctx, m)
    a, b = m.out.download(), m.lse.download()
    run(ctx, m)
    np.testing.assert_array_equal(a, m.out.download())
    np.testing.assert_array_equal(b, m.lse.download())


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shared_prefix_pages(ctx, dtype):
    """Two sequences whose first pages are the same ones."""
    m = Made(ctx, [1, 2], [100, 70], 4, 1, 64, 16, dtype)
    m.table[1, :3] = m.table[0, :3]
    m.batch = bridge.PagedBatch(ctx.array(m.q_start, "i32"), ctx.array(np.array(m.kv_lens, np.int32), "i32"), ctx.array(m.table, "i32"), m.rows)
    run(ctx, m)
    m.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lens", [([1], [1000]), ([2, 1], [40, 3000]), ([200], [700])])
def test_without_a_bound_on_the_rows_of_a_sequence(ctx, lens, dtype):
    """max_q 0 stands for all rows, of which there are many more than the sequences use."""
    m = Made(ctx, *lens, 8, 2, 128, 16, dtype, spare=150)
    m.batch = bridge.PagedBatch(*m.batch.arrays, m.rows)
    run(ctx, m)
    m.check()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_a_sequence_longer_than_the_bound_is_reported(ctx, dtype):
    m = Made(ctx, [1, 60], [100, 100], 8, 2, 64, 16, dtype)
    m.batch = bridge.PagedBatch(*m.batch.arrays, m.rows, 50)
    with pytest.raises(bridge.B200Error, match="paged batch"):
        run(ctx, m)
    m.batch = bridge.PagedBatch(*m.batch.arrays, m.rows, 60)
    run(ctx, m)
    m.check()


def test_arrays_of_the_wrong_kind_are_refused(ctx):
    m = Made(ctx, [1], [5], 4, 1, 64, 16, "f32")
    with pytest.raises(bridge.B200Error, match="int32"):
        bridge.PagedBatch(ctx.array(m.q_start.astype(np.float32)), *m.batch.arrays[1:], m.rows)
    with pytest.raises(bridge.B200Error, match="f32 or bf16"):
        bridge.PagedCache(ctx.empty((2, 16, 1, 64), "f64"), ctx.empty((2, 16, 1, 64), "f64"))
    for bad in (dict(q=ctx.empty((3, 4, 64), "bf16")), dict(out=ctx.empty((3, 4, 32))), dict(lse=ctx.empty((3, 5)))):
        kw = {**dict(q=m.d_q, out=m.out, lse=m.lse), **bad}
        with pytest.raises(bridge.B200Error):
            ctx.paged_attn(m.cache, m.batch, **kw)
    need = ctx.paged_attn_workspace(m.cache, m.batch, 4)
    with pytest.raises(bridge.B200Error, match="workspace"):
        ctx.paged_attn(m.cache, m.batch, m.d_q, out=m.out, workspace=ctx.empty((need // 4 - 1,)))
    with pytest.raises(bridge.B200Error):
        ctx.rope_positions_forward(bridge.RopeConfig.make(64), ctx.empty((32,), "f32"), ctx.empty((3,), "i32"), m.d_q)
    with pytest.raises(bridge.B200Error):
        ctx.sample_given(ctx.empty((3, 8), "i32"), ctx.empty((3,)))


def test_empty_batches_are_no_work(ctx):
    m = Made(ctx, [1], [5], 4, 1, 64, 16, "f32")
    before = ctx.launch_count()
    ctx._check(ctx.lib.b200_paged_attn(ctx.h, m.cache.ref, bridge.C.byref(bridge._PagedBatch(None, None, None, 0, 0, 0, 0)), None, 4 * 64, None, 4 * 64, None, 4, 0.0, None, 0))
    assert ctx.launch_count() == before
