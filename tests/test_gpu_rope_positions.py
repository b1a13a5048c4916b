"""Rotary embedding at given positions and the append to a paged cache against 64-bit forms.

Tolerances: one rounding to the output type (half a step: bf16 2^-8, fp32 2^-24 of the value), and of the pair's size |a| + |b|
5e-7: sine and cosine to 2 units of 2^-24, the angle's rounding to 32 bits (2^-25 turns at most, 1.9e-7 rad), three roundings of the products."""
import numpy as np
import pytest

import serving_reference as ref
from gpu_util import bridge, ctx, synth  # noqa: F401

pytestmark = pytest.mark.gpu
STEP = {"bf16": 2.0 ** -8, "f32": 2.0 ** -24}


def values(seed, name, shape, dtype):
    x = synth.normal(seed, name, shape)
    return synth.bf16_round(x) if dtype == "bf16" else x


def close(got, want, size, dtype):
    bound = STEP[dtype] * np.abs(want) + 5e-7 * size + (2.0 ** -8 * 5e-7 * size if dtype == "bf16" else 0)
    bad = ~(np.abs(got - want) <= bound)
    assert not bad.any(), (int(bad.sum()), float(np.abs(got - want).max()))


@pytest.mark.parametrize("scaling", ["plain", "linear", "ntk", "yarn", "bands"])
@pytest.mark.parametrize("rd", [2, 64, 128])
def test_frequencies(ctx, scaling, rd):
    cfg = bridge.RopeConfig.make(128, rd, scaling=scaling, base=500000.0, factor=8.0, original_len=8192.0)
    # pow and log of the device are within 2 units of 2^-53; their arguments' errors grow by ln(base)
    np.testing.assert_allclose(ctx.rope_frequencies(cfg).download(), ref.frequencies(cfg), rtol=1e-13)
    want = 0.1 * np.log(8.0) + 1 if scaling == "yarn" else 1.0
    assert abs(ctx.lib.b200_rope_amplitude(bridge.C.byref(cfg)) - want) < 1e-6


@pytest.mark.parametrize("backward", [False, True])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,qh,kvh,hd,rd,dtype", [(1, 16, 4, 128, 128, "bf16"), (7, 3, 1, 80, 24, "f32"), (33, 4, 2, 64, 10, "bf16"), (5, 2, 1, 7, 6, "f32"),
                                                       (3, 1, 1, 256, 256, "bf16"), (2, 2, 2, 96, 0, "bf16"), (1203, 4, 1, 128, 64, "f32"), (2500, 2, 2, 1024, 1024, "bf16")])
def test_rotation_matches(ctx, tokens, qh, kvh, hd, rd, dtype, layout, backward):
    cfg = bridge.RopeConfig.make(hd, rd, layout=layout, amplitude=1.25)
    freqs = 10000.0 ** (-2.0 * np.arange(max(1, rd // 2)) / max(rd, 1))
    pos = (synth.token_ids(3, "pos", (tokens,), 2000003).astype(np.int64) - 1000001).astype(np.int32)
    pos[0] = 2 ** 31 - 1 if tokens > 5 else 0
    q, k = values(1, "q", (tokens, qh, hd), dtype), values(2, "k", (tokens, kvh, hd), dtype)
    dq, dk, f, p = ctx.array(q, dtype), ctx.array(k, dtype), ctx.array(freqs, "f64"), ctx.array(pos, "i32")
    fn = ctx.rope_positions_backward if backward else ctx.rope_positions_forward
    oq, ok = fn(cfg, f, p, dq, dk)
    sign = -1.0 if backward else 1.0
    for got, x in ((oq, q), (ok, k)):
        want, size = ref.rope(x, pos, freqs[:rd // 2], rd, layout, 1.25, sign)
        close(got.download(), want, size, dtype)
    fn(cfg, f, p, dq, dk, out=(dq, dk))                      # in place: the same bits
    np.testing.assert_array_equal(dq.download(), oq.download())
    np.testing.assert_array_equal(dk.download(), ok.download())


def test_backward_is_the_derivative_of_forward(ctx):
    """Differences of the forward pass (which is linear, so one step of any size is exact up to rounding) against the backward."""
    tokens, heads, hd = 3, 2, 32
    cfg = bridge.RopeConfig.make(hd, 20, layout="half", amplitude=0.5)
    f, p = ctx.rope_frequencies(cfg), ctx.array(np.array([0, 17, 99999], np.int32), "i32")
    x, g = synth.normal(4, "x", (tokens, heads, hd)), synth.normal(5, "g", (tokens, heads, hd))
    dx = ctx.rope_positions_backward(cfg, f, p, ctx.array(g))[0].download()
    for i in range(0, hd, 3):
        step = np.zeros_like(x)
        step[..., i] = 1.0
        up, dn = (ctx.rope_positions_forward(cfg, f, p, ctx.array(x + s * step))[0].download().astype(np.float64) for s in (0.5, -0.5))
        # the inputs x +- 0.5 round to 32 bits (2^-24 x 5), the outputs too
        np.testing.assert_allclose(((up - dn) * g).sum(-1), dx[..., i], atol=2e-5)


def test_strided_rows_and_one_operand(ctx):
    """Queries read from rows of a fused projection, no keys; odd strides take the element-wise path."""
    tokens, heads, hd = 6, 3, 64
    for ld, off in ((heads * hd + 2 * hd, 0), (heads * hd + 5, 1)):
        buf = synth.normal(6, "rows", (tokens * ld + 8,))
        d, out = ctx.array(buf), ctx.empty((tokens, heads, hd))
        cfg = bridge.RopeConfig.make(hd)
        f, pos = ctx.rope_frequencies(cfg), np.arange(tokens, dtype=np.int32) * 1000
        p = ctx.array(pos, "i32")
        ctx._check(ctx.lib.b200_rope_positions_forward(ctx.h, bridge.C.byref(cfg), f.ptr, p.ptr, d.at(off), out.ptr, ld, heads * hd, heads, None, None, 0, 0, 0, tokens, 0))
        x = np.stack([buf[off + t * ld:off + t * ld + heads * hd].reshape(heads, hd) for t in range(tokens)])
        want, size = ref.rope(x, pos, ref.frequencies(cfg), hd, "interleaved")
        close(out.download(), want, size, "f32")


CASES = [([1, 1, 1], [1, 40, 17], 16, "bf16"), ([5, 0, 3], [5, 9, 130], 8, "f32"), ([4, 2], [2, 2], 1, "bf16"), ([70], [200], 24, "bf16"), ([1] * 300, list(range(1, 301)), 16, "f32")]


@pytest.mark.parametrize("layout", [None, "half", "interleaved"])
@pytest.mark.parametrize("q_lens,kv_lens,page,dtype", CASES)
def test_append_writes_exactly_the_new_slots(ctx, q_lens, kv_lens, page, dtype, layout):
    n_kv, qh, hd, n_seq, spare = 2, 6, 64, len(q_lens), 2
    need = [-(-m // page) for m in kv_lens]
    n_pages, wide = sum(need) + 3, max(need) + 1
    rng = np.random.RandomState(7)
    order, table, at = rng.permutation(n_pages), np.full((n_seq, wide), -1, np.int32), 0
    for s, n in enumerate(need):
        table[s, :n] = order[at:at + n]
        at += n
    rows = sum(q_lens) + spare                                 # two rows behind the last sequence
    q_start = np.concatenate(([0], np.cumsum(q_lens))).astype(np.int32)
    shape = (n_pages, page, n_kv, hd)
    kp, vp = values(1, "kp", shape, dtype), values(2, "vp", shape, dtype)
    k, v, q = (values(3, n, (rows, h, hd), dtype) for n, h in (("k", n_kv), ("v", n_kv), ("q", qh)))
    cache = bridge.PagedCache(ctx.array(kp, dtype), ctx.array(vp, dtype))
    batch = bridge.PagedBatch(ctx.array(q_start, "i32"), ctx.array(np.array(kv_lens, np.int32), "i32"), ctx.array(table, "i32"), rows)
    cfg = bridge.RopeConfig.make(hd, 32, layout=layout) if layout else None
    f = ctx.rope_frequencies(cfg) if layout else None
    q_out = ctx.array(np.full(q.shape, 9.0, np.float32), dtype)
    ctx.paged_append(cache, batch, ctx.array(k, dtype), ctx.array(v, dtype), rope=cfg, freqs=f, q=ctx.array(q, dtype), q_out=q_out)
    ctx.sync()
    pos = np.concatenate([m - n + np.arange(n) for n, m in zip(q_lens, kv_lens)] + [np.zeros(spare)])
    turn = (lambda x: ref.rope(x, pos, ref.frequencies(cfg), 32, layout)) if layout else (lambda x: (x.astype(np.float64), np.zeros(x.shape)))
    wk, sk = kp.astype(np.float64), np.zeros(shape)
    wv, (rk, rs) = vp.copy(), turn(k)
    for row, _, _, pg, slot in ref.slots(q_lens, kv_lens, table, page):
        wk[pg, slot], sk[pg, slot], wv[pg, slot] = rk[row], rs[row], v[row]
    close(cache.k.download(), wk, sk, dtype)
    np.testing.assert_array_equal(cache.v.download(), wv)
    got, (wq, sq) = q_out.download(), turn(q)
    close(got[:rows - spare], wq[:rows - spare], sq[:rows - spare], dtype)
    np.testing.assert_array_equal(got[rows - spare:], np.full((spare, qh, hd), 9.0))
