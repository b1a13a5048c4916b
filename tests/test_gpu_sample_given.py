"""Sampling from given random numbers against a 64-bit form: ids and counts are equal, probabilities to 2^-22 (one rounding to fp32; weights
are whole multiples of 2^-44 of the largest, a share of at least 2^-20 in these cases)."""
import numpy as np
import pytest

import serving_reference as ref
from gpu_util import bridge, ctx, synth  # noqa: F401

pytestmark = pytest.mark.gpu


def check(ctx, x, u, T=None, k=None, p=None, m=None, dtype="f32"):
    B = x.shape[0]
    if dtype == "bf16":
        x = synth.bf16_round(x)
    full = lambda v, t: None if v is None else np.broadcast_to(np.asarray(v, t), (B,)).copy()  # noqa: E731
    u, T, p, m, k = full(u, np.float32), full(T, np.float32), full(p, np.float32), full(m, np.float32), full(k, np.int32)
    dev = lambda v, t="f32": None if v is None else ctx.array(v, t)  # noqa: E731
    tok, kept, prob = ctx.sample_given(ctx.array(x, dtype), dev(u), dev(T), dev(k, "i32"), dev(p), dev(m))
    tok, kept, prob = tok.download(), kept.download(), prob.download()
    for b in range(B):
        want = ref.sample(x[b], float(u[b]), 1.0 if T is None else float(T[b]), 0 if k is None else int(k[b]), 1.0 if p is None else float(p[b]), 0.0 if m is None else float(m[b]))
        assert (int(tok[b]), int(kept[b])) == want[:2], (b, int(tok[b]), int(kept[b]), want)
        assert abs(float(prob[b]) - want[2]) <= 2.0 ** -22 * max(want[2], 2.0 ** -20), (b, float(prob[b]), want)
    return tok, kept


SETTINGS = [dict(), dict(T=0.7), dict(k=1), dict(k=7, T=1.3), dict(p=0.9), dict(p=0.3, T=0.5), dict(m=0.1), dict(k=40, p=0.8, m=0.02, T=0.8), dict(T=0.0), dict(k=3, p=0.999), dict(p=0.0), dict(p=0.99999994)]


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("B,V", [(1, 1), (3, 2), (5, 33), (4, 1000), (2, 4099), (7, 32000), (1, 100256), (200, 517)])
@pytest.mark.parametrize("s", range(len(SETTINGS)))
def test_settings(ctx, B, V, s, dtype):
    x = synth.normal(B + V, "logits", (B, V)) * np.float32(3.0)
    u = (synth.token_ids(s, "u", (B,), 1 << 24).astype(np.float64) / (1 << 24)).astype(np.float32)
    check(ctx, x, u, dtype=dtype, **SETTINGS[s])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_settings_differ_by_row(ctx, dtype):
    B, V = 24, 5000
    r = np.random.RandomState(1)
    x = (r.randn(B, V) * 2.5).astype(np.float32)
    check(ctx, x, r.rand(B).astype(np.float32), np.where(r.rand(B) < 0.2, 0.0, r.rand(B) + 0.3), r.randint(0, 60, B), np.where(r.rand(B) < 0.5, 1.0, r.rand(B)), np.where(r.rand(B) < 0.5, 0.0, r.rand(B) * 0.2), dtype)


@pytest.mark.parametrize("V", [600, 40000, 100003])
@pytest.mark.parametrize("kind", ["all equal", "two values", "powers", "one far above", "lowest masks", "steps", "signed zeros"])
def test_ties_and_extreme_ranges(ctx, V, kind):
    """Equal values (lowest id first), more than the candidates a border is searched among; ranges that crowd one histogram bin."""
    r = np.random.RandomState(V)
    x = {"all equal": lambda: np.zeros(V), "two values": lambda: np.where(r.rand(V) < 0.5, 1.0, 0.0),
         "powers": lambda: -2.0 ** r.randint(-100, 100, V), "one far above": lambda: np.where(np.arange(V) == V // 2, 1e30, r.randn(V)),
         "lowest masks": lambda: np.where(r.rand(V) < 0.9, np.finfo(np.float32).min, r.randn(V)), "steps": lambda: np.floor(r.randn(V) * 2) / 2,
         "signed zeros": lambda: np.where(r.rand(V) < 0.5, -0.0, 0.0)}[kind]().astype(np.float32)
    u = np.array([0.0, 0.1, 0.37, 0.5, 0.83, 0.9999999], np.float32)
    x = np.broadcast_to(x, (6, V)).copy()
    for kw in (dict(), dict(k=5), dict(k=V // 2), dict(k=700, p=0.7), dict(p=0.6), dict(k=V - 1, p=0.95, m=0.5), dict(T=1e-3, p=0.5), dict(T=100.0, p=0.5, k=599)):
        check(ctx, x, u, **kw)


def test_masked_infinite_and_empty_rows(ctx):
    inf, nan = np.inf, np.nan
    x = np.zeros((6, 40), np.float32)
    x[0] = -inf
    x[1] = nan
    x[2] = np.where(np.arange(40) % 7 == 3, 1.0, -inf)
    x[3] = np.where(np.arange(40) == 11, inf, 2.0)
    x[4] = np.where(np.arange(40) % 2 == 0, nan, np.arange(40) / 10)
    x[5] = np.where(np.arange(40) >= 38, inf, -inf)
    for kw in (dict(), dict(T=0.0), dict(k=2), dict(p=0.5), dict(k=30, p=0.9, m=0.3)):
        tok, kept = check(ctx, x, np.full(6, 0.6, np.float32), **kw)
        assert tok[0] == -1 and kept[0] == 0 and tok[1] == -1


def test_settings_out_of_range_and_uniforms_out_of_range(ctx):
    """NaN and negative temperatures are greedy, top_k <= 0 or >= vocab, top_p >= 1 and min_p <= 0 are off; uniform is taken into [0, 1)."""
    x = np.random.RandomState(5).randn(8, 300).astype(np.float32)
    nan = float("nan")
    check(ctx, x, np.array([1.0, 2.0, -1.0, 0.5, 0.5, 0.5, 0.5, 1.0], np.float32), T=np.array([1, 1, 1, nan, -2, 1, 1, 1]), k=np.array([0, -5, 300, 0, 0, 10 ** 6, 0, 0]),
          p=np.array([1.5, 1.0, 1.0, 1, 1, nan, 1, 1]), m=np.array([0, 0, -1, 0, 0, 0, nan, 2.0]))


def test_the_draw_follows_the_weights(ctx):
    """Every uniform of a fine grid against the cumulative weights of one small row: the borders are where they have to be."""
    x = np.array([0.0, 1.0, -1.0, 0.5, 0.25], np.float32)
    n = 4096
    u = ((np.arange(n) + 0.5) / n).astype(np.float32)
    check(ctx, np.broadcast_to(x, (n, 5)).copy(), u)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strided_rows_and_optional_outputs(ctx, dtype):
    B, V, ld = 3, 1001, 1003
    big = np.full((B, ld), 50.0, np.float32)                    # what lies behind a row would win
    big[:, :V] = synth.bf16_round(synth.normal(9, "l", (B, V)))
    d, u, tok = ctx.array(big, dtype), ctx.array(np.full(B, 0.4, np.float32)), ctx.empty((B,), "i32")
    ctx._check(ctx.lib.b200_sample_given(ctx.h, d.ptr, d.code, B, V, ld, None, None, None, None, u.ptr, tok.ptr, None, None))
    assert tok.download().tolist() == [ref.sample(big[b, :V], 0.4000000059604645)[0] for b in range(B)]


def test_large_vocabulary_beyond_shared_memory(ctx):
    B, V = 2, 700001
    x = np.random.RandomState(2).randn(B, V).astype(np.float32) * 3
    for kw in (dict(), dict(k=50), dict(p=0.9, T=0.7)):
        check(ctx, x, np.array([0.2, 0.9], np.float32), **kw)


def test_the_largest_vocabulary(ctx):
    x = np.random.RandomState(4).randn(1, 1 << 24).astype(np.float32) * 2
    for kw in (dict(k=50, p=0.9), dict(p=0.5), dict(k=1 << 20, m=1e-4)):
        check(ctx, x, np.array([0.7], np.float32), dtype="bf16", **kw)
