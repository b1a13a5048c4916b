"""What the serving-step entry points refuse, without a GPU: every check of arguments comes before the first use of the device, so a
zeroed context serves.  And the device's checks of a batch, run on the host over the same code."""
import ctypes as C
import importlib

import numpy as np
import pytest

bridge = importlib.import_module("large-language-model_b200.bridge")
INVALID, UNSUPPORTED = -1, -3
P = 0x1000                                      # stands for a device pointer; nothing is read through it


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__ as ge
    ge.build_cuda()
    return bridge.load_library()


@pytest.fixture
def ctx():
    return C.create_string_buffer(1 << 14)      # larger than the context structure, all members empty


def cache(**kw):
    return bridge._PagedCache(**{**dict(k=P, v=P, n_pages=4, page_size=16, n_kv=2, head_dim=64, page_stride=2048, token_stride=128, head_stride=64, dtype=1), **kw})


def batch(**kw):
    return bridge._PagedBatch(**{**dict(q_start=P, kv_len=P, page_table=P, n_seq=1, table_ld=2, rows=3, max_q=3), **kw})


def attn(lib, ctx, c=None, b=None, q=P, ld_q=512, o=P, ld_o=512, nH=8, scale=0.0, ws=P, n=1 << 30):
    return lib.b200_paged_attn(ctx, C.byref(c or cache()), C.byref(b or batch()), q, ld_q, o, ld_o, None, nH, scale, ws, n)


BAD_CACHE = [dict(k=None), dict(v=None), dict(n_pages=0), dict(page_size=0), dict(page_size=65537), dict(n_kv=0), dict(head_dim=0), dict(head_dim=2048), dict(page_stride=0),
             dict(token_stride=0), dict(head_stride=63), dict(dtype=2), dict(n_pages=1 << 31), dict(page_stride=1 << 41)]
BAD_BATCH = [dict(q_start=None), dict(kv_len=None), dict(page_table=None), dict(table_ld=0), dict(table_ld=1 << 28), dict(n_seq=65537), dict(rows=1 << 30)]


@pytest.mark.parametrize("kw", BAD_CACHE)
def test_bad_caches(lib, ctx, kw):
    assert attn(lib, ctx, c=cache(**kw)) == INVALID
    assert lib.b200_paged_append(ctx, C.byref(cache(**kw)), C.byref(batch()), P, P, 128, 128, None, None, None, None, 0, 0, 0) == INVALID
    assert lib.b200_last_error(ctx)


@pytest.mark.parametrize("kw", BAD_BATCH)
def test_bad_batches(lib, ctx, kw):
    assert attn(lib, ctx, b=batch(**kw)) == INVALID
    assert lib.b200_paged_append(ctx, C.byref(cache()), C.byref(batch(**kw)), P, P, 128, 128, None, None, None, None, 0, 0, 0) == INVALID


@pytest.mark.parametrize("kw", [dict(q=None), dict(o=None), dict(ld_q=511), dict(ld_o=511), dict(nH=0), dict(nH=7), dict(scale=float("nan")), dict(scale=-1.0), dict(ws=None), dict(ws=P + 4)])
def test_bad_attention_calls(lib, ctx, kw):
    assert attn(lib, ctx, **kw) == INVALID


def test_heads_no_kernel_takes(lib, ctx):
    c = cache(head_dim=512, head_stride=512, token_stride=1024, page_stride=16384)
    assert attn(lib, ctx, c=c, ld_q=4096, ld_o=4096) == UNSUPPORTED


def test_null_contexts_and_descriptors(lib, ctx):
    n = C.c_size_t(0)
    assert lib.b200_paged_attn(None, C.byref(cache()), C.byref(batch()), P, 512, P, 512, None, 8, 0.0, P, 1 << 30) == INVALID
    assert lib.b200_paged_attn(ctx, None, C.byref(batch()), P, 512, P, 512, None, 8, 0.0, P, 1 << 30) == INVALID
    assert lib.b200_paged_attn(ctx, C.byref(cache()), None, P, 512, P, 512, None, 8, 0.0, P, 1 << 30) == INVALID
    assert lib.b200_paged_attn_workspace(ctx, C.byref(cache()), C.byref(batch()), 8, None) == INVALID
    assert lib.b200_paged_attn_workspace(ctx, C.byref(cache()), C.byref(batch()), 9, C.byref(n)) == INVALID
    assert lib.b200_sample_given(None, P, 0, 1, 8, 8, None, None, None, None, P, P, None, None) == INVALID
    assert lib.b200_rope_frequencies(ctx, None, P) == INVALID


@pytest.mark.parametrize("kw", [dict(rotary_dim=3), dict(rotary_dim=66), dict(head_dim=0, rotary_dim=0), dict(head_dim=2048), dict(layout=2), dict(scaling=5), dict(scaling=-1), dict(amplitude=float("inf")),
                                dict(amplitude=-1.0)])
def test_bad_rope_configurations(lib, ctx, kw):
    cfg = bridge.RopeConfig.make(64)
    for n, v in kw.items():
        setattr(cfg, n, v)
    for fn in (lib.b200_rope_positions_forward, lib.b200_rope_positions_backward):
        assert fn(ctx, C.byref(cfg), P, P, P, P, 4096, 4096, 2, None, None, 0, 0, 0, 5, 1) == INVALID
    assert lib.b200_rope_frequencies(ctx, C.byref(cfg), P) == INVALID
    assert lib.b200_paged_append(ctx, C.byref(cache()), C.byref(batch()), P, P, 128, 128, C.byref(cfg), P, None, None, 0, 0, 0) == INVALID


@pytest.mark.parametrize("kw", [dict(base=1.0), dict(base=float("nan")), dict(scaling=1, factor=0.5), dict(scaling=3, factor=2, original_len=0.0), dict(scaling=3, factor=2, beta_slow=0.0),
                                dict(scaling=3, factor=2, beta_fast=0.5), dict(scaling=4, factor=2, high_freq_factor=1.0)])
def test_bad_frequencies(lib, ctx, kw):
    cfg = bridge.RopeConfig.make(64)
    for n, v in kw.items():
        setattr(cfg, n, v)
    assert lib.b200_rope_frequencies(ctx, C.byref(cfg), P) == INVALID


def test_bad_rope_and_append_calls(lib, ctx):
    cfg = bridge.RopeConfig.make(64)
    go = lambda freqs=P, pos=P, q=P, qo=P, ld=128, ldo=128, heads=2, t=5, dt=1, k=None, ko=None: lib.b200_rope_positions_forward(  # noqa: E731
        ctx, C.byref(cfg), freqs, pos, q, qo, ld, ldo, heads, k, ko, 128, 128, 2, t, dt)
    for kw in (dict(freqs=None), dict(pos=None), dict(qo=None), dict(ld=127), dict(ldo=127), dict(dt=3), dict(k=P), dict(heads=65537), dict(t=1 << 31)):
        assert go(**kw) == INVALID, kw
    assert go(t=0) == 0 and go(q=None, qo=None) == 0              # no work, no device
    ap = lambda k=P, v=P, ldk=128, ldv=128, rope=None, f=None, q=None, qo=None, ldq=0, nq=0: lib.b200_paged_append(  # noqa: E731
        ctx, C.byref(cache()), C.byref(batch()), k, v, ldk, ldv, rope, f, q, qo, ldq, ldq, nq)
    for kw in (dict(k=None), dict(v=None), dict(ldk=127), dict(ldv=1), dict(q=P), dict(qo=P), dict(q=P, qo=P, ldq=127, nq=2), dict(rope=C.byref(cfg)),
               dict(rope=C.byref(bridge.RopeConfig.make(128)), f=P)):
        assert ap(**kw) == INVALID, kw


@pytest.mark.parametrize("kw", [dict(logits=None), dict(u=None), dict(tok=None), dict(V=0), dict(V=(1 << 24) + 1, ld=1 << 25), dict(ld=7), dict(dt=2), dict(B=(1 << 24) + 1)])
def test_bad_sampling_calls(lib, ctx, kw):
    a = {**dict(logits=P, dt=0, B=2, V=8, ld=8, u=P, tok=P), **kw}
    assert lib.b200_sample_given(ctx, a["logits"], a["dt"], a["B"], a["V"], a["ld"], None, None, None, None, a["u"], a["tok"], None, None) == INVALID


# ---- the batch checks that the kernels make ------------------------------------------------------------------------------
def probe(lib, q_start, kv_len, table, rows, max_q, n_pages, page):
    """(largest row + 1, largest slot + 1, status) that the kernels' own index code reaches for this batch."""
    fn = lib.b200_internal_paged_probe
    fn.argtypes, fn.restype = [C.c_void_p] * 2 + [C.POINTER(C.c_longlong)], C.c_int
    arr = [np.ascontiguousarray(x, np.int32) for x in (q_start, kv_len, table)]
    c = cache(n_pages=n_pages, page_size=page, n_kv=1, head_dim=1, head_stride=1, token_stride=1, page_stride=page)
    b = bridge._PagedBatch(*[x.ctypes.data for x in arr], arr[1].size, arr[2].shape[1], rows, max_q)
    out = (C.c_longlong * 5)()
    assert fn(C.byref(c), C.byref(b), out) == 0
    return list(out)


def test_good_batches_reach_exactly_their_rows_and_slots(lib):
    r = probe(lib, [0, 1, 4], [5, 20], [[0, -1], [1, 2]], 4, 3, 3, 16)
    assert r == [4, 36, 0, 0, 0]                                  # rows 0..3, slots of pages 0, 1, 2 up to position 19, nothing below 0, status 0


@pytest.mark.parametrize("q_start,kv_len,table", [([0, 1, 4], [5, 20], [[7, -1], [1, 2]]), ([0, 1, 4], [5, 20], [[-1, -1], [1, 2]]), ([0, 1, 4], [5, 99], [[0, 1], [1, 2]]),
                                                  ([0, 1, 9], [5, 20], [[0, 1], [1, 2]]), ([-3, 1, 4], [5, 20], [[0, 1], [1, 2]]), ([0, 4, 1], [5, 20], [[0, 1], [1, 2]]),
                                                  ([0, 1, 4], [-5, 20], [[0, 1], [1, 2]]), ([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 1], [2 ** 31 - 1, -2 ** 31], [[2 ** 31 - 1, -2 ** 31], [3, 3]]),
                                                  ([0, 4, 4], [5, 20], [[0, 1], [1, 2]])])
def test_bad_batches_stay_inside_and_are_recorded(lib, q_start, kv_len, table):
    rows_end, slots_end, row_low, slot_low, status = probe(lib, q_start, kv_len, table, 4, 3, 3, 16)
    assert rows_end <= 4 and slots_end <= 48 and row_low >= 0 and slot_low >= 0
    assert status == 3


def test_random_tables_stay_inside(lib):
    r = np.random.RandomState(0)
    for _ in range(200):
        n, w, page, n_pages, rows = r.randint(1, 6), r.randint(1, 5), r.randint(1, 40), r.randint(1, 9), r.randint(1, 50)
        out = probe(lib, r.randint(-60, 120, n + 1), r.randint(-50, 300, n), r.randint(-3, 14, (n, w)), rows, r.randint(1, 60), n_pages, page)
        assert out[0] <= rows and out[1] <= n_pages * page and out[2] >= 0 and out[3] >= 0


# ---- the division of the work ------------------------------------------------------------------------------------------
def cover(lib, q_lens, kv_lens, n_kv, G, few, n_cta, min_units):
    """Every (sequence, KV head, block, tile) that the CTAs' runs visit, by the kernels' own stepping."""
    fn = lib.b200_internal_paged_cover
    fn.argtypes, fn.restype = [C.c_void_p] * 2 + [C.c_int] * 9 + [C.c_void_p, C.c_longlong], C.c_longlong
    q_start = np.concatenate(([0], np.cumsum(q_lens))).astype(np.int32)
    kv, table = np.array(kv_lens, np.int32), np.zeros((len(kv_lens), max(1, max(kv_lens))), np.int32)
    c = cache(n_pages=1, page_size=1, n_kv=n_kv, head_dim=1, head_stride=1, token_stride=1, page_stride=1)
    b = bridge._PagedBatch(q_start.ctypes.data, kv.ctypes.data, table.ctypes.data, kv.size, table.shape[1], int(q_start[-1]), 0)
    out = np.empty((200000, 7), np.int32)
    n = fn(C.byref(c), C.byref(b), G, few["tokens"], few["rows"], int(np.log2(few["tile"])), few["extra"], few["lo"], few["hi"], n_cta, min_units, out.ctypes.data, len(out))
    assert 0 <= n <= len(out)
    return out[:n]


@pytest.mark.parametrize("seed", range(30))
def test_runs_cover_every_tile_once(lib, seed):
    r = np.random.RandomState(seed)
    n, G, n_kv = r.randint(1, 9), int(r.choice([1, 2, 3, 4, 8, 40])), int(r.randint(1, 4))
    kv = r.randint(0, 900, n)
    q = np.minimum(np.where(r.rand(n) < 0.5, r.randint(0, 3, n), r.randint(0, 200, n)), kv + 3)
    by_rows = seed % 2
    plan = dict(extra=int(r.choice([0, 1, 3])), tokens=0 if by_rows else int(r.choice([2, 64, 128])), rows=32 if by_rows else 0, tile=int(r.choice([16, 32, 128])), lo=int(r.choice([0, 17])), hi=int(r.choice([16, 1 << 30])))
    got = cover(lib, q.tolist(), kv.tolist(), n_kv, G, plan, int(r.choice([1, 5, 148, 296])), int(r.choice([1, 4])))
    want = set()
    for s in range(n):
        if q[s] == 0 or not plan["lo"] <= q[s] * G <= plan["hi"]:
            continue
        blocks = -(-q[s] * G // 32) if by_rows else -(-q[s] // plan["tokens"])
        for b in range(blocks):
            last = min(q[s] - 1, ((b + 1) * 32 - 1) // G) if by_rows else min(q[s], (b + 1) * plan["tokens"]) - 1
            seen = min(max(kv[s] - q[s] + last + 1, 0), kv[s])
            for t in range(max(1, -(-seen // plan["tile"]))):
                want.update((s, h, b, t) for h in range(n_kv))
    seen_ = [tuple(x[1:5]) for x in got.tolist()]
    assert len(seen_) == len(set(seen_)) and set(seen_) == want
    # equal runs: tiles and the blocks' extra units of a CTA, up to the extra of a block at either end
    cost, blocks, joined = {}, {}, {}
    for ct, sq, h, b, t, whole, parts in got.tolist():
        cost.setdefault(ct, [0, set()])
        cost[ct][0] += 1
        cost[ct][1].add((sq, h, b))
        blocks.setdefault((sq, h, b), []).append((ct, t, whole))
        joined[ct] = parts
    per = [n + plan["extra"] * len(bl) for n, bl in cost.values()]
    assert not per or max(per) - min(per) <= 2 * plan["extra"] + 1 or len(per) < 2 or max(per) <= -(-sum(per) // len(per)) + 2 * plan["extra"] + 1
    # a block's CTAs follow each other; the second of them, and no other CTA, joins all of them
    second = {}
    for key, xs in blocks.items():
        ctas = sorted({x[0] for x in xs})
        assert ctas == list(range(ctas[0], ctas[-1] + 1))
        assert all(bool(x[2]) == (len(ctas) == 1) for x in xs)
        if len(ctas) > 1:
            second[ctas[1]] = len(ctas)
    assert {ct: n for ct, n in joined.items() if n} == second
