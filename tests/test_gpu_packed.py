"""Operators over packed runs (several new tokens per sequence of a paged cache), verification of drafted tokens, pages that are handed on:
each against a plain 64-bit computation, and all of them together as one decoding loop."""
import numpy as np
import pytest

import packed_cases as R

pytestmark = pytest.mark.gpu

KV = {"f32": 0, "f16": 1, "q8_0": 2}
EPS, THETA = 1e-6, 1e6


@pytest.fixture(scope="module")
def B():
    import brasa_b200
    return brasa_b200


@pytest.fixture(scope="module")
def ctx(B):
    c = B.Context(0)
    yield c
    c.close()


@pytest.fixture(scope="module")
def K(B, ctx):
    return B.Kernels(ctx)


def go(ctx, f):
    cmd = ctx.command()
    try:
        f(cmd)
    finally:
        cmd.wait()


class OnDevice:
    """A Run in device buffers."""

    def __init__(self, ctx, K, run, longest=None, tokens=None, starts=None):
        self.run = run
        self.bufs = [ctx.buffer_from(x) for x in (run.k, run.v, run.table, run.lens, run.starts if starts is None else np.array(starts, np.uint32), run.q)]
        k, v, t, n, s, self.q = self.bufs
        self.kpool, self.vpool = k, v
        self.paged = K.paged_kv(k, v, t, n, len(run.seqs), run.max_pages, run.num_pages, KV[run.kv])
        self.packed = K.packed_run(s, tokens or run.tokens, longest or run.longest)

    def free(self):
        for b in self.bufs:
            b.free()


def attend(ctx, K, run, half, **kw):
    dev = OnDevice(ctx, K, run, **kw)
    n = run.tokens * run.hq * 128
    o = ctx.buffer(n * (2 if half else 4))
    o.fill(0x3C)
    go(ctx, lambda c: K.attention_packed(c, dev.q, dev.paged, dev.packed, o, run.hq, run.hkv, 0 if half else 1))
    got = o.download(np.float16 if half else np.float32).astype(np.float64).reshape(run.tokens, run.hq, 128)
    untouched = np.frombuffer(b"\x3c" * 4, np.float16 if half else np.float32)[0].astype(np.float64)
    o.free()
    dev.free()
    return got, untouched


def check(got, want, tol):
    off = np.abs(got - want)
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(off - tol), off.shape)
    assert (off <= tol).all(), (worst, got[worst], want[worst], tol[worst])


SHAPES = {
    "one": [(1, 0)],
    "one-deep": [(1, 700)],
    "page-ends": [(1, 15), (1, 16), (1, 17), (2, 14), (16, 0), (17, 0), (15, 1), (1, 127), (1, 128), (129, 0)],
    "drafts": [(5, 130), (1, 63), (3, 300), (0, 40), (4, 0), (5, 511), (2, 64)],
    "prompts": [(70, 0), (1, 0), (200, 33), (0, 0), (129, 250)],
    "mixed": [(150, 100), (1, 400), (3, 90), (260, 0), (1, 0)],
}


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("q8_0", False), ("f32", False), ("f32", True)])
def test_attention(ctx, K, kv, half, shape):
    run = R.Run(SHAPES[shape], 8, 2, kv, seed=len(shape), spare_tokens=3)
    got, untouched = attend(ctx, K, run, half)
    want, tol = run.attention(half)
    n = int(run.starts[-1])
    check(got[:n], want[:n], tol[:n])
    assert (got[n:] == untouched).all()  # rows behind the last sequence


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (5, 1), (8, 1), (6, 2), (7, 7), (14, 2), (16, 8)])
@pytest.mark.parametrize("kv,half", [("f16", True), ("q8_0", False), ("q8_0", True), ("f32", False)])
def test_attention_head_layouts(ctx, K, kv, half, hq, hkv):
    run = R.Run([(3, 70), (75, 20), (1, 200), (18, 0)], hq, hkv, kv, seed=hq)
    want, tol = run.attention(half)
    check(attend(ctx, K, run, half)[0], want, tol)


@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("f32", False)])
def test_attention_large_scores(ctx, K, kv, half):
    """Scores far apart: the running maximum moves often, and what it leaves underflows."""
    run = R.Run([(2, 500), (140, 90)], 4, 2, kv, seed=9, scale=12.0)
    want, tol = run.attention(half)
    check(attend(ctx, K, run, half)[0], want, tol)


@pytest.mark.parametrize("n", [6000, 32000])
@pytest.mark.parametrize("kv", ["f16", "q8_0", "f32"])
def test_attention_small_weights_count(ctx, K, kv, n):
    """F32 precision: one key 18 nats above all others, whose weights are near 2^-26 each and a hundredth of a percent and more together. 300 sequences over the same
    pages, so that a block has whole rows.
    A weight is off by 2^-19 of itself at most (its exponential and the step's, terms of 2^-22, sums of sixteen); the sums in 32 bits round once for every 16 keys
    and part, 2^-24 of what they hold: 2^-24 (n / 16 + 40) of sum p |v|."""
    S, hq = 300, 4
    run = R.Run([(1, n - 1)], hq, 1, kv, seed=61)
    g = np.random.default_rng(62)
    u = g.standard_normal(128)
    u /= np.linalg.norm(u)
    k, v = 0.05 * g.standard_normal((n, 1, 128)), 1.0 + 0.1 * g.standard_normal((n, 1, 128))
    k[5, 0], v[5, 0] = 12.8 * u, -1.0
    for pool, x in ((run.k, k), (run.v, v)):
        rows = R.to_bytes(x.astype(np.float32), kv)
        for i in range(n):
            pool[run.table[0, i // R.PAGE], i % R.PAGE] = rows[i]
    run.seqs, run.tokens = [(1, n - 1)] * S, S
    run.table, run.lens, run.starts = np.repeat(run.table, S, 0), np.repeat(run.lens, S), np.arange(S + 1, dtype=np.uint32)
    run.q = (16 * u + 0.3 * g.standard_normal((S, hq, 128))).astype(np.float32)
    got, _ = attend(ctx, K, run, False)
    kk, vv = (run.rows(pool, 0, n)[0][:, 0] for pool in (run.k, run.v))
    for t in range(0, S, 13):
        for h in range(hq):
            q = run.q[t, h].astype(np.float64)
            a = kk @ q / np.sqrt(128)
            p = np.exp(a - a.max())
            p /= p.sum()
            o = p @ vv
            ds = 2.0 ** -22 * 130 * (np.abs(kk) @ np.abs(q)).max() / np.sqrt(128)
            check(got[t, h], o, ds * (p @ np.abs(vv - o)) + (2.0 ** -19 + 2.0 ** -24 * (n / 16 + 40)) * (p @ np.abs(vv)))


@pytest.mark.parametrize("new", [1, 9])
@pytest.mark.parametrize("kv", ["f16", "q8_0"])
def test_attention_small_weights_count_in_f16(ctx, K, kv, new):
    """F16 precision, the same: weights near 2^-26 of the largest are off by half of f16's last step, 2^-25, under a factor of 2^7 at least, so 2^-32 of the largest each.
    Beside that what F16 precision rounds (see Run.attention), with half a step of o below 1, 2^-12."""
    n, S, hq = 32000, 100, 4
    run = R.Run([(new, n - new)], hq, 1, kv, seed=64)
    g = np.random.default_rng(65)
    u = g.standard_normal(128)
    u /= np.linalg.norm(u)
    k, v = 0.05 * g.standard_normal((n, 1, 128)), 0.95 + 0.04 * g.standard_normal((n, 1, 128))
    k[5, 0], v[5, 0] = 12.8 * u, -0.95
    for pool, x in ((run.k, k), (run.v, v)):
        rows = R.to_bytes(x.astype(np.float32), kv)
        for i in range(n):
            pool[run.table[0, i // R.PAGE], i % R.PAGE] = rows[i]
    run.seqs, run.tokens = [(new, n - new)] * S, S * new
    run.table, run.lens, run.starts = np.repeat(run.table, S, 0), np.repeat(run.lens, S), np.arange(0, S * new + 1, new, dtype=np.uint32)
    run.q = (16 * u + 0.3 * g.standard_normal((S * new, hq, 128))).astype(np.float32)
    got, _ = attend(ctx, K, run, True)
    kk, vv = (run.rows(pool, 0, n)[0][:, 0] for pool in (run.k, run.v))
    for t in range(0, S * new, 29):
        for h in range(hq):
            see = n - new + t % new + 1
            q = run.q[t, h].astype(np.float64)
            a = kk[:see] @ q / np.sqrt(128)
            p = np.exp(a - a.max())
            p /= p.sum()
            o = p @ vv[:see]
            off = np.abs(vv[:see] - o)
            spread = p @ off
            dq = 6 * 2.0 ** -11 / np.sqrt(3) * np.sqrt((kk ** 2) @ (q ** 2)).max() / np.sqrt(128) * (np.sqrt(2) if kv == "q8_0" else 1)
            tol = (dq + 2.0 ** -11) * spread + 2.0 ** -32 * off.sum(0) + 2.0 ** -12 + 2.0 ** -22 * (see / 16 + 200)
            if kv == "q8_0":
                tol = tol + 2.0 ** -12  # (the dominant value's own rounding, below 1)
            check(got[t, h], o, tol)


@pytest.mark.parametrize("q,k", [(1e5, 1e-4), (1e-5, 1e4), (1e-30, 1.0), (1e30, 0.0)])
@pytest.mark.parametrize("kv", ["f16", "q8_0", "f32"])
def test_attention_queries_of_any_size(ctx, K, kv, q, k):
    """F32 precision: queries beyond f16's range and in its last bits."""
    run = R.Run([(5, 130), (1, 600), (40, 20)], 4, 2, kv, seed=63, scale=q)
    real = ~np.isnan(R.from_bytes(run.k, kv)).any(-1, keepdims=True)
    run.k = np.where(real, R.to_bytes(np.where(real, k * R.from_bytes(run.k, kv), 0).astype(np.float32), kv), run.k)
    run.q[1, 2, 3:] *= 1e-7  # (a row whose values lie far apart)
    want, tol = run.attention(False)
    check(attend(ctx, K, run, False)[0], want, tol)


@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("f32", False)])
def test_attention_positions_without_pages(ctx, K, kv, half):
    """Pages that are none stand for positions that hold nothing; a row that sees nothing gives zeros."""
    run = R.Run([(4, 60), (100, 150), (2, 20), (140, 0)], 4, 2, kv, seed=3)
    run.table[0, 1], run.table[1, 0], run.table[1, 9], run.table[1, 15] = -1, run.num_pages, -7, 2 ** 31 - 1
    run.table[2, :] = -1
    run.table[3, :8] = -1
    want, tol = run.attention(half)
    got, _ = attend(ctx, K, run, half)
    check(got, want, tol)
    a, b = int(run.starts[2]), int(run.starts[3])
    assert (got[a:b] == 0).all() and (got[b:b + 128] == 0).all()


@pytest.mark.parametrize("bad", ["nan", "inf in v", "inf in k"])
@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("q8_0", False), ("f32", False), ("f32", True)])
def test_attention_rows_before_a_bad_one(ctx, K, kv, half, bad):
    """A token whose key or value is not finite counts for its own row and those behind it, never for a row before it: one piece of the work or several,
    few rows and many."""
    run = R.Run([(5, 130), (3, 0), (4, 3000), (200, 33), (129, 250), (150, 2200)], 4, 2, kv, seed=21)
    want, tol = run.attention(half)
    first = [3, 1, 2, 150, 128, 60]  # of each sequence's new tokens, the bad one
    for s, j in enumerate(first):
        at = int(run.lens[s]) + j
        row = np.full((run.hkv, R.D), np.nan if bad == "nan" else np.inf, np.float32)
        if kv == "q8_0":  # (codes of 1 under a scale that is not finite)
            raw = np.concatenate([np.ones((run.hkv, 128), np.uint8), row[:, :4].astype(np.float16).view(np.uint8)], -1)
        else:
            raw = R.to_bytes(row, kv)
        for pool in (run.k, run.v):
            if bad == "nan" or (bad == "inf in v") == (pool is run.v):
                pool[run.table[s, at // R.PAGE], at % R.PAGE] = raw
    got, _ = attend(ctx, K, run, half)
    for s, j in enumerate(first):
        a, b, e = int(run.starts[s]), int(run.starts[s]) + j, int(run.starts[s + 1])
        check(got[a:b], want[a:b], tol[a:b])
        if bad != "inf in k":
            assert not np.isfinite(got[b:e]).any()


@pytest.mark.parametrize("bad", ["k", "v"])
@pytest.mark.parametrize("kv", ["f16", "q8_0"])
def test_attention_many_short_items_behind_a_bad_one(ctx, K, kv, bad):
    """An item of two row tiles whose second holds a value that is not finite, and more short items behind it in the same block's share of the work than the
    block hands on at a time: every other sequence has the bits of the run without that value."""
    seqs = [(60, 2000)] + [(9, 0)] * 2400  # 240 rows, then 36 each
    run = R.Run(seqs, 8, 2, kv, seed=51)
    clean, _ = attend(ctx, K, run, True)
    tall, last = 60, [1, 9, 700, 2400]
    run.seqs = [x if s == 0 or s in last else (0, x[1]) for s, x in enumerate(seqs)]
    want, tol = run.attention(True)
    for s in [0] + last:
        a, b = int(run.starts[s]), int(run.starts[s + 1])
        check(clean[a:b], want[a:b], tol[a:b])
    j = 33 if bad == "k" else 59  # (rows 132 and on; all rows before the last token)
    row = np.full((2, R.D), np.inf, np.float32)
    raw = R.to_bytes(row, kv) if kv == "f16" else np.concatenate([np.ones((2, 128), np.uint8), row[:, :4].astype(np.float16).view(np.uint8)], -1)
    (run.k if bad == "k" else run.v)[run.table[0, (2000 + j) // R.PAGE], (2000 + j) % R.PAGE] = raw
    got, _ = attend(ctx, K, run, True)
    check(got[:j], want[:j], tol[:j])
    assert (got[tall:] == clean[tall:]).all()


def put_row(run, pool, s, at, row):
    """One position's row of all key heads, f32 [hkv, 128]; in 8 bits values that are not finite are codes of 1 under such a scale, others codes of 100."""
    if run.kv == "q8_0":
        block = row.reshape(run.hkv, 4, 32)[:, :, 0]
        odd = ~np.isfinite(block)
        raw = np.concatenate([np.repeat(np.where(odd, 1, 100), 32, -1).astype(np.uint8), np.where(odd, block, block / 100).astype(np.float16).view(np.uint8).reshape(run.hkv, 8)], -1)
    else:
        raw = R.to_bytes(row, run.kv)
    pool[run.table[s, at // R.PAGE], at % R.PAGE] = raw


@pytest.mark.parametrize("where", ["first", "every"])
@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("q8_0", False), ("f32", False)])
def test_attention_a_bad_value_that_all_rows_see(ctx, K, kv, half, where):
    """A NaN at the first position, or at every new one, makes the rows NaN that see it, and the call takes no longer for it than a call takes."""
    run = R.Run([(500, 6000), (2, 50)], 8, 2, kv, seed=52)
    seqs = run.seqs
    run.seqs = [(0, 0), seqs[1]]
    want, tol = run.attention(half)
    run.seqs = seqs
    row = np.full((2, R.D), np.nan, np.float32)
    times = []
    for bad in (False, True):
        if bad:
            for j in [0] if where == "first" else range(6000, 6500):
                put_row(run, run.k, 0, j, row)
                put_row(run, run.v, 0, j, row)
        dev = OnDevice(ctx, K, run)
        o = ctx.buffer(run.tokens * 8 * 128 * 4)
        took = []
        for _ in range(4):
            cmd = ctx.command()
            K.attention_packed(cmd, dev.q, dev.paged, dev.packed, o, 8, 2, 0 if half else 1)
            took.append(cmd.wait())
        times.append(min(took))
        got = o.download(np.float16 if half else np.float32)[:run.tokens * 8 * 128].astype(np.float64).reshape(run.tokens, 8, 128)
        o.free()
        dev.free()
    assert np.isnan(got[:500]).all()
    check(got[500:], want[500:], tol[500:])
    assert times[1] < 2 * times[0] + 2e-4, times


@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("q8_0", False), ("f32", False), ("f32", True)])
def test_attention_bad_values_dim_by_dim(ctx, K, kv, half):
    """NaN in 32 dims of one token, infinities in 32 other dims of a later one: of the rows between them only the first dims are NaN; a row before both has neither."""
    run = R.Run([(150, 700), (6, 1500)], 4, 2, kv, seed=53)
    want, tol = run.attention(half)
    for s, (first, then) in enumerate(((40, 120), (2, 4))):
        for j, dims, value in ((first, slice(0, 32), np.nan), (then, slice(64, 96), np.inf)):
            at = int(run.lens[s]) + j
            row = np.array(R.from_bytes(run.v[run.table[s, at // R.PAGE], at % R.PAGE], kv), np.float32)
            row[:, dims] = value
            if kv == "q8_0":  # (the other dims as they are)
                raw = run.v[run.table[s, at // R.PAGE], at % R.PAGE]
                raw[:, dims] = 1
                raw[:, 128:].view(np.float16)[:, dims.start // 32] = value
            else:
                put_row(run, run.v, s, at, row)
    got, _ = attend(ctx, K, run, half)
    for s, (first, then) in enumerate(((40, 120), (2, 4))):
        a, n = int(run.starts[s]), run.seqs[s][0]
        check(got[a:a + first], want[a:a + first], tol[a:a + first])
        assert np.isnan(got[a + first:a + n, :, :32]).all()
        check(got[a + first:a + then, :, 32:], want[a + first:a + then, :, 32:], tol[a + first:a + then, :, 32:])
        for d in (slice(32, 64), slice(96, 128)):
            check(got[a + then:a + n, :, d], want[a + then:a + n, :, d], tol[a + then:a + n, :, d])
        assert not np.isfinite(got[a + then:a + n, :, 64:96]).any()


@pytest.mark.parametrize("seqs", [[(1, 300)], [(6, 90), (1, 2000)], [(70, 30)]])
@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("q8_0", False), ("f32", False), ("f32", True)])
def test_attention_infinities_that_a_row_sees(ctx, K, kv, half, seqs):
    """An infinity of V at an old position makes its dims that infinity, of both signs NaN; in 8 bits a block of 32 dims."""
    run = R.Run(seqs, 6, 2, kv, seed=59)
    want, tol = run.attention(half)
    at = seqs[0][1] // 2
    for j, dims, values in ((at, slice(32, 64), (np.inf, -np.inf)), (at + 1, slice(64, 96), (-np.inf, np.inf)), (at + 2, slice(64, 96), (-np.inf, -np.inf))):
        for h in range(2):
            raw = run.v[run.table[0, j // R.PAGE], j % R.PAGE, h]
            if kv == "q8_0":
                raw[dims] = 1
                raw[128:].view(np.float16)[dims.start // 32] = values[h]
            else:
                raw.view(np.float16 if kv == "f16" else np.float32)[dims] = values[h]
    got, _ = attend(ctx, K, run, half)
    n = seqs[0][0]
    for d in (slice(0, 32), slice(96, 128)):
        check(got[:n, :, d], want[:n, :, d], tol[:n, :, d])
    assert (got[:n, :3, 32:64] == np.inf).all() and (got[:n, 3:, 32:64] == -np.inf).all()
    assert (got[:n, :3, 64:96] == -np.inf).all() and np.isnan(got[:n, 3:, 64:96]).all()
    if len(seqs) > 1:
        check(got[n:], want[n:], tol[n:])


@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("f32", False), ("f32", True)])
def test_attention_infinite_keys(ctx, K, kv, half):
    """An infinity in one dim of old keys: a row whose query is negative there has scores of minus infinity and attends to the others, any other row is NaN."""
    run = R.Run([(3, 200), (40, 60), (1, 1500)], 8, 2, kv, seed=60)
    for s in range(3):
        run.k[run.table[s, 2]].reshape(16, 2, -1).view(np.float16 if kv == "f16" else np.float32)[:, :, 7] = np.inf
    table = run.table.copy()
    run.table[:, 2] = -1
    want, tol = run.attention(half)
    run.table = table
    got, _ = attend(ctx, K, run, half)
    down = run.q[:, :, 7] < 0
    check(got[down], want[down], tol[down])
    assert np.isnan(got[~down]).all()


@pytest.mark.parametrize("seqs", [[(500, 6000), (2, 50)], [(1200, 0), (1, 700)], [(7, 900)]])
@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("q8_0", False), ("f32", False)])
def test_attention_a_channel_that_overflows(ctx, K, kv, half, seqs):
    """Infinities in the last 32 dims of every new token of the first sequence, of the other sign from the fifth on, and a NaN key in its second but last: the rows are
    infinite there, then NaN, the last two NaN throughout, all else as without. The call takes no longer for it than a call takes."""
    run = R.Run(seqs, 4, 2, kv, seed=55)
    n, past = seqs[0]
    times = []
    for bad in (False, True):
        if bad:
            for j in range(n):
                raw = run.v[run.table[0, (past + j) // R.PAGE], (past + j) % R.PAGE]
                value = np.inf if j < 4 else -np.inf
                if kv == "q8_0":
                    raw[:, 96:128] = 1
                    raw[:, 128:].view(np.float16)[:, 3] = value
                else:
                    raw.view(np.float16 if kv == "f16" else np.float32)[:, 96:] = value
            put_row(run, run.k, 0, past + n - 2, np.full((2, R.D), np.nan, np.float32))
        dev = OnDevice(ctx, K, run)
        o = ctx.buffer(run.tokens * 4 * 512)
        took = []
        for _ in range(4):
            cmd = ctx.command()
            K.attention_packed(cmd, dev.q, dev.paged, dev.packed, o, 4, 2, 0 if half else 1)
            took.append(cmd.wait())
        times.append(min(took))
        got = o.download(np.float16 if half else np.float32)[:run.tokens * 4 * 128].astype(np.float64).reshape(run.tokens, 4, 128)
        if not bad:
            clean = got
        o.free()
        dev.free()
    rest = np.delete(np.arange(run.tokens), [n - 2, n - 1])
    assert (got[rest, :, :96] == clean[rest, :, :96]).all() and (got[n:] == clean[n:]).all()
    assert (got[:4, :, 96:] == np.inf).all() and np.isnan(got[4:n, :, 96:]).all() and np.isnan(got[n - 2:n]).all()
    assert times[1] < 2 * times[0] + 2e-4, times


@pytest.mark.parametrize("shape", [[(6, 40)], [(60, 900)]])
def test_attention_8_bit_values_past_f16(ctx, K, shape):
    """A new token's value that is finite in 8 bits and infinite in f16, as the products of F16 precision round it, does not reach the rows before it."""
    run = R.Run(shape, 8, 2, "q8_0", seed=54)
    want, tol = run.attention(True)
    n, past = shape[0]
    at = past + n - 2
    put_row(run, run.v, 0, at, np.full((2, R.D), 1e5, np.float32))
    got, _ = attend(ctx, K, run, True)
    check(got[:n - 2], want[:n - 2], tol[:n - 2])


def test_attention_keeps_to_what_the_call_says(ctx, K):
    """`longest` and `tokens` below what starts say, starts that fall, positions behind the table: such rows are left alone."""
    run = R.Run([(3, 40), (150, 20), (2, 30)], 4, 2, "f16", seed=5)
    want, tol = run.attention(True)
    got, untouched = attend(ctx, K, run, True, longest=20)
    check(got[:23], want[:23], tol[:23])
    assert (got[23:153] == untouched).all()
    check(got[153:], want[153:], tol[153:])
    got, _ = attend(ctx, K, run, True, tokens=10)
    check(got[:10], want[:10], tol[:10])
    assert (got[10:] == untouched).all()
    got, _ = attend(ctx, K, run, True, starts=[0, 3, 1, 155])
    check(got[:1], want[:1], tol[:1])
    run = R.Run([(20, 10)], 4, 2, "f16", seed=6)
    want, tol = run.attention(True)
    run.table, run.max_pages = np.ascontiguousarray(run.table[:, :1]), 1
    got, _ = attend(ctx, K, run, True)
    check(got[:6], want[:6], tol[:6])
    assert (got[6:] == untouched).all()


def test_attention_of_a_single_token_is_the_paged_one(ctx, K):
    """One token per sequence: what brasa_k_decode_attention_paged gives, to the rounding of its sums."""
    import brasa_b200 as B
    run = R.Run([(1, 90), (1, 300), (1, 0)], 8, 2, "f16", seed=8)
    dev = OnDevice(ctx, K, run)
    o, o2 = ctx.buffer(3 * 8 * 512), ctx.buffer(3 * 8 * 512)
    part = ctx.buffer(B.decode_partials_len(8, run.max_pages * 16) * 3 * 4)
    go(ctx, lambda c: (K.attention_packed(c, dev.q, dev.paged, dev.packed, o, 8, 2, 1), K.decode_attention_paged(c, dev.q, dev.paged, part, o2, 8, 2)))
    want, tol = run.attention(False)
    check(o.download(np.float32).reshape(3, 8, 128).astype(np.float64), want, tol)
    check(o2.download(np.float32).reshape(3, 8, 128).astype(np.float64), want, tol)
    dev.free()


def test_attention_long_cache(ctx, K):
    """One drafting sequence behind 20 000 positions, and two short ones: work of one item over many blocks."""
    run = R.Run([(4, 20000), (1, 3), (2, 500)], 4, 1, "f16", seed=10)
    for half in (True, False):
        want, tol = run.attention(half)
        check(attend(ctx, K, run, half)[0], want, tol)


@pytest.mark.parametrize("kv,half", [("f16", True), ("f16", False), ("q8_0", True), ("f32", False)])
def test_pages_behind_4_gib(B, ctx, K, kv, half):
    """The store, the attention and the page operators on pages whose offsets pass 32 bits: the bits of the same run in a small pool."""
    run = R.Run([(40, 30), (3, 200), (1, 0)], 16, 8, kv, seed=57)
    page = 16 * 8 * R.ROW[kv]
    num = 2 ** 32 // page + 2 * run.num_pages
    first = num - run.num_pages
    small = OnDevice(ctx, K, run)
    kpool, vpool = ctx.buffer(num * page), ctx.buffer(num * page)
    kpool.upload(run.k, first * page), vpool.upload(run.v, first * page)
    table = ctx.buffer_from((run.table + first).astype(np.int32))
    far = K.paged_kv(kpool, vpool, table, small.bufs[3], 3, run.max_pages, num, KV[kv])
    g = np.random.default_rng(58)
    k, v = (ctx.buffer_from(g.standard_normal((run.tokens, 8, 128)).astype(np.float32)) for _ in range(2))
    norm, rope = ctx.buffer_from(np.ones(128, np.float32)), B.RopeTable(ctx, THETA, 128, run.max_pages * 16)
    n = run.tokens * 16 * 128
    got = []
    for paged, pools, at in ((small.paged, (small.kpool, small.vpool), 0), (far, (kpool, vpool), first * page)):
        q, o = ctx.buffer(n * 4), ctx.buffer(n * 4)
        go(ctx, lambda c: K.qk_norm_rope_store_packed(c, small.q, k, v, norm, norm, EPS, rope, paged, small.packed, q, 16, 8))
        go(ctx, lambda c: K.attention_packed(c, q, paged, small.packed, o, 16, 8, 0 if half else 1))
        got.append([q.download(np.uint32), o.download(np.uint32)] + [p.download(np.uint8, run.k.size, at) for p in pools])
        q.free(), o.free()
    assert all((a == b).all() for a, b in zip(*got))
    result, moved, out = ctx.buffer(16), ctx.buffer(num * 4), ctx.buffer(run.table.nbytes)
    pool = K.page_pool(kpool, vpool, table, small.bufs[3], None, 3, run.max_pages, num, 1, 8, KV[kv])
    go(ctx, lambda c: K.pages_compact(c, pool, out, moved, result))  # (pages that the table names are entries of any page: those of no sequence too)
    want, to, counts, moves = R.compact(run.table + first, None, num)
    assert (out.download(np.int32).reshape(want.shape) == want).all() and list(result.download(np.uint32)) == counts and len(moves) == counts[1] > 0
    for p, was in zip((kpool, vpool), got[0][2:]):
        was = was.reshape(run.k.shape)
        for a, b in moves:
            assert (p.download(np.uint8, page, b * page) == was[a - first].reshape(-1)).all()
    for b in (kpool, vpool, table, k, v, norm, result, moved, out):
        b.free()
    small.free()


def test_attention_many_sequences(ctx, K):
    """More sequences than a warp has lanes, most without new tokens."""
    g = np.random.default_rng(2)
    seqs = [(int(n), int(p)) for n, p in zip(g.integers(0, 3, 1100) * (g.random(1100) < 0.2), g.integers(0, 40, 1100))]
    seqs[0], seqs[500], seqs[-1] = (0, 5), (90, 7), (3, 2)
    run = R.Run(seqs, 2, 1, "f16", seed=11, spare_tokens=1)
    want, tol = run.attention(True)
    got, untouched = attend(ctx, K, run, True)
    check(got[:-1], want[:-1], tol[:-1])
    assert (got[-1] == untouched).all()


def test_attention_repeats_and_replays(B, ctx, K):
    """The same bits again, and out of a recorded graph with new lengths and tables behind it."""
    run, other = R.Run([(130, 40), (2, 300), (5, 90)], 8, 2, "f16", seed=12), R.Run([(100, 70), (30, 272), (7, 88)], 8, 2, "f16", seed=13)
    assert run.tokens == other.tokens and run.max_pages >= other.max_pages
    dev = OnDevice(ctx, K, run)
    o = ctx.buffer(run.tokens * 8 * 256)
    go(ctx, lambda c: K.attention_packed(c, dev.q, dev.paged, dev.packed, o, 8, 2, 0))
    first = o.download(np.uint16)
    graph = ctx.capture(lambda c: K.attention_packed(c, dev.q, dev.paged, dev.packed, o, 8, 2, 0))
    for _ in range(2):
        o.fill(0)
        go(ctx, lambda c: graph.launch(c))
        assert (o.download(np.uint16) == first).all()
    table = np.zeros_like(run.table)
    table[:, :other.max_pages] = other.table
    big = other.num_pages <= run.num_pages
    assert big
    for buf, x in zip(dev.bufs, (other.k, other.v, table, other.lens, other.starts, other.q)):
        buf.upload(x)
    go(ctx, lambda c: graph.launch(c))
    want, tol = other.attention(True)
    check(o.download(np.float16).astype(np.float64).reshape(run.tokens, 8, 128), want, tol)
    graph.free()
    dev.free()


@pytest.mark.parametrize("kv", KV)
@pytest.mark.parametrize("hq,hkv", [(8, 2), (3, 1), (7, 7), (10, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_store(B, ctx, K, kv, hq, hkv, in_place):
    run = R.Run([(5, 30), (1, 0), (0, 9), (33, 15), (2, 4000)], hq, hkv, kv, seed=20, spare_tokens=2)
    run.table[3, 1] = -1  # positions 16 to 31 of that sequence have no place
    g = np.random.default_rng(21)
    k, v = (g.standard_normal((run.tokens, hkv, 128)).astype(np.float32) * 3 for _ in range(2))
    k[2], v[2] = 0, 0
    qn, kn = (1 + 0.2 * g.standard_normal(128).astype(np.float32) for _ in range(2))
    dev = OnDevice(ctx, K, run)
    gk, gv, gqn, gkn = (ctx.buffer_from(x) for x in (k, v, qn, kn))
    out = dev.q if in_place else ctx.buffer_from(np.full_like(run.q, 7.0))
    table = B.RopeTable(ctx, THETA, 128, run.max_pages * 16)
    go(ctx, lambda c: K.qk_norm_rope_store_packed(c, dev.q, gk, gv, gqn, gkn, EPS, table, dev.paged, dev.packed, out, hq, hkv))
    got_q = out.download(np.float32).reshape(run.q.shape)
    pools = [p.download(np.uint8).reshape(run.k.shape) for p in (dev.kpool, dev.vpool)]
    want = [run.k.copy(), run.v.copy()]
    written = np.zeros(run.k.shape[:2], bool)
    for s, (n, past) in enumerate(run.seqs):
        for j in range(n):
            t, pos = int(run.starts[s]) + j, past + j
            # 32-bit sums of 128 squares, a root, a product and two of the rotation, whose table is rounded to 2^-24: within 2^-20 of the row's largest
            wq, wk = R.norm_rope(run.q[t], qn, EPS, THETA, pos), R.norm_rope(k[t], kn, EPS, THETA, pos)
            assert np.abs(got_q[t] - wq).max() <= 2.0 ** -20 * np.abs(wq).max()
            page = run.table[s, pos // 16]
            if page < 0:
                continue
            written[page, pos % 16] = True
            gotk, gotv = (R.from_bytes(p[page, pos % 16], kv) for p in pools)
            # a rounding to the cache's type: half a step of the value, in 8 bits of the block's largest / 127 (and its scale's own rounding, 2^-11 of 127 steps)
            for got, w, exact in ((gotk, wk, False), (gotv, v[t].astype(np.float64), True)):
                block = np.repeat(np.abs(w).reshape(hkv, 4, 32).max(-1), 32, -1).reshape(hkv, 128)
                step = {"f32": 2.0 ** -24 * np.abs(w), "f16": 2.0 ** -11 * np.abs(w) + 2.0 ** -25, "q8_0": (0.5 / 127 + 2.0 ** -11) * block + 2.0 ** -24}[kv]
                assert (np.abs(got - w) <= step + (0 if exact else 2.0 ** -20) * block).all()
    for got, was in zip(pools, want):
        assert (got[~written] == was[~written]).all()
    n = int(run.starts[-1])
    assert (got_q[n:] == (run.q[n:] if in_place else 7.0)).all()


def random_verify(g, seqs, drafts, vocab, q_given, empty=0.0):
    n = [0 if g.random() < empty else int(g.integers(0, drafts + 1)) + 1 for _ in range(seqs)]
    starts = np.concatenate([[0], np.cumsum(n)]).astype(np.uint32)
    rows, nd = int(starts[-1]), int(sum(max(0, x - 1) for x in n))
    p = g.dirichlet(np.full(vocab, 0.3), rows).astype(np.float32) if rows else np.zeros((0, vocab), np.float32)
    q = g.dirichlet(np.full(vocab, 0.3), max(nd, 1)).astype(np.float32)
    d = np.array([g.integers(0, vocab) if not q_given else np.argmax(np.cumsum(q[i]) > g.random() * 0.999) for i in range(nd)], np.uint32)
    return p, q[:nd] if q_given else None, d, g.random(rows).astype(np.float32), starts


def run_verify(ctx, K, p, q, d, u, starts, spare=2):
    seqs, vocab, rows = len(starts) - 1, p.shape[1], len(p)
    bufs = [ctx.buffer_from(x) if x is not None and x.size else ctx.buffer(16) for x in (p, q, d, u, starts)]
    out, acc = ctx.buffer_from(np.full(rows + spare, 77, np.uint32)), ctx.buffer_from(np.full(seqs + 1, 77, np.uint32))
    go(ctx, lambda c: K.verify_drafts(c, bufs[0], bufs[1] if q is not None else None, bufs[2], bufs[3], bufs[4], seqs, rows, vocab, out, acc))
    got = out.download(np.uint32), acc.download(np.uint32)
    for b in bufs + [out, acc]:
        b.free()
    want_t, want_a = np.full(rows + spare, 77, np.uint32), np.full(seqs + 1, 77, np.uint32)
    R.verify(p, q, d, u, starts, want_t, want_a[:-1])
    return got, (want_t, want_a)


@pytest.mark.parametrize("vocab", [1, 2, 31, 127, 1000, 4099, 40003])
@pytest.mark.parametrize("given", [True, False])
def test_verify(ctx, K, vocab, given):
    g = np.random.default_rng(vocab)
    for seqs, drafts, empty in ((1, 0, 0), (1, 5, 0), (9, 4, 0.3), (40 if vocab < 5000 else 5, 7, 0)):
        case = random_verify(g, seqs, drafts, vocab, given, empty)
        if len(case[0]):
            got, want = run_verify(ctx, K, *case)
            assert (got[1] == want[1]).all() and (got[0] == want[0]).all()


def test_verify_odd_numbers(ctx, K):
    """Entries that are no positive finite numbers, drafts outside the vocabulary, u at both ends, nothing left of p - q, nothing in p."""
    V = 700
    g = np.random.default_rng(1)
    p, q = (g.dirichlet(np.full(V, 0.5), 14).astype(np.float32) for _ in range(2))
    starts = np.array([0, 2, 4, 6, 8, 10, 12, 14], np.uint32)
    d = g.integers(0, V, 7).astype(np.uint32)
    u = g.random(14).astype(np.float32)
    p[0, :50], p[0, 60], p[0, 61], p[0, 62] = np.nan, np.inf, -1.0, 0.0
    u[0] = 0.9999999
    d[1] = V
    d[2] = 2 ** 32 - 1
    q = q[:7].copy()
    q[3] = 1.0  # more than p everywhere: refused, and nothing is left
    u[6] = 0.9999999
    p[8], p[9] = 0.0, 0.0
    u[11], u[13] = 0.0, 0.99999994
    p[12, d[6]] = 1.0
    for qq in (q, None):
        got, want = run_verify(ctx, K, p, qq, d, u, starts)
        assert (got[1] == want[1]).all() and (got[0] == want[0]).all()
    u[9], p[9, 5:9] = 1.0, 0.1  # a u that is no number below 1: the last id that has any mass
    got, want = run_verify(ctx, K, p, None, d, u, starts)
    assert (got[0] == want[0]).all()


@pytest.mark.parametrize("vocab", [40, 4099])
@pytest.mark.parametrize("given", [True, False])
def test_verify_entries_that_are_no_numbers_count_as_0(ctx, K, vocab, given):
    """Infinities, NaN and negative numbers at drafts and elsewhere, in p and in q: the result is that of the same call with zeros in their places."""
    g = np.random.default_rng(vocab)
    odd = np.array([np.nan, np.inf, -np.inf, -0.25, -0.0], np.float32)
    p, q, d, u, starts = random_verify(g, 150, 4, vocab, given)
    at = 0
    for s in range(150):
        for i in range(int(starts[s]), int(starts[s + 1]) - 1):
            if g.random() < 0.5:
                p[i, d[at]] = g.choice(odd)
            if given and g.random() < 0.5:
                q[at, d[at]] = g.choice(odd)
            at += 1
    for x in (p, q) if given else (p,):
        x[g.random(x.shape) < 0.1] = g.choice(odd)
        x[:, ::7] = g.choice(odd, x[:, ::7].shape)
    zeros = lambda x: None if x is None else np.where(np.isfinite(x) & (x > 0), x, 0).astype(np.float32)
    with np.errstate(invalid="ignore"):
        got, _ = run_verify(ctx, K, p, q, d, u, starts)
    same, want = run_verify(ctx, K, zeros(p), zeros(q), d, u, starts)
    assert (same[0] == want[0]).all() and (same[1] == want[1]).all()
    assert (got[0] == want[0]).all() and (got[1] == want[1]).all()


def test_verify_draws_as_the_target_does(ctx, K):
    """First tokens of 20 000 verified drafts are distributed as p: each frequency within five standard deviations."""
    g = np.random.default_rng(4)
    n, V = 20000, 6
    p1, q1 = np.array([0.35, 0.05, 0.2, 0.3, 0.1, 0.0], np.float32), np.array([0.1, 0.3, 0.2, 0.05, 0.15, 0.2], np.float32)
    p, q = np.tile(p1, (2 * n, 1)), np.tile(q1, (n, 1))
    d = g.choice(V, n, p=q1 / q1.sum()).astype(np.uint32)
    (tokens, acc), want = run_verify(ctx, K, p, q, d, g.random(2 * n).astype(np.float32), np.arange(0, 2 * n + 1, 2).astype(np.uint32))
    assert (tokens == want[0]).all() and (acc == want[1]).all()
    share = np.bincount(tokens[0:2 * n:2], minlength=V) / n
    assert (np.abs(share - p1) <= 5 * np.sqrt(p1 * (1 - p1) / n) + 1e-9).all()


class Pages:
    def __init__(self, g, rows, max_pages, num_pages, layers, hkv, kv, fill):
        self.layers, self.hkv, self.kv = layers, hkv, kv
        self.num_pages = num_pages
        self.table = np.full((rows, max_pages), -1, np.int32)
        self.lens = np.zeros(rows, np.uint32)
        free = list(g.permutation(num_pages))
        for r in range(rows):
            n = int(g.integers(0, max_pages * 16 + 1) * fill)
            c = -(-n // 16)
            if c <= len(free):
                self.table[r, :c] = [free.pop() for _ in range(c)]
                self.lens[r] = n
        self.pinned = (g.random(num_pages) < 0.05).astype(np.uint32)
        shape = (layers, num_pages, 16, hkv, R.ROW[kv])
        self.k, self.v = (g.integers(0, 256, shape, dtype=np.uint8) for _ in range(2))

    def device(self, ctx, K, pinned=True):
        self.bufs = [ctx.buffer_from(x) for x in (self.k, self.v, self.table, self.lens, self.pinned)]
        return K.page_pool(*self.bufs[:4], self.bufs[4] if pinned else None, *self.table.shape, self.num_pages, self.layers, self.hkv, KV[self.kv])


def run_reassign(ctx, K, P, source, keep, room, pinned=True, accepted=None):
    pool = P.device(ctx, K, pinned)
    ins = [None if x is None else ctx.buffer_from(np.array(x, t)) for x, t in ((source, np.int32), (keep, np.uint32), (room, np.uint32), (accepted, np.uint32))]
    outs = [ctx.buffer_from(np.full_like(P.table, 99)), ctx.buffer_from(np.full_like(P.lens, 99)), ctx.buffer(16)]
    go(ctx, lambda c: K.pages_reassign(c, pool, *ins[:3], *outs, accepted=ins[3]))
    got = outs[0].download(np.int32).reshape(P.table.shape), outs[1].download(np.uint32), outs[2].download(np.uint32)
    pools = [b.download(np.uint8).reshape(P.k.shape) for b in P.bufs[:2]]
    for b in P.bufs + [x for x in ins if x] + outs:
        b.free()
    table, lens, result, copies = R.reassign(P.table, P.lens, P.pinned if pinned else None, P.num_pages, source, keep, room, accepted)
    assert list(got[2]) == result
    assert (got[1] == lens).all() and (got[0] == table).all()
    for have, was in zip(pools, (P.k, P.v)):
        want = was.copy()
        for a, b in copies:
            want[:, b] = was[:, a]
        assert (have == want).all()
    return table, lens, result


@pytest.mark.parametrize("rows,max_pages,num_pages,layers,hkv,kv", [(1, 1, 1, 1, 1, "f16"), (4, 5, 40, 2, 2, "q8_0"), (33, 9, 700, 1, 1, "f32"), (7, 40, 900, 3, 1, "f16"),
                                                                  (70, 3, 60, 1, 3, "q8_0"), (1500, 2, 5000, 1, 1, "q8_0")])
def test_reassign(ctx, K, rows, max_pages, num_pages, layers, hkv, kv):
    g = np.random.default_rng(rows)
    P = Pages(g, rows, max_pages, num_pages, layers, hkv, kv, 0.6)
    most = max_pages * 16
    same = np.arange(rows)
    seen_short = False
    for source, keep, room in (
            (same, P.lens, np.zeros(rows)),                                          # nothing changes
            (same, P.lens, g.integers(0, 40, rows)),                                 # room to go on
            (same, g.integers(0, most + 1, rows), np.full(rows, 3)),                 # rolled back
            (g.integers(0, rows, rows), np.full(rows, most), np.full(rows, 1)),      # beams: rows of any row
            (np.zeros(rows), np.full(rows, P.lens[0]), g.integers(0, 20, rows)),     # all of the first
            (g.integers(-2, rows + 2, rows), g.integers(0, most + 1, rows), g.integers(0, most, rows)),
            (np.full(rows, -1), np.full(rows, most), np.zeros(rows)),                # all given back
            (same, np.full(rows, 2 ** 32 - 1), np.full(rows, 2 ** 32 - 1))):         # as much as the table holds
        result = run_reassign(ctx, K, P, source.astype(np.int64), keep.astype(np.int64), room.astype(np.int64), pinned=rows != 7)[2]
        seen_short |= result[3] > 0
    assert seen_short or rows != 70
    got = g.integers(0, 9, rows)
    run_reassign(ctx, K, P, same, None, np.full(rows, 4), accepted=got)
    run_reassign(ctx, K, P, same[::-1], P.lens.astype(np.int64) + 3, np.full(rows, 4), accepted=got)
    run_reassign(ctx, K, P, same, None, np.zeros(rows), pinned=False)


def test_reassign_pages_held_more_than_once(ctx, K):
    """Rows that share pages already: the last page of one row is a whole page of another, or pinned, or named twice; entries that are no pages."""
    g = np.random.default_rng(0)
    P = Pages(g, 6, 4, 30, 2, 1, "f16", 0)
    P.table[:] = [[3, 4, 5, -1], [3, 4, -1, -1], [3, 9, -1, -1], [7, -5, 8, -1], [2, 2, -1, -1], [40, 6, 11, -1]]
    P.lens[:] = [40, 24, 20, 41, 30, 40]
    P.pinned[:] = 0
    P.pinned[9] = 1
    run_reassign(ctx, K, P, np.arange(6), P.lens.astype(np.int64), np.full(6, 7))
    run_reassign(ctx, K, P, [0, 0, 2, 2, 3, 5], [40, 33, 20, 17, 20, 5], [0, 30, 1, 0, 5, 17])


def test_steps_with_paused_and_free_rows(ctx, K):
    """Verification and reassignment in turn, with rows that have no tokens in a step, among them free ones of length 0: those keep their length, the others gain what
    stood. Every table against the host's."""
    g = np.random.default_rng(71)
    rows, V = 24, 90
    P = Pages(g, rows, 12, 400, 2, 1, "f16", 0.2)
    P.pinned[:] = 0
    P.lens[3], P.table[3], P.lens[9], P.table[9] = 0, -1, 0, -1
    tables, lens = [ctx.buffer_from(P.table), ctx.buffer(P.table.nbytes)], [ctx.buffer_from(P.lens), ctx.buffer(4 * rows)]
    pools = [ctx.buffer_from(P.k), ctx.buffer_from(P.v)]
    result, source = ctx.buffer(16), np.arange(rows)
    acc, now = None, 0
    for step in range(6):
        p, q, d, u, starts = random_verify(g, rows, 4, V, True, 0.4)
        starts_before = ctx.buffer_from(starts)
        out, acc = ctx.buffer(4 * len(p)), ctx.buffer(4 * rows)
        ins = [ctx.buffer_from(x) for x in (p, q, d, u)]
        go(ctx, lambda c: K.verify_drafts(c, *ins, starts_before, rows, len(p), V, out, acc))
        host = acc.download(np.uint32).astype(np.int64)
        host[np.diff(starts) == 0] = -1  # (+ 1: no position more)
        room = np.where(g.random(rows) < 0.3, 0, 5)
        table, length, res, copies = R.reassign(P.table, P.lens, None, P.num_pages, source, None, room, host)
        args = [ctx.buffer_from(x) for x in (source.astype(np.int32), room.astype(np.uint32))]
        pool = K.page_pool(*pools, tables[now], lens[now], None, rows, 12, 400, 2, 1, 1)
        go(ctx, lambda c: K.pages_reassign(c, pool, args[0], None, args[1], tables[1 - now], lens[1 - now], result, accepted=acc, starts=starts_before))
        now = 1 - now
        assert (lens[now].download(np.uint32) == length).all() and list(result.download(np.uint32)) == res
        assert (tables[now].download(np.int32).reshape(table.shape) == table).all()
        assert (length[np.diff(starts) == 0] == P.lens[np.diff(starts) == 0]).all()
        P.table, P.lens = table, length


@pytest.mark.parametrize("rows,max_pages,num_pages,layers,hkv,kv", [(1, 1, 1, 1, 1, "f16"), (4, 5, 40, 2, 2, "q8_0"), (33, 9, 1500, 1, 1, "f32"), (7, 40, 200, 3, 1, "f16"),
                                                                  (20, 300, 40000, 1, 1, "q8_0")])
@pytest.mark.parametrize("in_place", [False, True])
def test_compact(ctx, K, rows, max_pages, num_pages, layers, hkv, kv, in_place):
    g = np.random.default_rng(rows + 1)
    P = Pages(g, rows, max_pages, num_pages, layers, hkv, kv, 0.4)
    P.table[rows // 2] = P.table[0]  # shared pages
    P.table[0, -1] = num_pages + 3
    for pinned in (True, False):
        pool = P.device(ctx, K, pinned)
        out, moved, result = ctx.buffer(P.table.nbytes), ctx.buffer(num_pages * 4), ctx.buffer(16)
        go(ctx, lambda c: K.pages_compact(c, pool, P.bufs[2] if in_place else out, moved, result))
        table, want_moved, want_result, moves = R.compact(P.table, P.pinned if pinned else None, num_pages)
        assert list(result.download(np.uint32)) == want_result
        assert (moved.download(np.int32) == want_moved).all()
        assert ((P.bufs[2] if in_place else out).download(np.int32).reshape(table.shape) == table).all()
        for b, was in zip(P.bufs[:2], (P.k, P.v)):
            want = was.copy()
            for a, to in moves:
                want[:, to] = was[:, a]
            assert (b.download(np.uint8).reshape(was.shape) == want).all()
        for b in P.bufs + [out, moved, result]:
            b.free()


def test_recorded_steps_of_two_sizes(B, ctx, K):
    """Verification and pages out of recorded graphs: two graphs of one context share its workspaces, the second made them grow, and each replay follows what
    the buffers hold by then."""
    g = np.random.default_rng(31)

    class Step:
        def __init__(self, rows, max_pages, num_pages):
            self.P = P = Pages(g, rows, max_pages, num_pages, 2, 1, "f16", 0.5)
            self.p, self.q, self.d, self.u, self.starts = random_verify(g, rows, 3, 500, True)
            self.pool = P.device(ctx, K)
            self.ver = [ctx.buffer_from(x) for x in (self.p, self.q, self.d, self.u, self.starts)] + [ctx.buffer(4 * len(self.p)), ctx.buffer(4 * rows)]
            self.src, self.room = np.arange(rows, dtype=np.int32), np.full(rows, 4, np.uint32)
            self.ins = [ctx.buffer_from(self.src), ctx.buffer_from(self.room)]
            self.table, self.lens, self.moved = ctx.buffer(P.table.nbytes), ctx.buffer(4 * rows), ctx.buffer(4 * num_pages)
            self.results = ctx.buffer(16), ctx.buffer(16)
            self.after = K.page_pool(*P.bufs[:2], self.table, self.lens, P.bufs[4], rows, max_pages, num_pages, 2, 1, 1)

        def __call__(self, c):
            K.verify_drafts(c, *self.ver[:5], len(self.src), len(self.p), 500, *self.ver[5:])
            K.pages_reassign(c, self.pool, self.ins[0], None, self.ins[1], self.table, self.lens, self.results[0], accepted=self.ver[6])
            K.pages_compact(c, self.after, self.table, self.moved, self.results[1])

        def reset(self):
            self.u = g.random(len(self.u)).astype(np.float32)
            self.src = g.integers(-1, len(self.src), len(self.src)).astype(np.int32)
            for b, x in zip(self.P.bufs[:2] + [self.ver[3], self.ins[0]], (self.P.k, self.P.v, self.u, self.src)):
                b.upload(x)

        def check(self):
            P = self.P
            tokens, acc = np.zeros(len(self.p), np.uint32), np.zeros(len(self.src), np.uint32)
            R.verify(self.p, self.q, self.d, self.u, self.starts, tokens, acc)
            assert (self.ver[5].download(np.uint32) == tokens).all() and (self.ver[6].download(np.uint32) == acc).all()
            table, lens, result, copies = R.reassign(P.table, P.lens, P.pinned, P.num_pages, self.src, None, self.room, acc)
            last, moved, after, moves = R.compact(table, P.pinned, P.num_pages)
            assert (self.lens.download(np.uint32) == lens).all() and list(self.results[0].download(np.uint32)) == result
            assert (self.table.download(np.int32).reshape(last.shape) == last).all() and list(self.results[1].download(np.uint32)) == after
            for b, was in zip(P.bufs[:2], (P.k, P.v)):
                want = was.copy()
                for x, to in copies:
                    want[:, to] = was[:, x]
                then = want.copy()
                for x, to in moves:
                    then[:, to] = want[:, x]
                assert (b.download(np.uint8).reshape(was.shape) == then).all()

    small = Step(3, 5, 40)
    go(ctx, small)
    small.check()
    graphs = [ctx.capture(small)]
    large = Step(50, 9, 900)
    go(ctx, large)
    large.check()
    graphs.append(ctx.capture(large))
    for _ in range(3):
        for x in (small, large):
            x.reset()
        cmd = ctx.command()
        for graph in graphs:
            graph.launch(cmd)
        cmd.wait()
        for x in (small, large):
            x.check()
    for graph in graphs:
        graph.free()


def test_two_contexts_at_once(B, ctx, K):
    """Calls of two contexts, in flight together: each has its own stream and workspaces."""
    run = R.Run([(130, 600), (5, 2000), (1, 40)], 8, 2, "f16", seed=41)
    want, tol = run.attention(True)
    other = B.Context(0)
    sides = []
    for c in (ctx, other):
        k = B.Kernels(c)
        sides.append((c, k, OnDevice(c, k, run), c.buffer(run.tokens * 8 * 256)))
    for c, k, dev, o in sides:  # (the first call makes the workspaces)
        go(c, lambda cmd: k.attention_packed(cmd, dev.q, dev.paged, dev.packed, o, 8, 2, 0))
        o.fill(0)
    cmds = [c.command() for c, *_ in sides]
    for _ in range(8):
        for cmd, (c, k, dev, o) in zip(cmds, sides):
            k.attention_packed(cmd, dev.q, dev.paged, dev.packed, o, 8, 2, 0)
    for cmd in cmds:
        cmd.wait()
    for c, k, dev, o in sides:
        check(o.download(np.float16).astype(np.float64).reshape(run.tokens, 8, 128), want, tol)
        o.free()
        dev.free()
    other.close()


def test_refusals_of_positions_past_31_bits(B, ctx, K):
    run = R.Run([(2, 20)], 4, 2, "f16")
    dev = OnDevice(ctx, K, run)
    far = K.paged_kv(dev.kpool, dev.vpool, dev.bufs[2], dev.bufs[3], 1, 2 ** 27, run.num_pages, 1)
    o = ctx.buffer(run.tokens * 4 * 256)
    with pytest.raises(B.BrasaError, match="2\\^31 positions") as e:
        go(ctx, lambda c: K.attention_packed(c, dev.q, far, dev.packed, o, 4, 2, 0))
    assert e.value.code == B.EINVAL


def test_refusals_of_an_output_over_the_queries(B, ctx, K):
    run = R.Run([(2, 20)], 4, 2, "f16")
    dev = OnDevice(ctx, K, run)
    n = run.tokens * 4 * 128
    both = ctx.buffer(n * 8)
    for half, at in ((True, 0), (True, 2 * n), (False, 0), (False, 4 * n - 16)):
        with pytest.raises(B.BrasaError, match="overlap") as e:
            go(ctx, lambda c: K.attention_packed(c, both, dev.paged, dev.packed, both.at(at), 4, 2, 0 if half else 1))
        assert e.value.code == B.EINVAL
    both.upload(run.q, 0)
    go(ctx, lambda c: K.attention_packed(c, both, dev.paged, dev.packed, both.at(4 * n), 4, 2, 1))
    want, tol = run.attention(False)
    check(both.download(np.float32)[n:].astype(np.float64).reshape(run.tokens, 4, 128), want, tol)


def test_refusals_of_outputs_over_inputs(B, ctx, K):
    """Two sequences' rows, pages and tokens are written side by side: outputs over what is read, or over one another, are refused; the queries in place are not."""
    run = R.Run([(2, 20)], 4, 2, "f16")
    dev, T = OnDevice(ctx, K, run), run.tokens
    rope, norm, b = B.RopeTable(ctx, THETA, 128, run.max_pages * 16), ctx.buffer_from(np.ones(128, np.float32)), ctx.buffer(T * 512 * 16)
    kv, far = b.at(T * 512 * 4), b.at(T * 512 * 8)

    def store(q, out):
        go(ctx, lambda c: K.qk_norm_rope_store_packed(c, q, kv, kv, norm, norm, EPS, rope, dev.paged, dev.packed, out, 4, 2))

    x = ctx.buffer(4 * 300)
    f = {n: ctx.buffer(4096) for n in ("p", "q", "d", "u", "s", "t", "a")}

    def ver(out, acc):
        go(ctx, lambda c: K.verify_drafts(c, f["p"], f["q"], f["d"], f["u"], f["s"], 2, 4, 100, out, acc))

    pool = ctx.buffer(2 * 8 * 16 * 256)
    page = K.page_pool(pool, pool, ctx.buffer(48), ctx.buffer(16), None, 4, 3, 8, 2, 1, 1)
    a, room = ctx.buffer(16), ctx.buffer(64)

    def rea(out, lens, res):
        go(ctx, lambda c: K.pages_reassign(c, page, a, None, room, out, lens, res))

    def com(out, moved, res):
        go(ctx, lambda c: K.pages_compact(c, page, out, moved, res))
    store(b, b), store(b, far), ver(x, x.at(16)), rea(x, x.at(48), x.at(64)), com(x, x.at(48), x.at(80))
    before = ctx.launch_count()
    bad = [(store, b, b.at(512)), (store, b.at(512), b), (store, far, kv), (store, far, b.at(T * 512 * 3)), (store, far, b.at(T * 512 * 6 - 512)),
           (ver, f["d"], f["a"]), (ver, f["u"].at(12), f["a"]), (ver, f["p"].at(1596), f["a"]), (ver, f["q"].at(400), f["a"]), (ver, f["s"].at(8), f["a"]), (ver, f["t"], f["d"].at(4)),
           (ver, f["t"], f["u"]), (ver, f["t"], f["t"].at(12)), (ver, f["t"].at(4), f["t"]),
           (rea, x, x.at(44), x.at(64)), (rea, x, x.at(48), x.at(32)), (rea, x, x.at(48), x.at(60)), (rea, room, x.at(48), x.at(64)),
           (com, x, x.at(44), x.at(80)), (com, x, x.at(48), x.at(76)), (com, x, x.at(48), x.at(40))]
    for call, *args in bad:
        with pytest.raises(B.BrasaError, match="overlap") as e:
            call(*args)
        assert e.value.code == B.EINVAL
    assert ctx.launch_count() == before


def test_refusals_of_outputs_over_pools_and_tables(B, ctx, K):
    """Outputs over the pools, tables, norms and lengths that the same launch reads, and pools over what is read or over one another."""
    run = R.Run([(2, 20)], 4, 2, "f16")
    T, pages = run.tokens, run.num_pages
    size = pages * 16 * 2 * 256
    big = ctx.buffer(4 * size)
    n_rope = run.max_pages * 16 * 64 * 4

    class Rope:
        cos, sin = ctx.buffer(n_rope), ctx.buffer(n_rope)
    f = {x: ctx.buffer(4096) for x in ("q", "k", "v", "o", "qn", "kn", "table", "lens", "starts")}
    f["starts"].upload(run.starts), f["table"].upload(run.table), f["lens"].upload(run.lens)

    def calls(kpool=big, vpool=big.at(size), out=None, **over):
        x = {**f, **over}
        paged, packed = K.paged_kv(kpool, vpool, x["table"], x["lens"], 1, run.max_pages, pages, 1), K.packed_run(x["starts"], T, 2)
        return (lambda c: K.qk_norm_rope_store_packed(c, x["q"], x["k"], x["v"], x["qn"], x["kn"], EPS, Rope, paged, packed, out or x["o"], 4, 2),
                lambda c: K.attention_packed(c, x["q"], paged, packed, out or x["o"], 4, 2, 1))
    for call in calls():
        go(ctx, call)
    both = [dict(out=big.at(size - 16)), dict(out=big.at(2 * size - 512)), dict(out=f["table"]), dict(out=f["lens"]), dict(out=f["starts"])]
    store = [dict(out=f["qn"]), dict(out=f["kn"]), dict(out=Rope.cos), dict(out=Rope.sin.at(n_rope - 4096)), dict(vpool=big.at(16)), dict(vpool=big), dict(q=big), dict(k=big.at(size)), dict(v=big.at(2 * size - 2048)),
             dict(qn=big.at(64)), dict(table=big), dict(lens=big.at(size)), dict(starts=big.at(8)), dict(q=big.at(2 * size - 16), out=big.at(2 * size - 16))]
    pool = ctx.buffer(8 * 16 * 256)
    small = {x: ctx.buffer(256) for x in ("table", "lens", "pinned", "src", "keep", "acc", "st", "room", "out", "lens_out", "res", "moved")}

    def page_calls(**over):
        x = {**small, **over}
        g = K.page_pool(pool, pool, x["table"], x["lens"], x["pinned"], 4, 3, 8, 1, 1, 1)
        return (lambda c: K.pages_reassign(c, g, x["src"], x["keep"], x["room"], x["out"], x["lens_out"], x["res"], accepted=x["acc"], starts=x["st"]),
                lambda c: K.pages_compact(c, g, x["out"], x["moved"], x["res"]))
    for call in page_calls():
        go(ctx, call)
    before = ctx.launch_count()
    bad = [x for kw in both for x in calls(**kw)] + [calls(**kw)[0] for kw in store]
    bad += [page_calls(**{x: pool})[0] for x in ("table", "lens", "pinned", "src", "keep", "acc", "st", "room", "out", "lens_out", "res")]
    bad += [page_calls(**{x: pool.at(8 * 16 * 256 - 64)})[1] for x in ("table", "pinned", "out", "res", "moved")]
    for i, call in enumerate(bad):
        with pytest.raises(B.BrasaError) as e:
            go(ctx, call)
        assert e.value.code == B.EINVAL and "overlap" in str(e.value), i
    assert ctx.launch_count() == before


def test_refusals_of_starts(B, ctx, K):
    pool = ctx.buffer(2 * 8 * 16 * 256)
    page = K.page_pool(pool, pool, ctx.buffer(48), ctx.buffer(16), None, 4, 3, 8, 2, 1, 1)
    src, acc, room, out, starts, lens, res, small = (ctx.buffer(n) for n in (16, 16, 16, 48, 20, 16, 16, 16))

    def rea(acc=acc, starts=starts, lens_out=lens):
        go(ctx, lambda c: K.pages_reassign(c, page, src, None, room, out, lens_out, res, accepted=acc, starts=starts))
    rea(), rea(starts=None)
    for kw in (dict(starts=small), dict(starts=pool.at(2)), dict(acc=None), dict(lens_out=pool, starts=pool.at(12)), dict(starts=pool, lens_out=pool.at(16))):
        with pytest.raises(B.BrasaError) as e:
            rea(**kw)
        assert e.value.code == B.EINVAL, kw


def test_refusals(B, ctx, K):
    """Every precondition comes back as EINVAL, with nothing launched."""
    run = R.Run([(2, 20), (1, 3)], 4, 2, "f16")
    dev = OnDevice(ctx, K, run)
    k, v, t, n, s, q = dev.bufs
    o, small, w = ctx.buffer(run.tokens * 4 * 512), ctx.buffer(16), ctx.buffer(512)
    rope = B.RopeTable(ctx, THETA, 128, run.max_pages * 16)
    kv2, run2 = ctx.buffer(run.tokens * 2 * 512), dev.packed

    def paged(**kw):
        a = dict(kpool=k, vpool=v, table=t, lens=n, seqs=2, max_pages=run.max_pages, num_pages=run.num_pages, kv=1) | kw
        return K.paged_kv(*a.values())

    def store(c, paged=dev.paged, packed=run2, q=q, k=kv2, out=o, norm=w, rope=rope, hq=4, hkv=2):
        K.qk_norm_rope_store_packed(c, q, k, kv2, norm, w, EPS, rope, paged, packed, out, hq, hkv)

    def att(c, paged=dev.paged, packed=run2, q=q, o=o, hq=4, hkv=2, precision=0):
        K.attention_packed(c, q, paged, packed, o, hq, hkv, precision)
    short = B.RopeTable(ctx, THETA, 128, 16)
    f = {x: ctx.buffer(4096) for x in "pqudsta"}

    def ver(c, p=f["p"], q=f["q"], d=f["d"], u=f["u"], st=f["s"], seqs=2, rows=4, vocab=100, out=f["t"], acc=f["a"]):
        K.verify_drafts(c, p, q, d, u, st, seqs, rows, vocab, out, acc)
    kp = ctx.buffer(2 * 8 * 16 * 256)
    tb, tb2, ln, ln2, pins = ctx.buffer(4 * 3 * 4), ctx.buffer(4 * 3 * 4), ctx.buffer(16), ctx.buffer(16), ctx.buffer(32)

    def pool(**kw):
        a = dict(kpool=kp, vpool=kp, table=tb, lens=ln, pinned=pins, rows=4, max_pages=3, num_pages=8, layers=2, hkv=1, kv=1) | kw
        return K.page_pool(*a.values())
    src, keep, room, res, moved = (ctx.buffer(32) for _ in range(5))

    def rea(c, pool=pool(), source=src, keep=keep, acc=None, out=tb2, lens_out=ln2, result=res):
        K.pages_reassign(c, pool, source, keep, room, out, lens_out, result, accepted=acc)

    def com(c, pool=pool(), out=tb2, moved=moved, result=res):
        K.pages_compact(c, pool, out, moved, result)
    for f_ok in (store, att, ver, rea, com):
        go(ctx, f_ok)
    before = ctx.launch_count()
    bad = [(store, dict(paged=paged(num_pages=run.num_pages + 1))), (store, dict(paged=paged(kv=3))), (store, dict(paged=paged(seqs=0))), (store, dict(paged=paged(table=small))),
           (store, dict(packed=K.packed_run(s, 0, 2))), (store, dict(packed=K.packed_run(s, run.tokens, 0))),
           (store, dict(packed=K.packed_run(s.at(8), run.tokens, 2))), (store, dict(packed=K.packed_run(s.at(2), run.tokens, 2))), (store, dict(packed=K.packed_run(s, run.tokens + 1, 2))),
           (store, dict(q=small)), (store, dict(q=None)), (store, dict(k=small)), (store, dict(out=small)), (store, dict(out=o.at(4))), (store, dict(norm=small)), (store, dict(rope=short)),
           (store, dict(hq=0)), (store, dict(hkv=0)), (store, dict(hq=5)), (store, dict(hq=18, hkv=2)),
           (att, dict(paged=paged(lens=small.at(12)))), (att, dict(packed=K.packed_run(s, run.tokens + 9, 2))), (att, dict(q=small)), (att, dict(o=small)), (att, dict(o=o.at(8))),
           (att, dict(precision=2)), (att, dict(precision=-1)), (att, dict(hq=0)), (att, dict(hq=3)),
           (ver, dict(seqs=0)), (ver, dict(rows=0)), (ver, dict(vocab=0)), (ver, dict(rows=12)), (ver, dict(vocab=300)), (ver, dict(d=small.at(12))), (ver, dict(u=small.at(4))),
           (ver, dict(st=small.at(8))), (ver, dict(out=small.at(4))), (ver, dict(acc=small.at(12))), (ver, dict(p=f["p"].at(2))), (ver, dict(p=None)), (ver, dict(seqs=2 ** 30)),
           (rea, dict(pool=pool(kv=3))), (rea, dict(pool=pool(rows=0))), (rea, dict(pool=pool(layers=3))), (rea, dict(pool=pool(max_pages=4))), (rea, dict(pool=pool(num_pages=2 ** 19 + 1))),
           (rea, dict(pool=pool(rows=65537))), (rea, dict(pool=pool(pinned=small))), (rea, dict(pool=pool(kpool=kp.at(8)))), (rea, dict(source=small.at(4))), (rea, dict(source=None)), (rea, dict(acc=small.at(4))), (rea, dict(keep=small.at(4))),
           (rea, dict(out=tb)), (rea, dict(out=tb2.at(4))), (rea, dict(lens_out=ln)), (rea, dict(result=ln)), (rea, dict(result=small.at(4))),
           (com, dict(pool=pool(hkv=0))), (com, dict(moved=small)), (com, dict(moved=tb)), (com, dict(moved=pins)), (com, dict(out=small)), (com, dict(result=pins)), (com, dict(out=pins))]
    for call, kw in bad:
        with pytest.raises(B.BrasaError) as e:
            go(ctx, lambda c: call(c, **kw))
        assert e.value.code == B.EINVAL, (call.__name__, kw)
    assert ctx.launch_count() == before


@pytest.mark.parametrize("kv", ["f16", "q8_0"])
def test_a_decoding_loop_with_drafts(B, ctx, K, kv):
    """Two layers' caches through steps of drafting, verification, rollback and forks, as a program drives them; every attention against a cache that is
    kept densely on the host, in the values that the pool gives back."""
    g = np.random.default_rng(30)
    rows, max_pages, num_pages, layers, hq, hkv, V = 5, 12, 70, 2, 8, 2, 300
    half = True
    shape = (layers, num_pages, 16, hkv, R.ROW[kv])
    pools = [ctx.buffer_from(np.full(shape, 0xFF, np.uint8)) for _ in range(2)]
    layer_bytes = int(np.prod(shape[1:]))
    tables, lens = [ctx.buffer_from(np.full((rows, max_pages), -1, np.int32)) for _ in range(2)], [ctx.buffer(rows * 4) for _ in range(2)]
    rope = B.RopeTable(ctx, THETA, 128, max_pages * 16)
    norm = ctx.buffer_from(np.ones(128, np.float32))
    result = ctx.buffer(16)
    dense = [[[np.zeros((0, hkv, 128)) for _ in range(2)] for _ in range(layers)] for _ in range(rows)]  # [row][layer][k, v]
    source, keep, acc, now = np.arange(rows), np.zeros(rows, int), np.zeros(rows, int), 0
    for step in range(7):
        new = [int(g.integers(1, 6)) if step else int(g.integers(10, 60)) for _ in range(rows)]
        if step == 3:
            source = np.array([0, 0, 2, 2, 2])
            keep = keep[source]
        ins = [ctx.buffer_from(np.array(x, t)) for x, t in ((source, np.int32), (new, np.uint32), (acc, np.uint32))]
        pool = K.page_pool(*pools, tables[now], lens[now], None, rows, max_pages, num_pages, layers, hkv, KV[kv])
        go(ctx, lambda c: K.pages_reassign(c, pool, ins[0], None, ins[1], tables[1 - now], lens[1 - now], result, accepted=ins[2] if step else None))
        now = 1 - now
        assert result.download(np.uint32)[3] == 0 and (lens[now].download(np.uint32) == keep).all()
        dense = [[[x[:keep[r]] for x in dense[source[r]][li]] for li in range(layers)] for r in range(rows)]
        starts = np.concatenate([[0], np.cumsum(new)]).astype(np.uint32)
        T = int(starts[-1])
        run = K.packed_run(ctx.buffer_from(starts), T, max(new))
        table = tables[now].download(np.int32).reshape(rows, max_pages)
        for li in range(layers):
            paged = K.paged_kv(pools[0].at(li * layer_bytes), pools[1].at(li * layer_bytes), tables[now], lens[now], rows, max_pages, num_pages, KV[kv])
            q, k, v = (g.standard_normal((T, h, 128)).astype(np.float32) for h in (hq, hkv, hkv))
            gq, gk, gv, o = ctx.buffer_from(q), ctx.buffer_from(k), ctx.buffer_from(v), ctx.buffer(T * hq * 256)

            def layer(c):
                K.qk_norm_rope_store_packed(c, gq, gk, gv, norm, norm, EPS, rope, paged, run, gq, hq, hkv)
                K.attention_packed(c, gq, paged, run, o, hq, hkv, 0)
            go(ctx, layer)
            got = o.download(np.float16).astype(np.float64).reshape(T, hq, 128)
            raw = [p.download(np.uint8, layer_bytes, li * layer_bytes).reshape(shape[1:]) for p in pools]
            for r in range(rows):
                at = [(table[r, i // 16], i % 16) for i in range(keep[r] + new[r])]
                for w, pool_rows in enumerate(raw):
                    have = np.stack([R.from_bytes(pool_rows[a], kv) for a in at])
                    assert (have[:keep[r]] == dense[r][li][w]).all(), (step, li, r)  # what is kept is what was there
                    dense[r][li][w] = have
                ref = R.Run([(new[r], int(keep[r]))], hq, hkv, "f32")
                ref.q = np.stack([R.norm_rope(q[starts[r] + j], np.ones(128), EPS, THETA, keep[r] + j) for j in range(new[r])])
                pages = [R.to_bytes(np.concatenate([x, np.zeros((-len(x) % 16, hkv, 128))]).reshape(-1, 16, hkv, 128).astype(np.float32), "f32") for x in dense[r][li]]
                ref.k, ref.v, ref.num_pages = *pages, len(pages[0])
                ref.table[0, :len(pages[0])] = np.arange(len(pages[0]))
                want, tol = ref.attention(half, kv)
                check(got[starts[r]:starts[r + 1]], want, tol + 2.0 ** -18)  # (and q's own rounding to 32 bits)
        p = g.dirichlet(np.full(V, 0.2), T).astype(np.float32)
        nd = T - rows
        drafts = np.array([np.argmax(p[i]) for r in range(rows) for i in range(starts[r], starts[r + 1] - 1)], np.uint32)
        (tokens, taken), want = run_verify(ctx, K, p, None, drafts, (0.3 * g.random(T)).astype(np.float32), starts, spare=0)
        assert (tokens == want[0]).all() and (taken == want[1]).all() and len(drafts) == nd
        acc = taken[:rows].astype(int)
        source, keep = np.arange(rows), keep + acc + 1
    assert keep.max() <= max_pages * 16
