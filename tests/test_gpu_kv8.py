"""The 8-bit K/V cache through the C-ABI: append / read bit for bit, attention within derived bounds (tests/kv8_ref.py), eviction, the
operators together as a generation uses them, refusals, graphs and streams."""
import ctypes as C

import numpy as np
import pytest

from kv8_ref import EPS, RefCache, attention

pytestmark = pytest.mark.gpu


def rows(rng, n, Hkv, D, spread=True):
    x = rng.standard_normal((2, n, Hkv, D))
    if spread:
        x *= (0.3 + rng.random((2, 1, Hkv, D)) ** 4 * 3) * np.exp(rng.standard_normal((2, n, 1, 1)) * 0.5)
    return x.astype(np.float32)


class Pair:
    """A cache on the device and its plain form, fed alike."""

    def __init__(self, thk, ctx, n_ctx, H, Hkv, D):
        self.ctx, self.shape = ctx, (n_ctx, H, Hkv, D)
        self.dev, self.ref = thk.KvCache8(ctx, n_ctx, H, Hkv, D), RefCache(n_ctx, Hkv, D)

    def append(self, x, pos):
        dk, dv = self.ctx.from_numpy(x[0]), self.ctx.from_numpy(x[1])
        self.dev.append(dk, dv, pos, x.shape[1])
        self.ref.append(x[0], x[1], pos)

    def read(self, pos, n):
        Hkv, D = self.shape[2:]
        ko, vo = self.ctx.alloc(n * Hkv * D * 4), self.ctx.alloc(n * Hkv * D * 4)
        self.dev.read(pos, n, ko, vo)
        return np.stack([o.download(np.float32, (n, Hkv, D)) for o in (ko, vo)])

    def attend(self, q, n_past, mass=None, decode=False):
        """q [M, H, D]; mass f32 [Hkv, n_ctx] or None -> (out, mass)"""
        ctx, M = self.ctx, q.shape[0]
        dq, out = ctx.from_numpy(q), ctx.alloc(q.nbytes)
        dm = None if mass is None else ctx.from_numpy(mass)
        do = None if mass is None else ctx.from_numpy(np.full_like(mass, 7.0))
        if decode:
            self.dev.attn_decode(dq, n_past + 1, out, dm, do)
        else:
            self.dev.attn_prefill(dq, n_past, M, out, dm, do)
        return out.download(np.float32, q.shape), None if mass is None else do.download(np.float32, mass.shape)

    def check(self, q, n_past, mass=None, decode=False):
        out, m = self.attend(q, n_past, mass, decode)
        eo, em, to, tm = attention(self.ref.values(), q, n_past, mass)
        assert np.all(np.abs(out - eo) <= to), (float((np.abs(out - eo) / to).max()), float(np.abs(out - eo).max()))
        rel = np.linalg.norm(out - eo) / max(np.linalg.norm(eo), 1e-30)
        assert rel < 1e-5, rel                      # the bound above is a worst case; f32 work stays far below this norm
        if mass is not None:
            T = n_past + q.shape[0]
            assert np.all(np.abs(m[:, :T] - em) <= tm), float((np.abs(m[:, :T] - em) / tm).max())
            assert np.all(m[:, T:] == 7.0)          # entries behind the last position stay as they were


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("Hkv,cuts", [(1, [1]), (3, [15, 1, 1]), (2, [16, 16]), (5, [7, 40, 1, 64, 3]), (2, [1] * 18), (4, [33, 31, 129])])
def test_append_read_bits(thk, ctx, D, Hkv, cuts):
    """Codes and scales are defined to the bit; cutting the tokens into calls does not change them."""
    rng = np.random.default_rng(D + Hkv + len(cuts))
    n = sum(cuts)
    x = rows(rng, n, Hkv, D)
    p, whole = Pair(thk, ctx, n + 3, Hkv, Hkv, D), Pair(thk, ctx, n + 3, Hkv, Hkv, D)
    at = 0
    for c in cuts:
        p.append(x[:, at:at + c], at)
        at += c
    whole.append(x, 0)
    got = p.read(0, n)
    assert np.array_equal(got, whole.read(0, n))
    assert np.array_equal(got, p.ref.values(0, n))
    assert np.array_equal(p.read(n // 2, 1), got[:, n // 2:n // 2 + 1])
    assert np.abs(got - x).max() <= np.abs(x).max() / 127 * 0.5 * (1 + 4 * EPS)


def test_append_truncates_and_reopens(thk, ctx):
    rng = np.random.default_rng(5)
    p = Pair(thk, ctx, 200, 4, 2, 128)
    for pos, n in [(0, 100), (90, 1), (91, 2), (40, 3), (43, 60), (101, 5), (16, 16), (32, 1)]:
        p.append(rows(rng, n, 2, 128), pos)
        assert np.array_equal(p.read(0, pos + n), p.ref.values(0, pos + n)), (pos, n)
        end = -(-(pos + n) // 16) * 16
        assert not p.read(pos + n, end - pos - n).any() if end > pos + n else True


def test_append_extremes(thk, ctx):
    """Zero, denormal, huge, infinite and NaN blocks; ties; one head's NaN stays with it."""
    rng = np.random.default_rng(6)
    x = rows(rng, 96, 3, 64)
    x[:, 0:16] = 0
    x[:, 16:32] *= np.float32(1e-38)
    x[:, 32:48] *= np.float32(1e36)
    x[0, 50, 1, 7], x[1, 51, 2, 9], x[0, 70, 0, 0] = np.nan, np.inf, -np.inf
    x[0, 80, :, :] = 127.0
    x[0, 81:96] = np.round(x[0, 81:96] * 4) + 0.5                                # codes next to a tie
    p = Pair(thk, ctx, 96, 3, 3, 64)
    p.append(x, 0)
    got, exp = p.read(0, 96), p.ref.values(0, 96)
    assert np.array_equal(got, exp, equal_nan=True)
    assert not got[:, :32].any() and np.isnan(got[0, 48:64, 1]).all() and np.isfinite(got[0, 48:64, 0]).all() and np.isnan(got[1, 48:64, 2]).all()


SHAPES = [(8, 8, 64), (4, 4, 128), (2, 2, 256), (32, 8, 128), (40, 40, 128), (24, 8, 64), (16, 1, 128), (20, 1, 128), (64, 2, 64), (15, 3, 256), (6, 6, 128)]


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 63, 64, 65, 130, 511, 1025])
@pytest.mark.parametrize("H,Hkv,D", [(8, 8, 64), (4, 4, 128), (32, 8, 128), (20, 1, 128), (15, 3, 256)])
def test_decode(thk, ctx, H, Hkv, D, T):
    rng = np.random.default_rng(T * 7 + H)
    p = Pair(thk, ctx, T + 5, H, Hkv, D)
    p.append(rows(rng, T, Hkv, D), 0)
    q = rng.standard_normal((1, H, D)).astype(np.float32)
    p.check(q, T - 1, decode=True)
    p.check(q * 3, T - 1, mass=rng.random((Hkv, T + 5)).astype(np.float32), decode=True)


@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_decode_heads(thk, ctx, H, Hkv, D):
    rng = np.random.default_rng(H * D)
    p = Pair(thk, ctx, 333, H, Hkv, D)
    p.append(rows(rng, 333, Hkv, D), 0)
    p.check(rng.standard_normal((1, H, D)).astype(np.float32), 332, mass=np.zeros((Hkv, 333), np.float32), decode=True)


@pytest.mark.parametrize("n_past,M", [(0, 1), (0, 2), (0, 17), (0, 64), (0, 130), (1, 3), (15, 16), (63, 2), (64, 64), (300, 5), (511, 33), (1000, 100)])
@pytest.mark.parametrize("H,Hkv,D", [(8, 8, 64), (4, 4, 128), (8, 2, 128), (20, 1, 128), (3, 3, 256)])
def test_prefill(thk, ctx, H, Hkv, D, n_past, M):
    rng = np.random.default_rng(n_past * 31 + M + H)
    T = n_past + M
    p = Pair(thk, ctx, T + 2, H, Hkv, D)
    p.append(rows(rng, T, Hkv, D), 0)
    q = rng.standard_normal((M, H, D)).astype(np.float32)
    p.check(q, n_past, mass=rng.random((Hkv, T + 2)).astype(np.float32))
    p.check(q, n_past)


@pytest.mark.parametrize("H,Hkv,D", SHAPES)
def test_prefill_heads(thk, ctx, H, Hkv, D):
    rng = np.random.default_rng(H * D + 1)
    p = Pair(thk, ctx, 200, H, Hkv, D)
    p.append(rows(rng, 200, Hkv, D), 0)
    p.check(rng.standard_normal((75, H, D)).astype(np.float32), 125, mass=np.zeros((Hkv, 200), np.float32))


def test_prefill_rows_beyond_one_slab(thk, ctx):
    """More rows than one launch takes: the weights of later slabs add to the earlier ones, positions ahead of the first slab included."""
    rng = np.random.default_rng(9)
    H, Hkv, D, n_past, M = 4, 2, 64, 33, 2048 + 77
    p = Pair(thk, ctx, n_past + M + 3, H, Hkv, D)
    p.append(rows(rng, n_past + M, Hkv, D), 0)
    p.check(rng.standard_normal((M, H, D)).astype(np.float32), n_past, mass=rng.random((Hkv, n_past + M + 3)).astype(np.float32))


def test_decode_equals_prefill_of_one(thk, ctx):
    rng = np.random.default_rng(10)
    p = Pair(thk, ctx, 400, 8, 4, 128)
    p.append(rows(rng, 400, 4, 128), 0)
    q = rng.standard_normal((1, 8, 128)).astype(np.float32)
    assert np.array_equal(p.attend(q, 399, decode=True)[0], p.attend(q, 399)[0])


def test_mass_in_place_and_repeatable(thk, ctx):
    rng = np.random.default_rng(11)
    p = Pair(thk, ctx, 300, 8, 4, 128)
    p.append(rows(rng, 300, 4, 128), 0)
    q, mass = rng.standard_normal((1, 8, 128)).astype(np.float32), rng.random((4, 300)).astype(np.float32)
    out, apart = p.attend(q, 199, mass, decode=True)
    dq, do, dm = ctx.from_numpy(q), ctx.alloc(q.nbytes), ctx.from_numpy(mass)
    p.dev.attn_decode(dq, 200, do, dm, dm)
    got = dm.download(np.float32, mass.shape)
    assert np.array_equal(got[:, :200], apart[:, :200]) and np.array_equal(got[:, 200:], mass[:, 200:])
    assert np.array_equal(do.download(np.float32, q.shape), out)
    for _ in range(5):
        again, m = p.attend(q, 199, mass, decode=True)
        assert np.array_equal(again, out) and np.array_equal(m, apart)


def test_peaked_and_flat_scores(thk, ctx):
    """One score far above the rest, scores all alike, and values of very different size in one tile."""
    rng = np.random.default_rng(12)
    H, D, T = 4, 128, 700
    x = rows(rng, T, H, D, spread=False)
    q = rng.standard_normal((1, H, D)).astype(np.float32)
    x[0, 333] = q[0] * 3
    p = Pair(thk, ctx, T, H, H, D)
    p.append(x, 0)
    p.check(q * 4, T - 1, decode=True)
    x[0] = 0
    p.append(x, 0)
    p.check(q, T - 1, mass=np.zeros((H, T), np.float32), decode=True)
    x = rows(rng, T, H, D)
    x[1, 16:32] *= np.float32(1e6)
    x[1, 32:48] *= np.float32(1e-6)
    x[1, 48:64] = 0
    p.append(x, 0)
    p.check(q, T - 1, decode=True)
    p.check(np.repeat(q, 3, 0), T - 3)


@pytest.mark.parametrize("what", ["k", "v", "inf_k"])
def test_nan_reaches_only_rows_that_see_it(thk, ctx, what):
    rng = np.random.default_rng(13)
    H, Hkv, D, T = 8, 4, 64, 150
    x = rows(rng, T, Hkv, D)
    x[1 if what == "v" else 0, 100, 2, 5] = np.inf if what == "inf_k" else np.nan
    p = Pair(thk, ctx, T, H, Hkv, D)
    p.append(x, 0)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    for out in (p.attend(q, 0)[0], np.concatenate([p.attend(q[t:t + 1], t, decode=True)[0] for t in range(88, 104)])):
        first = 0 if len(out) == T else 88
        bad = np.isnan(out).all(2)
        assert np.array_equal(np.isnan(out).any(2), bad)
        seen = np.arange(first, first + len(out)) >= 96            # the block of position 100 starts at 96
        exp = seen[:, None] & (np.arange(H) // 2 == 2)[None]
        assert np.array_equal(bad, exp)
    clean = p.ref.values(0, 96)
    eo, _, to, _ = attention(clean, q[:96], 0)
    assert np.all(np.abs(p.attend(q, 0)[0][:96] - eo) <= to)
    if what == "v":                                                # a NaN value does not touch the weights
        mass = np.zeros((Hkv, T), np.float32)
        _, m = p.attend(q, 0, mass)
        val = p.ref.values(0, T)
        val[1] = 0
        _, em, _, tm = attention(val, q, 0, mass)
        assert np.all(np.abs(m - em) <= tm)


@pytest.mark.parametrize("H,Hkv,D,T", [(8, 4, 64, 150), (32, 32, 128, 300), (64, 64, 64, 200), (24, 8, 256, 120)])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_odd_queries(thk, ctx, H, Hkv, D, T, bad):
    """A query that is not finite gives NaN in its own row and on the weights of the positions it sees, nowhere else; a query of zeros gives the mean."""
    rng = np.random.default_rng(T + D)
    p = Pair(thk, ctx, T, H, Hkv, D)
    p.append(rows(rng, T, Hkv, D), 0)
    q = rng.standard_normal((T, H, D)).astype(np.float32)
    r, h, z = T // 2, H - 2, T - 3
    q[z] = 0
    mass = rng.random((Hkv, T)).astype(np.float32)
    clean = q.copy()
    q[r, h, 5] = bad
    eo, em, to, tm = attention(p.ref.values(0, T), clean, 0, mass)
    out, m = p.attend(q, 0, mass)
    nan = np.zeros((T, H), bool)
    nan[r, h] = True
    assert np.array_equal(np.isnan(out).any(2), nan) and np.isnan(out[r, h]).all()
    assert np.all((np.abs(out - eo) <= to)[~nan])
    touched = np.zeros((Hkv, T), bool)
    touched[h * Hkv // H, :r + 1] = True
    assert np.array_equal(np.isnan(m), touched)
    late = np.zeros((Hkv, T), bool)
    late[:, r + 1:] = True
    assert np.all((np.abs(m - em) <= tm)[late | ~touched])
    for t in (r, z):                                               # the same rows as single tokens
        out, m = p.attend(q[t:t + 1], t, mass, decode=True)
        assert np.array_equal(np.isnan(out[0]).any(1), nan[t]) and np.all((np.abs(out[0] - eo[t]) <= to[t])[~nan[t]])
        assert np.array_equal(np.isnan(m), touched & nan.any(1)[t]) and np.all(m[:, t + 1:] == 7.0)


def test_garbage_behind_the_last_position(thk, ctx):
    """Positions at and after T hold infinities and NaN: no row reads them."""
    rng = np.random.default_rng(14)
    p = Pair(thk, ctx, 256, 4, 2, 128)
    x = rows(rng, 256, 2, 128)
    x[:, 160:] = np.nan
    p.append(x, 0)
    q = rng.standard_normal((40, 4, 128)).astype(np.float32)
    p.ref.scale = np.nan_to_num(p.ref.scale)
    p.check(q, 120)
    for T in (1, 64, 130, 160):
        p.check(q[:1], T - 1, mass=np.zeros((2, 256), np.float32), decode=True)


@pytest.mark.parametrize("T,keep,sink,recent", [(1, 1, 0, 0), (40, 1, 0, 0), (40, 40, 0, 0), (64, 33, 4, 8), (500, 250, 4, 32), (300, 20, 10, 10), (300, 16, 16, 0), (1500, 1024, 0, 1),
                                                (2500, 100, 1, 7), (257, 256, 0, 0), (1024, 1000, 0, 0), (1025, 513, 3, 500), (4097, 700, 0, 64)])
@pytest.mark.parametrize("Hkv,D", [(3, 128), (2, 64), (1, 256)])
def test_evict(thk, ctx, Hkv, D, T, keep, sink, recent):
    rng = np.random.default_rng(T + keep + D)
    p, dst = Pair(thk, ctx, T + 4, Hkv, Hkv, D), Pair(thk, ctx, keep + 9, Hkv, Hkv, D)
    p.append(rows(rng, T, Hkv, D), 0)
    mass = np.exp(rng.standard_normal((Hkv, T + 4)) * 2).astype(np.float32)
    mass[:, ::5] = np.round(mass[:, ::5])                                           # ties
    mass[0, :T // 3] = 0
    dm, mo, kept = ctx.from_numpy(mass), ctx.from_numpy(np.full((Hkv, keep + 9), 7, np.float32)), ctx.alloc(Hkv * keep * 4)
    p.dev.evict(dst.dev, T, keep, sink, recent, dm, mo, kept)
    ek, em = p.ref.evict(dst.ref, T, keep, sink, recent, mass)
    assert np.array_equal(kept.download(np.int32, (Hkv, keep)), ek)
    got = mo.download(np.float32, (Hkv, keep + 9))
    assert np.array_equal(got[:, :keep], em) and np.all(got[:, keep:] == 7)
    assert np.array_equal(dst.read(0, keep), dst.ref.values(0, keep))
    assert np.array_equal(p.read(0, T), p.ref.values(0, T))                         # the source stays
    dst.append(rows(rng, 5, Hkv, D), keep)                                          # and the destination goes on
    assert np.array_equal(dst.read(0, keep + 5), dst.ref.values(0, keep + 5))


@pytest.mark.parametrize("T,keep,Hkv", [(32768, 9000, 2), (32769, 20011, 2), (70001, 5, 2), (140000, 139999, 2), (33001, 4500, 44), (50002, 1234, 30), (1 << 20, 70000, 1), (40001, 3, 2), (32001, 3, 2), (33333, 33333, 2)])
@pytest.mark.parametrize("sink,recent", [(1, 2), (0, 0), (700, 20000)])
def test_evict_long(thk, ctx, T, keep, Hkv, sink, recent):
    """The selection's other ranges: positions and weights only (the values of a few kept rows)."""
    sink, recent = min(sink, keep // 2), min(recent, keep - min(sink, keep // 2))
    rng = np.random.default_rng(T)
    kv, dst = thk.KvCache8(ctx, T, Hkv, Hkv, 64), thk.KvCache8(ctx, keep, Hkv, Hkv, 64)
    mass = np.exp(rng.standard_normal((Hkv, T)) * 3).astype(np.float32)
    mass[Hkv // 2:] = np.round(mass[Hkv // 2:])                                     # ties by the thousand
    dm, mo, kept = ctx.from_numpy(mass), ctx.alloc(Hkv * keep * 4), ctx.alloc(Hkv * keep * 4)
    kv.evict(dst, T, keep, sink, recent, dm, mo, kept)
    got, gm = kept.download(np.int32, (Hkv, keep)), mo.download(np.float32, (Hkv, keep))
    for h in range(Hkv):
        mid = np.arange(sink, T - recent)
        heavy = mid[np.argsort(-mass[h, sink:T - recent].astype(np.float64), kind="stable")][:keep - sink - recent]
        exp = np.concatenate([np.arange(sink), np.sort(heavy), np.arange(T - recent, T)])
        assert np.array_equal(got[h], exp)
        assert np.array_equal(gm[h], mass[h][exp])
    kv.close()
    dst.close()


def test_evict_odd_weights(thk, ctx):
    """NaN is lightest, infinity heaviest, -0 equals 0, negative weights are ordered."""
    rng = np.random.default_rng(16)
    T, keep = 100, 30
    p, dst = Pair(thk, ctx, T, 2, 2, 64), Pair(thk, ctx, T, 2, 2, 64)
    p.append(rows(rng, T, 2, 64), 0)
    mass = np.zeros((2, T), np.float32)
    mass[0, ::3], mass[0, 1::9], mass[0, 50:60], mass[0, 7] = np.nan, -0.0, 1.0, np.inf
    mass[1] = -rng.random(T)
    mass[1, 3] = -np.inf
    kept = ctx.alloc(2 * keep * 4)
    p.dev.evict(dst.dev, T, keep, 0, 0, ctx.from_numpy(mass), None, kept)
    ek, _ = p.ref.evict(dst.ref, T, keep, 0, 0, mass)
    assert np.array_equal(kept.download(np.int32, (2, keep)), ek)


def test_generation_over_a_budget(thk, ctx):
    """Prompt, single tokens, eviction into the spare cache, on and on: the operators as a decode loop uses them, against the plain form."""
    rng = np.random.default_rng(17)
    H, Hkv, D, n_ctx, keep = 8, 4, 64, 160, 70
    cur, spare = Pair(thk, ctx, n_ctx, H, Hkv, D), Pair(thk, ctx, n_ctx, H, Hkv, D)
    x = rows(rng, 100, Hkv, D)
    cur.append(x, 0)
    mass, T, evictions = np.zeros((Hkv, n_ctx), np.float32), 100, 0
    q = rng.standard_normal((100, H, D)).astype(np.float32)
    cur.check(q, 0, mass=mass)
    _, mass = cur.attend(q, 0, mass)
    mass[:, T:] = 0
    for step in range(150):
        if T == n_ctx:
            kept, mo = ctx.alloc(Hkv * keep * 4), ctx.from_numpy(np.zeros((Hkv, n_ctx), np.float32))
            cur.dev.evict(spare.dev, T, keep, 4, 20, ctx.from_numpy(mass), mo, kept)
            ek, _ = cur.ref.evict(spare.ref, T, keep, 4, 20, mass)
            assert np.array_equal(kept.download(np.int32, (Hkv, keep)), ek)
            mass, T = mo.download(np.float32, mass.shape), keep
            cur, spare = spare, cur
            evictions += 1
        cur.append(rows(rng, 1, Hkv, D), T)
        T += 1
        q = rng.standard_normal((1, H, D)).astype(np.float32)
        if step % 7 == 0 or T in (n_ctx, keep + 1):
            cur.check(q, T - 1, mass=mass, decode=True)
        _, m = cur.attend(q, T - 1, mass, decode=True)
        mass[:, :T] = m[:, :T]
        assert np.array_equal(cur.read(0, T), cur.ref.values(0, T))
    assert evictions == 1 or evictions == 2


def test_offsets_beyond_32_bits(thk, ctx):
    """Codes behind 2^31 bytes of the K array: the last head's positions of a long, wide cache."""
    rng = np.random.default_rng(18)
    H, D, T, piece = 64, 256, 140_000, 2_000
    kv = thk.KvCache8(ctx, T, H, H, D)
    k, v = rng.standard_normal((2, piece, H, D), np.float32)
    vals = RefCache(piece, 1, D)
    vals.append(k[:, -1:], v[:, -1:], 0)
    vals = vals.values()
    dk, dv, ko = ctx.from_numpy(k), ctx.from_numpy(v), ctx.alloc(16 * H * D * 4)
    for at in range(0, T, piece):
        kv.append(dk, dv, at, piece)
    kv.read(T - 16, 16, ko, None)
    assert np.array_equal(ko.download(np.float32, (16, H, D))[:, -1], vals[0, -16:, 0])
    q = rng.standard_normal((1, H, D), np.float32)
    dq, out = ctx.from_numpy(q), ctx.alloc(H * D * 4)
    kv.attn_decode(dq, T, out)
    exp, _, tol, _ = attention(vals, q[:, -1:], piece - 1)            # the same rows over and over: the attention over one piece
    got = out.download(np.float32, (H, D))[-1]
    assert np.linalg.norm(got - exp[0, 0]) / np.linalg.norm(exp[0, 0]) < 1e-5
    kv.close()


@pytest.mark.parametrize("H,Hkv,D", [(64, 64, 64), (64, 64, 128), (128, 64, 64), (48, 48, 256)])
@pytest.mark.parametrize("M", [129, 200, 300, 600, 700])
def test_prefill_many_columns(thk, ctx, H, Hkv, D, M):
    """Every shape of the many-rows kernel: one or two groups of waves, narrow and wide columns, columns that end inside one."""
    rng = np.random.default_rng(M + H + D)
    n_past = M % 97
    T = n_past + M
    p = Pair(thk, ctx, T + 1, H, Hkv, D)
    p.append(rows(rng, T, Hkv, D), 0)
    p.check(rng.standard_normal((M, H, D)).astype(np.float32), n_past, mass=rng.random((Hkv, T + 1)).astype(np.float32))


def test_decode_of_many_heads(thk, ctx):
    """More K/V heads than the positions are split for: a single row on the many-rows kernel."""
    rng = np.random.default_rng(21)
    p = Pair(thk, ctx, 131, 600, 600, 64)
    p.append(rows(rng, 131, 600, 64), 0)
    for T in (1, 64, 131):
        p.check(rng.standard_normal((1, 600, 64)).astype(np.float32), T - 1, mass=np.zeros((600, 131), np.float32), decode=True)


@pytest.mark.parametrize("H,Hkv,T", [(260, 260, 4100), (400, 400, 130), (1024, 1, 700), (1024, 512, 65)])
def test_decode_without_a_split(thk, ctx, H, Hkv, T):
    """Column groups enough to fill the chip, or nearly: one part, weights counted in the launch (to 4096 positions) or by one of their own."""
    rng = np.random.default_rng(H + T)
    p = Pair(thk, ctx, T, H, Hkv, 64)
    p.append(rows(rng, T, Hkv, 64), 0)
    p.check(rng.standard_normal((1, H, 64)).astype(np.float32), T - 1, mass=rng.random((Hkv, T)).astype(np.float32), decode=True)
    p.check(rng.standard_normal((3, H, 64)).astype(np.float32), T - 3, mass=rng.random((Hkv, T)).astype(np.float32))


@pytest.mark.parametrize("T", [4095, 4096, 4097, 9001])
@pytest.mark.parametrize("H,Hkv,D", [(2, 2, 64), (9, 3, 128), (16, 1, 128), (32, 2, 64), (17, 1, 64), (4, 2, 256)])
def test_weights_of_longer_caches(thk, ctx, H, Hkv, D, T):
    """Weights counted by the launch itself, by the joining launch and (groups of more than 16 heads) by one of their own."""
    rng = np.random.default_rng(T + H)
    p = Pair(thk, ctx, T + 3, H, Hkv, D)
    p.append(rows(rng, T, Hkv, D), 0)
    q = rng.standard_normal((1, H, D)).astype(np.float32)
    p.check(q, T - 1, mass=rng.random((Hkv, T + 3)).astype(np.float32), decode=True)
    p.check(q, T - 1, decode=True)


@pytest.mark.parametrize("H,Hkv,D,pieces", [(16, 16, 128, 17), (64, 32, 64, 17), (8, 8, 256, 17), (32, 2, 128, 130)])
def test_long_cache_past_the_caches(thk, ctx, H, Hkv, D, pieces):
    """Codes of 64 MB and more: a piece of 1024 positions over and over, so that out is the piece's and each weight a share of the piece's."""
    rng = np.random.default_rng(D + pieces)
    n = 1024
    T = n * pieces
    x = rows(rng, n, Hkv, D)
    ref = RefCache(n, Hkv, D)
    ref.append(x[0], x[1], 0)
    kv = thk.KvCache8(ctx, T, H, Hkv, D)
    dk, dv = ctx.from_numpy(x[0]), ctx.from_numpy(x[1])
    for at in range(0, T, n):
        kv.append(dk, dv, at, n)
    q = rng.standard_normal((1, H, D)).astype(np.float32)
    dm, do = ctx.from_numpy(np.zeros((Hkv, T), np.float32)), ctx.alloc(q.nbytes)
    kv.attn_decode(ctx.from_numpy(q), T, do, dm, dm)
    eo, em, to, tm = attention(ref.values(), q, n - 1, np.zeros((Hkv, n), np.float32))
    more = (T - n) / 16 * EPS                                       # the longer sums' share of the bounds
    out, m = do.download(np.float32, q.shape), dm.download(np.float32, (Hkv, pieces, n))
    assert np.all(np.abs(out - eo) <= to + 2 * more * np.abs(ref.values()[1]).max())
    assert np.linalg.norm(out - eo) / np.linalg.norm(eo) < 1e-5
    assert np.all(np.abs(m * pieces - em[:, None]) <= (tm + more * em)[:, None] + 1e-12)
    kv.close()


class Hip:
    """The HIP runtime the library runs on: streams and graphs for the tests."""

    def __init__(self):
        path = next(line.split()[-1] for line in open("/proc/self/maps") if "libamdhip64.so" in line)
        self.lib = C.CDLL(path)

    def __getattr__(self, name):
        fn = getattr(self.lib, name)

        def call(*args):
            rc = fn(*args)
            assert rc == 0, (name, rc)

        return call


def test_captured_and_replayed(thk):
    """Append, attention with weights and eviction in one graph, replayed with eager work between; every replay against the eager result."""
    rng = np.random.default_rng(19)
    H, Hkv, D, T, keep, M = 8, 4, 128, 300, 128, 20
    with thk.Context(0) as c:
        hip, st = Hip(), C.c_void_p(c.stream)
        kv, to = thk.KvCache8(c, T + 8, H, Hkv, D), thk.KvCache8(c, keep, H, Hkv, D)
        x = rows(rng, T, Hkv, D)
        k, v, k1, v1 = (c.from_numpy(a) for a in (x[0], x[1], x[0, :1], x[1, :1]))
        q, qm = c.from_numpy(rng.standard_normal((1, H, D)).astype(np.float32)), c.from_numpy(rng.standard_normal((M, H, D)).astype(np.float32))
        mass, m1 = c.from_numpy(rng.random((Hkv, T + 8)).astype(np.float32)), c.alloc(Hkv * (T + 8) * 4)
        outs = [m1, c.alloc(Hkv * (T + 8) * 4), c.alloc(Hkv * keep * 4), c.alloc(H * D * 4), c.alloc(Hkv * keep * 4), c.alloc(keep * Hkv * D * 4), c.alloc(M * H * D * 4)]
        _, m2, m3, out, kept, ko, om = outs
        kv.append(k, v, 0, T)

        def step():
            kv.append(k1, v1, T, 1)
            kv.attn_decode(q, T + 1, out, mass, m1)
            kv.attn_prefill(qm, T + 1 - M, M, om, m1, m2)
            kv.evict(to, T + 1, keep, 4, 16, m2, m3, kept)
            to.read(0, keep, ko, None)

        step()
        c.sync()
        graph, run = C.c_void_p(), C.c_void_p()
        hip.hipStreamBeginCapture(st, 2)                               # relaxed: other threads' calls do not matter here
        try:
            step()
            with pytest.raises(thk.ThkError, match="captured"):
                thk.KvCache8(c, 16, 4, 4, 64)
        finally:
            hip.hipStreamEndCapture(st, C.byref(graph))
        hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0))
        for i in range(5):
            for buf, shape in ((k1, (Hkv, D)), (v1, (Hkv, D)), (q, (H, D)), (qm, (M, H, D))):
                buf.upload(rng.standard_normal(shape).astype(np.float32))
            for o in outs:
                o.upload(np.zeros(o.nbytes // 4, np.float32))
            hip.hipGraphLaunch(run, st)
            c.sync()
            got = [o.download(np.int32, o.nbytes // 4) for o in outs]
            for o in outs:
                o.upload(np.zeros(o.nbytes // 4, np.float32))
            step()
            c.sync()
            for a, o in zip(got, outs):
                assert np.array_equal(a, o.download(np.int32, o.nbytes // 4)), i
        hip.hipGraphExecDestroy(run)
        hip.hipGraphDestroy(graph)
        kv.close()
        to.close()


def test_captured_long_prompt_and_eviction(thk):
    """The kernels that need more LDS than a launch gets unasked, and the selection in slices, first called inside a capture."""
    rng = np.random.default_rng(22)
    H, D, T, M, keep = 24, 64, 33000, 500, 700
    with thk.Context(0) as c:
        hip, st = Hip(), C.c_void_p(c.stream)
        kv, a, b = thk.KvCache8(c, T, H, H, D), thk.KvCache8(c, keep, H, H, D), thk.KvCache8(c, keep, H, H, D)
        x = rng.standard_normal((2, 1000, H, D), np.float32)
        k, v = c.from_numpy(x[0]), c.from_numpy(x[1])
        for at in range(0, T, 1000):
            kv.append(k, v, at, 1000)
        q, mass = c.from_numpy(rng.standard_normal((M, H, D)).astype(np.float32)), c.from_numpy(np.exp(rng.standard_normal((H, T)) * 2).astype(np.float32))
        outs = [c.alloc(M * H * D * 4), c.alloc(H * T * 4)] + [c.alloc(H * keep * 4) for _ in range(4)]
        om, m1, ka, ma, kb, mb = outs

        def step():
            kv.attn_prefill(q, 900, M, om, mass, m1)
            kv.evict(a, T, keep, 4, 16, mass, ma, ka)
            kv.evict(b, 20000, keep, 0, 0, mass, mb, kb)

        c.sync()
        graph, run = C.c_void_p(), C.c_void_p()
        hip.hipStreamBeginCapture(st, 2)
        try:
            step()
        finally:
            hip.hipStreamEndCapture(st, C.byref(graph))
        hip.hipGraphInstantiate(C.byref(run), graph, None, None, C.c_size_t(0))
        for i in range(3):
            q.upload(rng.standard_normal((M, H, D)).astype(np.float32))
            mass.upload(np.exp(rng.standard_normal((H, T)) * 2).astype(np.float32))
            for o in outs:
                o.upload(np.zeros(o.nbytes // 4, np.float32))
            hip.hipGraphLaunch(run, st)
            c.sync()
            got = [o.download(np.int32, o.nbytes // 4) for o in outs]
            for o in outs:
                o.upload(np.zeros(o.nbytes // 4, np.float32))
            step()
            c.sync()
            for g, o in zip(got, outs):
                assert np.array_equal(g, o.download(np.int32, o.nbytes // 4)), i
        hip.hipGraphExecDestroy(run)
        hip.hipGraphDestroy(graph)
        for cache in (kv, a, b):
            cache.close()


def test_two_caches_on_two_streams(thk):
    """Caches of different contexts share nothing: overlapping work on two streams gives the results of one after the other."""
    H, D, T, M = 8, 128, 2000, 40
    ctxs = [thk.Context(0) for _ in range(2)]
    pairs = []
    for i, c in enumerate(ctxs):
        rng = np.random.default_rng(20 + i)
        p = thk.KvCache8(c, T, H, H, D)
        x = rows(rng, T, H, D)
        k, v = c.from_numpy(x[0]), c.from_numpy(x[1])
        p.append(k, v, 0, T)
        c.sync()
        pairs.append((p, c.from_numpy(rng.standard_normal((M, H, D)).astype(np.float32)), c.alloc(M * H * D * 4), c.alloc(H * T * 4)))

    def run(sync):
        for c, (p, q, o, m) in zip(ctxs, pairs):
            m.upload(np.zeros(H * T, np.float32))
        for c, (p, q, o, m) in zip(ctxs, pairs):
            for _ in range(3):
                p.attn_prefill(q, T - M, M, o, m, m)
                p.attn_decode(q, T, o, m, m)
            if sync:
                c.sync()
        for c in ctxs:
            c.sync()
        return [(o.download(np.float32, M * H * D), m.download(np.float32, H * T)) for _, _, o, m in pairs]

    apart = run(True)
    for _ in range(3):
        for (o1, m1), (o2, m2) in zip(apart, run(False)):
            assert np.array_equal(o1, o2) and np.array_equal(m1, m2)
    for p, *_ in pairs:
        p.close()
    del pairs
    for c in ctxs:
        c.close()


def test_refusals(thk, ctx):
    """Every refusal is an error before any launch (the same checks run without a GPU in test_kv8_host.py)."""
    for bad in [(0, 4, 4, 64), (10, 4, 3, 64), (10, 4, 4, 96), (10, 0, 4, 64), ((1 << 26) + 1, 4, 4, 64)]:
        with pytest.raises(thk.ThkError, match="thk_kv8_create"):
            thk.KvCache8(ctx, *bad)
    kv, to = thk.KvCache8(ctx, 100, 8, 4, 64), thk.KvCache8(ctx, 50, 8, 4, 64)
    other = thk.KvCache8(ctx, 100, 8, 8, 64)
    d = ctx.alloc(1 << 20)
    for call, text in [(lambda: kv.append(d, d, 99, 2), "outside the cache"), (lambda: kv.append(d, d, -1, 2), "bad arguments"), (lambda: kv.append(d, d, 0, 0), "bad arguments"),
                       (lambda: kv.append(None, d, 0, 1), "bad arguments"), (lambda: kv.append(d.ptr + 4, d, 0, 1), "aligned"), (lambda: kv.read(0, 101, d, d), "outside"),
                       (lambda: kv.attn_decode(d, 0, d), "outside"), (lambda: kv.attn_decode(d, 101, d), "outside"), (lambda: kv.attn_decode(d, 5, d, d, None), "go together"),
                       (lambda: kv.attn_prefill(d, 90, 11, d), "outside"), (lambda: kv.attn_prefill(d, 0, 0, d), "outside"), (lambda: kv.evict(kv, 50, 20, 0, 0, d, None, d), "same cache"),
                       (lambda: kv.evict(to, 100, 51, 0, 0, d, None, d), "T=100"), (lambda: kv.evict(to, 100, 20, 15, 6, d, None, d), "exceed"),
                       (lambda: kv.evict(other, 100, 20, 0, 0, d, None, d), "differ"), (lambda: kv.evict(to, 100, 20, 0, 0, d, d, d), "mass_out")]:
        with pytest.raises(thk.ThkError, match=text):
            call()
