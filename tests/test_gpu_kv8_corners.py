"""The 8-bit K/V cache where its kernels' ranges end, beginning with every number of parts a long axis is cut into.  Plain form and bounds:
tests/kv8_ref.py; caches and their plain twins: test_gpu_kv8.py."""
import numpy as np
import pytest

from kv8_ref import EPS, attention
from test_gpu_kv8 import Pair, rows

pytestmark = pytest.mark.gpu

# heads, K/V heads, head dim, rows: the kernel for many rows in each of its shapes (more than 512 groups of 16 columns x K/V heads)
MANY = [(64, 64, 64, 129), (64, 64, 128, 300), (64, 64, 64, 600), (64, 64, 64, 700), (48, 48, 256, 200)]


def towards(rng, x, q, lo, gap):
    """Keys [lo, end) of every K/V head get scores about `gap` above the others' for the head's first query."""
    G, D = q.shape[0] // x.shape[2], q.shape[1]
    for j in range(x.shape[2]):
        u = q[j * G]
        x[0, lo:, j] += u * (gap * np.sqrt(D) / (u @ u))


@pytest.mark.parametrize("H,Hkv,D,step", [(6, 1, 64, 512), (4, 1, 128, 512), (4, 1, 256, 256)])
def test_every_number_of_parts(thk, ctx, H, Hkv, D, step):
    """A single row over 2 .. 64 parts (a part per `step` positions), joined in the launch or by one of its own, distinct values everywhere."""
    rng = np.random.default_rng(D)
    p = Pair(thk, ctx, 64 * step, H, Hkv, D)
    p.append(rows(rng, 64 * step, Hkv, D), 0)
    val, ld = p.ref.values(), 64 * step
    for parts in range(2, 65):
        T = parts * step - int(rng.integers(0, step - 64))
        q = rng.standard_normal((1, H, D)).astype(np.float32)
        mass = rng.random((Hkv, ld)).astype(np.float32)
        eo, em, to, tm = attention(val[:, :T], q, T - 1, mass)
        for m in (None, mass):
            out, got = p.attend(q, T - 1, m, decode=True)
            assert np.all(np.abs(out - eo) <= to), (parts, T, float((np.abs(out - eo) / to).max()))
        assert np.all(np.abs(got[:, :T] - em) <= tm), (parts, T)


@pytest.mark.parametrize("H,Hkv,D,T,M", [(16, 1, 64, 8500, 1), (30, 15, 64, 9001, 1), (32, 4, 128, 16500, 1), (16, 2, 128, 20500, 1), (8, 8, 64, 8600, 5), (16, 1, 64, 10300, 3), (4, 2, 128, 16700, 19)])
def test_newest_positions_of_a_long_cache(thk, ctx, H, Hkv, D, T, M):
    """The last part holds a large share of the weight: odd numbers of parts, single rows and a few rows."""
    rng = np.random.default_rng(T)
    p = Pair(thk, ctx, T + 3, H, Hkv, D)
    x, q = rows(rng, T, Hkv, D), rng.standard_normal((M, H, D)).astype(np.float32)
    towards(rng, x, q[M - 1], T - 40, 6)
    p.append(x, 0)
    p.check(q, T - M, decode=M == 1)
    p.check(q, T - M, mass=rng.random((Hkv, T + 3)).astype(np.float32), decode=M == 1)


@pytest.mark.parametrize("H,Hkv,D,M", MANY + [(8, 8, 64, 3), (8, 2, 128, 1), (40, 1, 64, 4)])
@pytest.mark.parametrize("fq,fk", [(2.0 ** -60, 2.0 ** -75), (2.0 ** -63, 2.0 ** -63), (2.0 ** -95, 2.0 ** -95), (2.0 ** -20, 2.0 ** -98)])
def test_small_queries_and_keys(thk, ctx, H, Hkv, D, M, fq, fk):
    """Queries and keys whose product leaves f32's range downwards: every score is 0, output and weights those of the mean."""
    rng = np.random.default_rng(M + D)
    n_past = 70
    T = n_past + M
    x, q = rows(rng, T, Hkv, D, spread=False), (rng.standard_normal((M, H, D)) * fq).astype(np.float32)
    x[0] *= np.float32(fk)
    p = Pair(thk, ctx, T + 1, H, Hkv, D)
    p.append(x, 0)
    mass = rng.random((Hkv, T + 1)).astype(np.float32)
    p.check(q, n_past, mass=mass, decode=M == 1)
    p.check(q, n_past, decode=M == 1)


def tops(rng, H, Hkv, D, M, n_past, gap, at):
    """q and rows in which positions [at, at + 16) score about `gap` above all others, for every row and head."""
    u = rng.standard_normal((Hkv, D))
    G = H // Hkv
    q = (np.repeat(u, G, 0)[None] + 0.1 * rng.standard_normal((M, H, D))).astype(np.float32)
    x = rows(rng, n_past + M, Hkv, D, spread=False)
    x[0] *= 0.1
    x[0, at:at + 16] = u * (gap * np.sqrt(D) / (u * u).sum(1))[:, None]
    return q, x


@pytest.mark.parametrize("H,Hkv,D,M", MANY + [(8, 8, 64, 3), (8, 2, 128, 1)])
@pytest.mark.parametrize("gap", [60, 82, 95, 250])
def test_zero_values_under_the_top_scores(thk, ctx, H, Hkv, D, M, gap):
    """The block with nearly all of the weight has zero values: the output is the others' small share, or nothing, and not NaN."""
    rng = np.random.default_rng(M + gap)
    n_past = 150
    q, x = tops(rng, H, Hkv, D, M, n_past, gap, 16)
    x[1, 16:32] = 0
    p = Pair(thk, ctx, n_past + M, H, Hkv, D)
    p.append(x, 0)
    out, _ = p.attend(q, n_past)
    eo, _, to, _ = attention(p.ref.values(), q, n_past)
    assert np.all(np.abs(out - eo) <= to)
    if gap == 60:                                                    # the small share is right, too, to its scores' error
        share = np.linalg.norm(out.astype(np.float64) - eo) / np.linalg.norm(eo)
        e = (D + 16) * EPS * np.abs(q).max() * np.abs(p.ref.values()[0]).sum(2).max() / np.sqrt(D)
        assert share <= 2 * e + 1e-5, (share, e)


# the kernel for few rows: the same wave's next tile; the one for many rows: any
@pytest.mark.parametrize("H,Hkv,D,M,n_past,lo", [(*m, 300, 128) for m in MANY] + [(32, 32, 64, 70, 1200, 512), (64, 32, 128, 33, 1200, 512), (32, 32, 256, 65, 900, 256)])
@pytest.mark.parametrize("big,gap", [(1e34, 200), (1e36, 200), (1e36, 81)])
def test_large_values_of_next_to_no_weight(thk, ctx, H, Hkv, D, M, n_past, lo, big, gap):
    """Values near the end of f32's range at positions of next to no weight: the product of the two is what counts, zero or not."""
    rng = np.random.default_rng(M)
    q, x = tops(rng, H, Hkv, D, M, n_past, gap, 16)
    x[1, lo:lo + 64] *= np.float32(big)
    p = Pair(thk, ctx, n_past + M, H, Hkv, D)
    p.append(x, 0)
    out, _ = p.attend(q, n_past)
    val = p.ref.values()
    eo, _, _, _ = attention(val, q, n_past)
    apart = val.copy()                                               # the bound of either part by itself
    apart[1, lo:lo + 64] = 0
    _, _, to, _ = attention(apart, q, n_past)
    e = (D + 16) * EPS * np.abs(q).max(2)[..., None] * np.repeat(np.abs(val[0]).sum(2).max(0), H // Hkv)[None, :, None] / np.sqrt(D)
    share = attention(np.stack([val[0], np.abs(val[1]) - np.abs(apart[1])]), q, n_past)[0]
    # the large values' part: weights good to their scores' error (twice) and to 2^-22 of the largest of their tile, whose 64 lie within a factor of 2
    to = to + share * (2 * e + 400 * EPS)
    assert np.all(np.abs(out - eo) <= to), float((np.abs(out - eo) / to).max())


@pytest.mark.parametrize("H,Hkv,D,M", MANY + [(8, 8, 64, 3), (8, 2, 128, 1), (4, 1, 64, 9)])
@pytest.mark.parametrize("down", [60, 100])
def test_values_near_the_least_block(thk, ctx, H, Hkv, D, M, down):
    """Values down to 2^-100, the least a block holds, under flat scores: as good, relative to them, as ordinary ones (a power of two changes no code)."""
    rng = np.random.default_rng(M + D)
    n_past = 2007
    x, q = rows(rng, n_past + M, Hkv, D, spread=False), (0.01 * rng.standard_normal((M, H, D))).astype(np.float32)
    p = Pair(thk, ctx, n_past + M, H, Hkv, D)
    p.append(x, 0)
    val = p.ref.values()
    one, _ = p.attend(q, n_past)
    x[1] *= np.float32(2.0 ** -down)
    p.append(x, 0)
    assert np.array_equal(p.ref.values()[1], val[1] * np.float32(2.0 ** -down))
    out, _ = p.attend(q, n_past)
    # a power of two changes no rounding above 2^-126; below, sums are rounded to 2^-149: once a tile of 64 and part, and at the end
    least = (n_past + M) / 16 * 2.0 ** -150 * 2.0 ** down
    off = np.abs(out.astype(np.float64) * 2.0 ** down - one)
    assert np.all(off <= 4 * EPS * np.abs(one) + least), float((off / (4 * EPS * np.abs(one) + least)).max())


@pytest.mark.parametrize("H,Hkv,D,M", MANY)
@pytest.mark.parametrize("what", ["k", "v"])
def test_many_rows_nan_reaches_only_rows_that_see_it(thk, ctx, H, Hkv, D, M, what):
    rng = np.random.default_rng(M + D)
    n_past, at, head = 20, 20 + M // 2, 5
    T = n_past + M
    x = rows(rng, T + 40, Hkv, D)
    x[1 if what == "v" else 0, at, head, 3] = np.nan
    x[:, T:] = np.nan                                                # and in the blocks behind the last position's
    p = Pair(thk, ctx, T + 40, H, Hkv, D)
    p.append(x[:, :T], 0)
    if T % 16 == 0:
        p.append(x[:, T:], T)
    else:
        p.append(x[:, T + 16 - T % 16:], T + 16 - T % 16)
    q, mass = rng.standard_normal((M, H, D)).astype(np.float32), rng.random((Hkv, T + 40)).astype(np.float32)
    out, m = p.attend(q, n_past, mass)
    first = at // 16 * 16                                            # the block's first position: the first row that sees it
    bad = (np.arange(M)[:, None] + n_past >= first) & (np.arange(H) == head)[None]
    assert np.array_equal(np.isnan(out).all(2), bad) and np.array_equal(np.isnan(out).any(2), bad)
    val = p.ref.values(0, T)
    val[1 if what == "v" else 0, first:first + 16, head] = 0
    eo, em, to, tm = attention(val, q, n_past, mass)
    assert np.all((np.abs(out - eo) <= to)[~bad])
    if what == "v":                                                  # the weights do not know of it
        assert np.all(np.abs(m[:, :T] - em) <= tm)
    else:
        nan = np.zeros((Hkv, T), bool)
        nan[head] = True
        assert np.array_equal(np.isnan(m[:, :T]), nan) and np.all((np.abs(m[:, :T] - em) <= tm)[~nan])
    assert np.all(m[:, T:] == 7.0)


def test_many_rows_in_slabs(thk, ctx):
    """Launches of the kernel for many rows and a last one of few, or of one: weights of later slabs add to earlier ones'."""
    rng = np.random.default_rng(31)
    H, D, n_past = 8, 64, 33
    for M in (2048 + 1, 2048 + 1100, 4096 + 21):
        p = Pair(thk, ctx, n_past + M + 3, H, H, D)
        p.append(rows(rng, n_past + M, H, D), 0)
        p.check(rng.standard_normal((M, H, D)).astype(np.float32), n_past, mass=rng.random((H, n_past + M + 3)).astype(np.float32))


# the many-rows kernel, a single row and few rows, one and several tiles a wave and parts
LARGE = MANY + [(8, 8, 64, 3), (8, 2, 128, 1), (40, 1, 64, 4), (300, 300, 64, 1)]


def one_hot(rng, thk, ctx, H, Hkv, D, M, n_past, big):
    """Scores around `big` and more, one position's above the next by more than that for every row -> cache, q, the position."""
    T, at = n_past + M, 37
    x = rows(rng, T, Hkv, D, spread=False)
    u = rng.standard_normal((Hkv, D))
    x[0] *= np.float32(big ** 0.5)
    x[0, at] = u * 20 * big ** 0.5
    q = (np.repeat(u, H // Hkv, 0)[None] * (1 + rng.random((M, 1, 1))) * big ** 0.5).astype(np.float32)
    p = Pair(thk, ctx, T, H, Hkv, D)
    p.append(x, 0)
    k = p.ref.values()[0].astype(np.float64)
    for j in range(Hkv):
        s = np.sort(q[:, j * (H // Hkv)].astype(np.float64) @ k[:, j].T / np.sqrt(D), 1)
        assert np.all(s[:, -1] - s[:, -2] > big)
    return p, q, at


@pytest.mark.parametrize("H,Hkv,D,M", LARGE)
@pytest.mark.parametrize("big,n_past", [(1e7, 90), (1e9, 90), (1e12, 90), (1e9, 1400)])
def test_scores_beyond_the_steps_of_f32(thk, ctx, H, Hkv, D, M, big, n_past):
    """Scores so large that f32 tells them apart by no less than 1 to 10^5: a row's weight is on its single largest one, whatever that was rounded to."""
    p, q, at = one_hot(np.random.default_rng(M + D), thk, ctx, H, Hkv, D, M, n_past, big)
    out, _ = p.attend(q, n_past, None, decode=M == 1)
    want = np.repeat(p.ref.values()[1, at], H // Hkv, 0)[None]
    # one weight of 1: held to 22 bits, its value by one product and one quotient
    assert np.all(np.abs(out - want) <= 16 * EPS * np.abs(want).max()), float(np.abs(out - want).max())


@pytest.mark.parametrize("H,Hkv,D,M", LARGE)
@pytest.mark.parametrize("big,n_past", [(1e7, 90), (1e9, 90), (1e12, 90), (1e9, 1400)])
def test_weights_of_scores_beyond_the_steps_of_f32(thk, ctx, H, Hkv, D, M, big, n_past):
    rng = np.random.default_rng(M + D)
    p, q, at = one_hot(rng, thk, ctx, H, Hkv, D, M, n_past, big)
    mass = rng.random((Hkv, n_past + M)).astype(np.float32)
    _, got = p.attend(q, n_past, mass, decode=M == 1)
    exp, G = mass.astype(np.float64), H // Hkv
    exp[:, at] += M * G
    # a weight of exp2(0) times 1 / 1, or of 0; at most an addition for each row and head of the group, exact among whole numbers, and the last one
    assert np.all(np.abs(got - exp) <= (M * G + 8) * EPS * exp), float(np.abs(got - exp).max())
