"""Attention over the 4-bit cache where its numbers are far apart: keys and values of very different sizes next to
each other, seen, hidden and of no weight; against 64 bits.

The bound is per key, so that a key of no weight allows no error. With p the probabilities and a stored number's parts
(code + 8) step + |offset - 8 step|, an output is off by at most
    sum p 2^-9 parts(v) + sum p 2 e |v - o| + 2^-8 |o|,    e = 2^-19 |scale| sum |q| parts(k) + 2^-18:
2^-9 for four roundings of 2^-11 (of a probability, of a value, and of both where they are small beside the largest),
e for a score's f32 sums and its exponential (a score that is off by d moves p to p (1 + d), and o by p d (v - o); twice
that, for the terms of second order), 2^-8 for the output's own rounding to bf16."""
import numpy as np
import pytest

import furiosa_opt_b200 as fb
from oracle import cache_ref as R
from test_gpu_kvcache import WIDE, _bf, _down, _m, _up

pytestmark = pytest.mark.gpu

F = np.float32


def _bound(q, ref, pages, q_len, n, scale, causal):
    """(o, bound) [T, Hq, D] of one sequence's queries."""
    T, Hq, D = q.shape
    group = Hq // ref.heads
    o, tol = np.zeros((T, Hq, D)), np.zeros((T, Hq, D))
    K, V, KA, VA = ref.values("k"), ref.values("v"), ref.parts("k"), ref.parts("v")
    for h in range(ref.heads):
        k, v, ka, va = (x[pages, h].reshape(-1, D)[:n] for x in (K, V, KA, VA))
        rows = slice(h * group, (h + 1) * group)
        for t in range(T):
            seen = max(0, n - q_len + t + 1) if causal else n
            if not seen:
                continue
            qd = q[t, rows].astype(np.float64)
            x = qd @ k[:seen].T * scale
            p = np.exp(x - x.max(-1, keepdims=True))
            p /= p.sum(-1, keepdims=True)
            e = 2.0 ** -19 * abs(scale) * (np.abs(qd) @ ka[:seen].T) + 2.0 ** -18
            o[t, rows] = p @ v[:seen]
            tol[t, rows] = 2.0 ** -9 * (p @ va[:seen]) + 2.0 ** -8 * np.abs(o[t, rows])
            for r, (pr, er) in enumerate(zip(p, e)):
                of = pr > 1e-30
                tol[t, h * group + r] += 2 * (pr[of] * er[of]) @ np.abs(v[:seen][of] - o[t, h * group + r])
    return o, tol


def _check(be, q, k, v, D, group, scale=None, causal=True, wide=False, page=16, slack=0.0):
    """q [T, H group, D] over k, v [n, H, D] (f32), the last T tokens; beside it a sequence of one ordinary token, which
    has nothing to do with it. Two runs give the same bits. `slack`: an error that is allowed besides."""
    n, H, _ = k.shape
    T = q.shape[0]
    need = -(-n // page)
    rng = np.random.default_rng(n)
    order = rng.permutation(need + 2)
    mine = order[:need]
    ref, cache = R.Cache(need + 2, page, H, D), fb.PagedCache(be, need + 2, page, H, D)
    slots = mine[np.arange(n) // page] * page + np.arange(n) % page
    other = _bf(rng.standard_normal((1, H, D)))
    for a, b, s in ((k, v, slots), (other, other, [order[need] * page])):
        be.cache_append(cache, _up(be, a, "f32"), _up(be, b, "f32"), _up(be, s, "i32"))
        ref.append(a, b, s)
    width = max(need, -(-WIDE // page)) if wide else need
    table = np.full((2, width), -1, np.int64)
    table[0, :need], table[1, 0] = mine, order[need]
    scale = D ** -0.5 if scale is None else scale
    both = np.concatenate([q, _bf(rng.standard_normal((1, H * group, D)))])
    args = (_up(be, both, "bf16"), cache, _up(be, table, "i32"), _up(be, [0, T, T + 1], "i32"), _up(be, [n, 1], "i32"), H * group)
    got = _down(be.cache_attention(*args, scale=scale, causal=causal), both.shape).astype(np.float64)
    again = _down(be.cache_attention(*args, scale=scale, causal=causal), both.shape)
    be.sync()
    assert np.array_equal(got, again.astype(np.float64), equal_nan=True)
    want, tol = _bound(both[:T], ref, mine, T, n, scale, causal)
    alone, tol1 = _bound(both[T:], ref, order[need:need + 1], 1, 1, scale, causal)
    want, tol = np.concatenate([want, alone]), np.concatenate([tol, tol1])
    assert np.isfinite(got).all(), np.argwhere(~np.isfinite(got))[:4]
    err = np.abs(got - want) - tol - slack
    assert np.all(err <= 0), (err.max(), np.unravel_index(err.argmax(), err.shape), np.count_nonzero(err > 0))


def _plain(rng, n, H, D):
    """Ordinary keys and values: channels of different sizes and means."""
    k = rng.standard_normal((n, H, D)) * (0.5 + np.abs(rng.standard_normal((1, H, D)))) + rng.standard_normal((1, H, D))
    v = rng.standard_normal((n, H, D)) + 0.2 * rng.standard_normal((1, H, D))
    return k.astype(F), v.astype(F)


KINDS = [(1, False), (20, False), (40, True)]  # new tokens, and whether the prompts' kernel takes them


# ---- hidden keys beside scores that are zero ----
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [-30, -100])
@pytest.mark.parametrize("size,scale", [(0.0, None), (1.0, 0.0), (2.0 ** -20, None)])
@pytest.mark.parametrize("T,wide", KINDS)
def test_zero_scores_of_small_keys(b200, D, power, size, scale, T, wide):
    """Queries, the scale or both so small that every score is zero, over small keys: the mean of what a row sees."""
    rng = np.random.default_rng(1)
    k, v = _plain(rng, 150, 1, D)
    q = _bf(rng.standard_normal((T, 4, D)) * size)
    _check(b200, q, np.ldexp(k, power), v, D, 4, scale=scale, wide=wide)


# ---- values far smaller or larger than 1, and of both kinds in one sequence ----
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [-115, -100, 97])
@pytest.mark.parametrize("T,wide", KINDS)
def test_many_equal_scores_over_values_of_any_size(b200, D, power, T, wide):
    """The sum of the probabilities stays in range however the values are scaled."""
    rng = np.random.default_rng(2)
    k, v = _plain(rng, 900, 1, D)
    q = np.zeros((T, 4, D), F)
    v = np.ldexp(np.clip(v, -6, 6) + F(2), power)  # means that do not cancel
    _check(b200, q, k, v, D, 4, wide=wide, slack=2.0 ** -126)  # smaller numbers are zeros


def _aimed(rng, T, group, D):
    """Queries near the direction of ones: keys of `a` in every channel score a sqrt(D) (1 +- 0.1) or so."""
    return _bf(1 + 0.25 * rng.standard_normal((T, group, D)))


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("low,high", [(-60, 90), (-100, 40), (-20, 20)])
@pytest.mark.parametrize("weight", [True, False])  # whether the large values have any
@pytest.mark.parametrize("large_first", [True, False])
@pytest.mark.parametrize("T,wide", KINDS)
def test_small_values_beside_large_ones(b200, D, low, high, weight, large_first, T, wide):
    """Runs of tiny values and of huge ones, which different warps and blocks meet: where the huge ones have no
    weight, the output is of the tiny ones."""
    rng = np.random.default_rng(3)
    k, v = _plain(rng, 2500, 1, D)
    large = np.arange(2500) < 1100 if large_first else np.arange(2500) >= 1400
    large[-T:] = False  # the new tokens' own
    v = np.ldexp(v, np.where(large, high, low)[:, None, None]).astype(F)
    if not weight:
        k[large] = -60
    _check(b200, _aimed(rng, T, 4, D), k, v, D, 4, wide=wide, slack=2.0 ** -126)


# ---- one key apart from all others ----
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [10, 14, 18, 22, 40, 128])
@pytest.mark.parametrize("at", [0, 137, 940])
@pytest.mark.parametrize("T,wide", KINDS)
def test_a_large_value_of_no_weight(b200, D, power, at, T, wide):
    """One key that no query wants, with a value 2^power times as large as the others (past 2^127: infinite)."""
    rng = np.random.default_rng(4)
    k, v = _plain(rng, 1000, 1, D)
    k[at] = -60
    with np.errstate(over="ignore"):
        v[at] = v[at] * F(2) ** F(power)
    _check(b200, _aimed(rng, T, 4, D), k, v, D, 4, wide=wide)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [16, 30, 60, 128])
@pytest.mark.parametrize("which", ["k", "v", "kv"])
@pytest.mark.parametrize("T,wide", [(20, False), (40, True)])
def test_a_large_key_and_value_that_most_rows_do_not_see(b200, D, power, which, T, wide):
    """A new token whose key, value or both are 2^power times the others' or infinite: the tokens before it do not
    see it, and their answers are what they are without it."""
    rng = np.random.default_rng(5)
    k, v = _plain(rng, 300, 2, D)
    q = _bf(rng.standard_normal((T, 8, D)))
    with np.errstate(over="ignore"):
        for n, x in (("k", k), ("v", v)):
            if n in which:
                x[296] = np.abs(x[296]) * F(2) ** F(power)
    q[-4:] = -np.abs(q[-4:])  # who sees it does not want it
    if "k" not in which:
        k[296] = 60
    _check(b200, q, k, v, D, 4, wide=wide)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [12, 20, 60, 128])
@pytest.mark.parametrize("at", [3, 137])
@pytest.mark.parametrize("T,wide", KINDS)
def test_a_large_key_of_no_weight(b200, D, power, at, T, wide):
    """A key 2^power times as long as the others that every query turns away from."""
    rng = np.random.default_rng(6)
    k, v = _plain(rng, 300, 1, D)
    with np.errstate(over="ignore"):
        k[at] = -F(8) * F(2) ** F(power)
    _check(b200, _aimed(rng, T, 4, D), k, v, D, 4, wide=wide)


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,wide,power", [(T, False, p) for T in (1, 20) for p in (8, 16, 40, 128)] + [(40, True, 8), (40, True, 16)])
def test_a_large_channel_leaves_other_groups_alone(b200, D, T, wide, power):
    """A key like any other, one of whose channels has a value 2^power times the rest: what its group's other channels
    can say goes, other groups' outputs stay. The prompts' kernel follows a token's largest group, and the others as
    long as they are no less than 2^-18 of it."""
    rng = np.random.default_rng(7)
    k, v = _plain(rng, 400, 1, D)
    with np.errstate(over="ignore"):
        v[77, 0, 5] = F(3) * F(2) ** F(power)
    _check(b200, _bf(rng.standard_normal((T, 4, D))), k, v, D, 4, wide=wide)


# ---- many keys of little weight each ----
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("bits", [14, 18, 22, 25])
@pytest.mark.parametrize("sink", [1.0, 2.0 ** -6])  # the size of the heavy key's own value
@pytest.mark.parametrize("T,wide", KINDS)
def test_a_long_flat_tail_behind_one_heavy_key(b200, D, bits, sink, T, wide):
    """The first key has 2^bits times the weight of each of 20000 equal others."""
    rng = np.random.default_rng(8)
    n = 20000
    k = np.zeros((n, 1, D), F)
    v = np.broadcast_to(rng.standard_normal((1, 1, D)).astype(F) + F(1), (n, 1, D)).copy()
    k[0] = bits * np.log(2) / D ** 0.5  # times ones
    v[0] = rng.standard_normal((1, D)) * sink
    _check(b200, np.ones((T, 2, D), F), k, v, D, 2, wide=wide, page=64)


# ---- scores far from zero ----
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [-100, 0, 10, 24, 40, 97])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("size", [-30, 0, 60])
@pytest.mark.parametrize("T,wide", KINDS)
def test_equal_keys_of_any_size(b200, D, power, sign, size, T, wide):
    """Keys that are all the same: the mean of the values that a row sees, however far the scores are from zero."""
    rng = np.random.default_rng(9)
    n, group = T + 30, 4
    k = np.full((n, 1, D), np.ldexp(sign * 3.0, power), F)
    v = np.ldexp(rng.standard_normal((n, 1, D)) + 1, size).astype(F)
    q = _aimed(rng, T, group, D)
    cache, ref = fb.PagedCache(b200, 8, 32, 1, D), R.Cache(8, 32, 1, D)
    b200.cache_append(cache, _up(b200, k, "f32"), _up(b200, v, "f32"), _up(b200, np.arange(n), "i32"))
    ref.append(k, v, np.arange(n))
    table = np.full((1, WIDE // 32 if wide else 8), -1)
    table[0, :8] = np.arange(8)
    got = _down(b200.cache_attention(_up(b200, q, "bf16"), cache, _up(b200, table, "i32"), _up(b200, [0, T], "i32"),
                                     _up(b200, [n], "i32"), group), q.shape).astype(np.float64)
    b200.sync()
    V, A = (x.reshape(-1, D)[:n] for x in (ref.values("v")[:, 0], ref.parts("v")[:, 0]))
    for t in range(T):
        seen = n - T + t + 1
        want, tol = V[:seen].mean(0), (2.0 ** -9 + 2.0 ** -18) * A[:seen].mean(0)
        assert np.all(np.abs(got[t] - want) <= tol + 2.0 ** -8 * np.abs(want)), (t, np.abs(got[t] - want).max())


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("power", [10, 20, 24, 40, 97])
@pytest.mark.parametrize("size", [-30, 0, 60])
@pytest.mark.parametrize("T,wide", KINDS)
def test_ordinary_keys_behind_ones_far_below(b200, D, power, size, T, wide):
    """Runs that begin with keys of no weight whose scores are far below all others'."""
    rng = np.random.default_rng(10)
    k, v = _plain(rng, 700, 1, D)
    k[:100], k[300:400] = -np.ldexp(3.0, power), -np.ldexp(5.0, power)
    _check(b200, _aimed(rng, T, 4, D), k, np.ldexp(v, size), D, 4, wide=wide)
