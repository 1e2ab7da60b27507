"""Rotary positions, the paged 4-bit key / value cache and attention over it, against plain forms in 64
bits (oracle/cache_ref.py).

Tolerances, from the roundings alone (half a step of bf16 is 2^-8 of the value, of f16 2^-11, of f32 2^-24):
  * rotary: the sine and cosine (each half an f32 step, and the f64 evaluation's ulp), two products and a
    sum: |error| <= (|a| + |b|) m 2^-22 for a pair (a, b) scaled by m; a bf16 result adds 2^-8 |y|;
  * stored codes, steps and offsets: none, every step of the rule is one IEEE operation;
  * attention: each probability carries the f32 error of its score and at most one rounding to 11 bits
    or more before it multiplies a value's code. A value is (code + 8) step + (offset - 8 step), and the two
    products may be rounded apart: sum (p (1 + d)) (code + 8) step + p (offset - 8 step), |d| <= 2^-11. The error
    is then relative to w = sum p ((code + 8) step + |offset - 8 step|), which exceeds sum p |v| where the parts
    cancel: (2^-10 + 2 s) w with s = 2^-19 scale sum |q| max |k| + 2^-18 (a score's f32 sums, of parts up to
    (15 + 8) / 8 as large as a code's own; the exponential is good to 2^-21); the output rounds to
    bf16: 2^-8 |o|."""
import ctypes as C

import numpy as np
import pytest

import furiosa_opt_b200 as fb
from furiosa_opt_b200 import _lib, dtypes, workloads as W
from oracle import cache_ref as R
from oracle import workloads_ref as WR

pytestmark = pytest.mark.gpu

F = np.float32


def _m(n):
    return fb.Mapping("[N]", dict(N=n))


def _up(be, a, dtype):
    a = np.ascontiguousarray(a).reshape(-1)
    return be.from_vec(_m(a.size), a, dtype)


def _down(s, shape):
    a = s.to_numpy()
    return (dtypes.bf16_bits_to_f32(a) if s.dtype == "bf16" else a).reshape(shape)


def _bf(a):
    """Values that bf16 holds, as f32."""
    return dtypes.bf16_bits_to_f32(dtypes.f32_to_bf16_bits(np.asarray(a, F)))


def _freqs(rot, base=500000.0):
    return [base ** (-2.0 * p / rot) for p in range(rot // 2)]


# ---------------------------------------------------------------------------------------------
# rotary
# ---------------------------------------------------------------------------------------------
POS = np.array([0, 1, -1, 5, 4095, 131071, 1000003, 2 ** 31 - 1, -2 ** 31, 77], np.int64)


@pytest.mark.parametrize("T,H,D,rot,layout,dtype,offset,gap", [
    (1, 32, 128, 128, "half", "bf16", 0, 0),
    (10, 3, 128, 128, "half", "f32", 0, 0),
    (10, 2, 96, 64, "interleaved", "f32", 480, 480),
    (10, 2, 96, 64, "half", "bf16", 8, 16),
    (9, 5, 80, 26, "half", "bf16", 0, 0),          # pairs that are no whole vectors
    (9, 5, 80, 26, "interleaved", "f32", 3, 7),    # rows off any alignment
    (7, 1, 2, 2, "half", "f32", 0, 0),
    (5, 1, 7, 6, "interleaved", "bf16", 1, 1),
    (2, 4, 256, 256, "half", "bf16", 0, 0),
    (1001, 3, 64, 48, "interleaved", "bf16", 0, 0),
    (1001, 2, 128, 112, "half", "f32", 0, 0),
])
def test_rotary(b200, T, H, D, rot, layout, dtype, offset, gap):
    rng = np.random.default_rng(T * 7 + D)
    stride = H * D + gap
    x = _bf(rng.standard_normal(offset + T * stride) * np.exp(rng.uniform(-3, 3, offset + T * stride)))
    pos = np.resize(POS, T) + (np.arange(T) // len(POS) if T > 10 else 0)
    rope = fb.Rope(_freqs(rot), layout=layout, magnitude=1.25)
    xs, ps = _up(b200, x, dtype), _up(b200, pos.astype(np.int32), "i32")
    got = _down(b200.rotary(xs, ps, rope, H, D, x_offset=offset, x_stride=stride), (T, H, D)).astype(np.float64)
    rows = np.stack([x[offset + t * stride:][:H * D] for t in range(T)]).reshape(T, H, D)
    pos32 = pos.astype(np.int32)
    a = np.asarray(pos32, np.longdouble)[:, None] * np.asarray(rope.inv_freq, np.longdouble)
    c, s = np.cos(a).astype(np.float64)[:, None] * 1.25, np.sin(a).astype(np.float64)[:, None] * 1.25
    one, two = (slice(0, rot // 2), slice(rot // 2, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    r = rows.astype(np.float64)
    want, size = r.copy(), np.zeros_like(r)
    want[..., one], want[..., two] = r[..., one] * c - r[..., two] * s, r[..., two] * c + r[..., one] * s
    size[..., one] = size[..., two] = np.abs(r[..., one]) + np.abs(r[..., two])
    tol = size * 1.25 * 2.0 ** -22 + (2.0 ** -8 * np.abs(want) if dtype == "bf16" else 0)
    tol[..., rot:] = 0  # not rotated: the same bits
    assert np.all(np.abs(got - want) <= tol), np.max(np.abs(got - want) - tol)
    if gap == 0 and offset == 0:  # in place gives the same bits
        before = got.astype(F)
        assert b200.rotary(xs, ps, rope, H, D, out=xs) is xs
        assert np.array_equal(_down(xs, (T, H, D)), before)


def test_rotary_in_place_leaves_the_rest_of_a_row(b200):
    T, H, D, stride = 6, 2, 64, 300
    x = np.random.default_rng(1).standard_normal(T * stride).astype(F)
    rope = fb.Rope(_freqs(32, base=10.0), layout="half")
    xs = _up(b200, x, "f32")
    b200.rotary(xs, _up(b200, np.arange(T), "i32"), rope, H, D, out=xs, x_offset=20, x_stride=stride - 4)
    got = xs.to_numpy()
    touched = np.zeros(x.size, bool)
    for t in range(T):
        for h in range(H):
            touched[20 + t * (stride - 4) + h * D:][:32] = t > 0  # position 0 turns nothing
    assert np.array_equal(got[~touched], x[~touched]) and not np.any(got[touched] == x[touched])


def test_rotary_is_undone_by_the_opposite_position(b200):
    """The rotation by -position: the transposed map, which is also its gradient."""
    T, H, D = 33, 4, 128
    x = np.random.default_rng(2).standard_normal((T, H, D)).astype(F)
    rope = fb.Rope.scaled(D, base=10000.0, scaling="by_parts", factor=8.0, original_length=8192)
    p = np.arange(T) * 7919
    y = b200.rotary(_up(b200, x, "f32"), _up(b200, p, "i32"), rope, H, D)
    z = _down(b200.rotary(y, _up(b200, -p, "i32"), rope, H, D), x.shape)
    # two rotations of relative size 1: twice the bound of one, on pairs of size |a| + |b| <= 2 max
    assert np.max(np.abs(z - x)) <= 2 * 2 * np.abs(x).max() * 2 * 2.0 ** -22


# ---------------------------------------------------------------------------------------------
# the cache's images
# ---------------------------------------------------------------------------------------------
def _cache_images(cache):
    return {"k": cache.k.to_numpy(), "v": cache.v.to_numpy(),
            "ks": dtypes.bf16_bits_to_f32(cache.k_scale.to_numpy()), "vs": dtypes.bf16_bits_to_f32(cache.v_scale.to_numpy())}


def _assert_cache(cache, ref):
    got = _cache_images(cache)
    for n in "kv":
        assert np.array_equal(got[n + "s"], ref.scale_image(n)), f"{n}: steps or offsets differ"
        assert np.array_equal(got[n], ref.image(n)), f"{n}: codes differ"


@pytest.mark.parametrize("T,H,D,page,pages,rot,layout,dtype", [
    (1, 1, 64, 16, 1, 0, "half", "bf16"),
    (5, 2, 128, 16, 2, 128, "half", "bf16"),
    (37, 3, 128, 48, 4, 64, "half", "f32"),
    (50, 5, 64, 16, 5, 26, "half", "bf16"),          # pairs that are no whole vectors
    (50, 1, 64, 32, 3, 30, "interleaved", "f32"),
    (33, 8, 256, 64, 1, 256, "interleaved", "bf16"),
    (33, 3, 256, 16, 3, 192, "half", "f32"),
    (700, 2, 128, 64, 12, 128, "half", "bf16"),
    (601, 1, 64, 16, 40, 64, "interleaved", "bf16"),
])
def test_append_is_the_rule_bit_for_bit(b200, T, H, D, page, pages, rot, layout, dtype):
    rng = np.random.default_rng(T + D)
    x = _bf if dtype == "bf16" else (lambda a: np.asarray(a, F))
    k = x(rng.standard_normal((T, H, D)) * np.exp(rng.uniform(-8, 8, (T, H, 1))) + 3)
    v = x(rng.standard_normal((T, H, D)))
    v[0, 0, :32] = v[0, 0, 0]              # a constant group: step 0
    v[-1, -1, -32:] = np.arange(32) * 0.5  # values on code borders
    slots = rng.permutation(pages * page)[:T]
    slots[rng.random(T) < 0.1] = -1
    slots[0] = pages * page - 1 if pages * page - 1 not in slots[1:] else slots[0]
    pos = rng.integers(0, 200000, T)
    ref = R.Cache(pages, page, H, D)
    cache = fb.PagedCache(b200, pages, page, H, D)
    rope = fb.Rope(_freqs(rot), layout=layout, magnitude=1.1) if rot else None
    ref.append(R.rotate(k, pos, _freqs(rot), layout, 1.1) if rot else k, v, slots)
    b200.cache_append(cache, _up(b200, k, dtype), _up(b200, v, dtype), _up(b200, slots, "i32"),
                      positions=_up(b200, pos, "i32") if rot else None, rope=rope)
    b200.sync()
    _assert_cache(cache, ref)
    # read back: every slot, then some with holes, in both types
    want = {n: ref.values(n).transpose(0, 2, 1, 3).reshape(-1, H, D) for n in "kv"}
    for dt in ("f32", "bf16"):
        pick = np.concatenate([np.arange(pages * page), [-1]])
        out = b200.cache_read(cache, _up(b200, pick, "i32"), dt)
        for n, s in zip("kv", out):
            got = _down(s, (pick.size, H, D))
            w = want[n].astype(F)
            assert np.array_equal(got[:-1], w if dt == "f32" else R.bf16_round(w)), n
            assert not got[-1].any()


def test_append_into_rows_of_a_wider_projection(b200):
    """Keys and values as parts of fused rows, aligned and not."""
    T, H, D, page = 19, 2, 64, 16
    rng = np.random.default_rng(5)
    for offset, stride in ((128, 3 * H * D), (5, 3 * H * D + 3)):
        row = _bf(rng.standard_normal(offset + T * stride + H * D))
        pick = lambda at: np.stack([row[at + t * stride:][:H * D] for t in range(T)]).reshape(T, H, D)  # noqa: E731
        ref, cache = R.Cache(2, page, H, D), fb.PagedCache(b200, 2, page, H, D)
        f = _freqs(64)
        ref.append(R.rotate(pick(offset), np.arange(T) + 9, f), pick(offset + H * D), np.arange(T))
        s = _up(b200, row, "bf16")
        b200.cache_append(cache, s, s, _up(b200, np.arange(T), "i32"), positions=_up(b200, np.arange(T) + 9, "i32"),
                          rope=fb.Rope(f), k_offset=offset, k_stride=stride, v_offset=offset + H * D, v_stride=stride)
        b200.sync()
        _assert_cache(cache, ref)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_append_of_what_no_code_says(b200, dtype):
    """NaN, infinities, the types' largest, smallest and subnormal values: stored values are finite."""
    T, H, D = 8, 1, 64
    rng = np.random.default_rng(8)
    x = rng.standard_normal((T, H, D)).astype(F)
    x[0, 0, 3], x[0, 0, 40] = np.nan, np.inf
    x[1, 0, :32], x[1, 0, 32:] = np.nan, -np.inf
    x[2] = np.where(rng.random((H, D)) < 0.5, 3.3e38, -3.3e38)
    x[3] *= F(1e-38)
    x[4] *= F(1e-40)
    x[5, 0, ::2] = 0
    x[6] = -0.0
    x[7, 0, 0] = 1e30
    x = _bf(x) if dtype == "bf16" else x
    ref, cache = R.Cache(1, 16, H, D), fb.PagedCache(b200, 1, 16, H, D)
    ref.append(x, x[::-1], np.arange(T))
    b200.cache_append(cache, _up(b200, x, dtype), _up(b200, x[::-1], dtype), _up(b200, np.arange(T), "i32"))
    b200.sync()
    _assert_cache(cache, ref)
    k, v = b200.cache_read(cache, _up(b200, np.arange(16), "i32"), "f32")
    assert np.isfinite(k.to_numpy()).all() and np.isfinite(v.to_numpy()).all()


@pytest.mark.parametrize("rot", [0, 48])  # 24 pairs: a half ends inside the channels of one thread
@pytest.mark.parametrize("power", [-140, -126, -104, -97, -60, 0, 60, 97, 124])
def test_append_on_and_beside_the_borders_between_codes(b200, power, rot):
    """Values at the middle of two codes, which go to the even one, and their neighbours, in steps of all sizes."""
    T, H, D = 64, 2, 64
    rng = np.random.default_rng(power % 97)
    n = (T, H, D // 32)
    step = _bf(np.exp2(rng.uniform(0, 1, n)))
    at = rng.integers(0, 31, n + (32,)) * F(0.5)
    at[..., 0], at[..., 1] = 0, 15
    with np.errstate(over="ignore", under="ignore"):
        x = (at * step[..., None] + rng.integers(-2, 3, n)[..., None] * step[..., None]).astype(F)
        x = np.where(rng.random(x.shape) < 0.5, x, np.nextafter(x, F(np.inf) * rng.choice([-1, 1], x.shape).astype(F)))
        x = np.ldexp(x.astype(F), power).astype(F).reshape(T, H, D)
    pos = rng.integers(0, 50, T)
    f = _freqs(48)
    for dtype in ("f32", "bf16"):
        a = _bf(x) if dtype == "bf16" else x
        ref, cache = R.Cache(4, 16, H, D), fb.PagedCache(b200, 4, 16, H, D)
        ref.append(R.rotate(a, pos, f) if rot else a, a, np.arange(T))
        b200.cache_append(cache, _up(b200, a, dtype), _up(b200, a, dtype), _up(b200, np.arange(T), "i32"),
                          positions=_up(b200, pos, "i32") if rot else None, rope=fb.Rope(f) if rot else None)
        b200.sync()
        _assert_cache(cache, ref)


@pytest.mark.parametrize("rot,layout", [(64, "half"), (64, "interleaved"), (48, "half"), (26, "half")])
def test_rotary_of_what_bf16_says_specially(b200, rot, layout):
    """NaN, infinities, the largest, the smallest and subnormal values: rounded under the bf16 rule, and only
    their own pairs touched."""
    T, H, D = 40, 2, 64
    rng = np.random.default_rng(rot)
    x = _bf(rng.standard_normal((T, H, D)))
    for v in (np.nan, np.inf, -np.inf, 3.3e38, -3.3e38, 1.2e-38, 1e-39, -1e-40, 0.0, -0.0):
        x[rng.integers(0, T, 12), rng.integers(0, H, 12), rng.integers(0, D, 12)] = _bf(v)
    pos, f = np.arange(T), _freqs(rot)
    got = b200.rotary(_up(b200, x, "bf16"), _up(b200, pos, "i32"), fb.Rope(f, layout=layout), H, D).to_numpy()
    y = R.rotate(x, pos, f, layout)
    want = dtypes.f32_to_bf16_bits(R.bf16_round(y)).reshape(T, H, D)
    got = np.asarray(got).reshape(T, H, D)
    want[np.isnan(y)] = 0x7FC0
    want[..., rot:] = dtypes.f32_to_bf16_bits(x[..., rot:])  # copied, not rounded
    assert np.array_equal(got, want)


def test_append_leaves_other_slots_and_reports_slots_past_the_cache(b200):
    T, H, D, page, pages = 6, 2, 128, 16, 3
    rng = np.random.default_rng(3)
    cache, ref = fb.PagedCache(b200, pages, page, H, D), R.Cache(pages, page, H, D)
    old, new = _bf(rng.standard_normal((pages * page, H, D))), _bf(rng.standard_normal((T, H, D)))
    b200.cache_append(cache, _up(b200, old, "bf16"), _up(b200, old, "bf16"), _up(b200, np.arange(pages * page), "i32"))
    ref.append(old, old, np.arange(pages * page))
    slots = np.array([40, -1, pages * page, 7, -2 ** 31, 2 ** 31 - 1])
    b200.cache_append(cache, _up(b200, new, "bf16"), _up(b200, new, "bf16"), _up(b200, slots, "i32"))
    with pytest.raises(fb._lib.FoptError, match="slot past"):
        b200.sync()
    b200.sync()  # reported once
    ref.append(new, new, np.where(slots < pages * page, slots, -1))
    _assert_cache(cache, ref)
    b200.cache_read(cache, _up(b200, [pages * page], "i32"))
    with pytest.raises(fb._lib.FoptError, match="slot past"):
        b200.sync()


def test_the_images_are_storages_of_their_mappings(b200):
    """A relayout from the cache's mapping to [P, S, H, D] gives the codes in plain order."""
    P, S, H, D = 2, 16, 3, 128
    rng = np.random.default_rng(4)
    cache, ref = fb.PagedCache(b200, P, S, H, D), R.Cache(P, S, H, D)
    x = _bf(rng.standard_normal((P * S, H, D)))
    b200.cache_append(cache, _up(b200, x, "bf16"), _up(b200, x, "bf16"), _up(b200, np.arange(P * S), "i32"))
    ref.append(x, x, np.arange(P * S))
    plain = fb.Mapping("[P, S, H, D]", cache.k_map.axes)
    for s, m, n in ((cache.k, cache.k_map, "k"), (cache.v, cache.v_map, "v")):
        got = b200.relayout(s, m, plain).to_numpy().reshape(P, S, H, D)
        assert np.array_equal(got, ref.codes[n].transpose(0, 2, 1, 3))


# ---------------------------------------------------------------------------------------------
# attention
# ---------------------------------------------------------------------------------------------
GARBAGE = 2 ** 30  # a page number that must not be read


class Case:
    """A filled cache, its sequences and their queries; spare slots and pages hold NaN."""

    def __init__(self, be, q_lens, kv_lens, H, group, D, page, seed=0, pad=0, spare=2, bias=1.0, size=1.0, wide=0):
        rng = np.random.default_rng(seed)
        self.be, self.H, self.group, self.D = be, H, group, D
        need = [-(-n // page) for n in kv_lens]
        pages = sum(need) + spare
        order = rng.permutation(pages)
        self.width = max(max(1, max(need)) + 1, -(-wide // page))  # a table wide enough for `wide` keys
        self.table = np.full((len(q_lens), self.width), GARBAGE, np.int64)
        self.ref, self.cache = R.Cache(pages, page, H, D), fb.PagedCache(be, pages, page, H, D)
        slots, at = [], 0
        for b, n in enumerate(kv_lens):
            mine = order[at:at + need[b]]
            at += need[b]
            self.table[b, :need[b]] = mine
            i = np.arange(n)
            slots.append(mine[i // page] * page + i % page if n else np.zeros(0, np.int64))
        slots = np.concatenate(slots).astype(np.int64)
        N = slots.size
        k = rng.standard_normal((N, H, D)) * np.exp(rng.uniform(-1, 1, (1, H, D))) + bias * rng.standard_normal((1, H, D))
        v = (rng.standard_normal((N, H, D)) + 0.5 * rng.standard_normal((1, H, D))) * np.exp(rng.uniform(-4, 4, (N, 1, 1)))
        for s in (self.cache.k_scale, self.cache.v_scale):  # what no append wrote is NaN
            nan = np.full(s.n, 0x7fc0, np.uint16)
            _lib.check(_lib.lib().fopt_h2d(be.ctx, s.ptr, nan.ctypes.data, nan.nbytes), be.ctx)
            be.sync()
        if N:
            k, v = _bf(k), _bf(v)
            be.cache_append(self.cache, _up(be, k, "bf16"), _up(be, v, "bf16"), _up(be, slots, "i32"))
            self.ref.append(k, v, slots)
        self.kv_lens = np.asarray(kv_lens)
        self.q_start = np.concatenate([[0], np.cumsum(q_lens)])
        self.T = int(self.q_start[-1]) + pad
        self.q = _bf(rng.standard_normal((self.T, H * group, D)) * size)
        self.dev = dict(q=_up(be, self.q, "bf16"), table=_up(be, self.table, "i32"),
                        q_start=_up(be, self.q_start, "i32"), kv_len=_up(be, self.kv_lens, "i32"))

    def run(self, causal=True, scale=None, out=None):
        d = self.dev
        return self.be.cache_attention(d["q"], self.cache, d["table"], d["q_start"], d["kv_len"], self.H * self.group,
                                       scale=scale, causal=causal, out=out)

    def check(self, causal=True, scale=None):
        out = self.be.from_vec(_m(self.q.size), np.full(self.q.size, 7.0, F), "bf16")
        got = _down(self.run(causal, scale, out), self.q.shape).astype(np.float64)
        self.be.sync()
        live = int(self.q_start[-1])
        assert np.all(got[live:] == 7.0)  # rows behind the last sequence
        sc = self.D ** -0.5 if scale is None else scale
        want, weight = R.attention(self.q, self.ref, self.table, self.q_start, self.kv_lens, sc, causal)
        kmax = np.abs(self.ref.values("k")).max((0, 2)) if self.kv_lens.any() else np.zeros((self.H, self.D))
        s = 2.0 ** -19 * abs(sc) * np.einsum("thd,hd->th", np.abs(self.q).astype(np.float64),
                                             np.repeat(kmax, self.group, 0)) + 2.0 ** -18
        tol = (2.0 ** -10 + 2 * s[..., None]) * weight + 2.0 ** -8 * np.abs(want)
        err = np.abs(got - want)[:live] - tol[:live]
        assert np.isfinite(got[:live]).all()
        assert np.all(err <= 0), (np.max(err), np.unravel_index(np.argmax(err), err.shape))
        return got


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("group", [1, 4, 7, 8, 12, 16])
def test_attention_single_tokens(b200, D, group):
    lens = [1, 0, 15, 16, 17, 128, 129, 300]
    Case(b200, [1] * len(lens), lens, 2, group, D, 16, seed=group).check()


@pytest.mark.parametrize("page", [16, 48, 64, 1024])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_pieces_and_single_tokens(b200, page, causal):
    """Sequences without new tokens, without keys, with fewer keys than queries, and ragged pieces."""
    Case(b200, [1, 37, 0, 5, 3, 1, 64, 2], [260, 37, 99, 3, 0, 0, 129, 2], 2, 4, 128, page, pad=3).check(causal)


@pytest.mark.parametrize("D,H,group,q,n", [(128, 2, 4, 130, 300), (64, 1, 7, 200, 200), (256, 1, 2, 70, 257),
                                           (128, 1, 1, 257, 513), (64, 2, 16, 40, 41), (128, 1, 32, 33, 100),
                                           (128, 1, 128, 2, 70), (128, 1, 200, 1, 40)])
def test_attention_prompts(b200, D, H, group, q, n):
    for causal in (True, False):
        Case(b200, [q], [n], H, group, D, 32, seed=q).check(causal)


def test_attention_long_contexts(b200):
    """Contexts that many blocks share, beside short ones; a second run gives the same bits."""
    c = Case(b200, [1, 1, 2, 1], [9001, 3, 4097, 1], 2, 4, 128, 64, seed=3)
    first = c.check()
    for _ in range(3):
        assert np.array_equal(_down(c.run(), c.q.shape), first.astype(F))


# Tables for contexts of this many keys: calls of more than 32 query rows to a key head then are the prompt kernel's
# whatever their size (narrow tables leave small ones to the kernel for single tokens).
WIDE = 400000


@pytest.mark.parametrize("page,D", [(16, 128), (48, 128), (64, 128), (1024, 128), (16, 64), (48, 256), (1024, 256)])
@pytest.mark.parametrize("causal", [True, False])
def test_attention_pieces_and_single_tokens_in_wide_tables(b200, page, D, causal):
    Case(b200, [1, 37, 0, 5, 3, 1, 64, 2], [260, 37, 99, 3, 0, 0, 129, 2], 2, 4, D, page, pad=3, wide=WIDE).check(causal)


@pytest.mark.parametrize("D,H,group,q,n", [(128, 2, 4, 130, 300), (64, 1, 7, 200, 200), (128, 1, 1, 257, 513),
                                           (64, 2, 16, 40, 41), (128, 1, 32, 33, 100), (128, 1, 128, 2, 70),
                                           (128, 1, 40, 16, 20000), (64, 1, 40, 5, 16385), (256, 1, 2, 70, 257),
                                           (256, 2, 5, 130, 700), (256, 1, 40, 1, 64), (256, 1, 8, 16, 9000)])
def test_attention_prompts_in_wide_tables(b200, D, H, group, q, n):
    for causal in (True, False):
        c = Case(b200, [q], [n], H, group, D, 32, seed=q, wide=WIDE)
        first = c.check(causal)
        assert np.array_equal(_down(c.run(causal), c.q.shape), first.astype(F))


@pytest.mark.parametrize("size,bias", [(30.0, 1.0), (1e-4, 0.0), (0.0, 1.0), (1.0, 300.0)])
def test_attention_of_sharp_and_flat_scores_in_wide_tables(b200, size, bias):
    for D in (128, 256):
        c = Case(b200, [1, 40], [500, 150], 1, 4, D, 16, seed=11, size=size, bias=bias, wide=WIDE)
        c.check()
        c.check(scale=0.0)
        c.check(scale=-0.05)


@pytest.mark.parametrize("D", [64, 128, 256])
def test_attention_in_a_wide_table_reads_no_further_than_the_lengths(b200, D):
    c = Case(b200, [1, 20, 1], [33, 40, 16], 2, 4, D, 16, seed=14, wide=WIDE)
    want = c.check()
    q = c.q.copy()
    q[2, 3, 5], q[0, 1, 0] = np.nan, np.inf  # one row each
    c.dev["q"] = _up(b200, q, "bf16")
    got = _down(c.run(), q.shape)
    clean = np.ones(q.shape[:2], bool)
    clean[2, 3] = clean[0, 1] = False
    assert np.array_equal(got[clean], want.astype(F)[clean])
    assert np.isnan(got[2, 3]).all()


@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("power", [-100, -30, 30, 90])
def test_attention_of_values_of_any_size_in_wide_tables(b200, power, D):
    c = Case(b200, [1, 33], [200, 50], 1, 4, D, 16, seed=12, wide=WIDE)
    s = F(2.0) ** F(power)
    for n in ("k", "v"):
        st = c.ref
        st.step[n] = st.step[n] * s
        st.offset[n] = st.offset[n] * s
        img = dtypes.f32_to_bf16_bits(st.scale_image(n))
        dev = getattr(c.cache, n + "_scale")
        _lib.check(_lib.lib().fopt_h2d(b200.ctx, dev.ptr, img.ctypes.data, img.nbytes), b200.ctx)
        b200.sync()
    c.q = (c.q / s).astype(F)
    c.dev["q"] = _up(b200, c.q, "bf16")
    c.check()


@pytest.mark.parametrize("D,H,group,q,n", [(64, 1, 1, 1, 30011), (128, 1, 3, 1, 20021), (256, 1, 2, 1, 9001),
                                           (128, 1, 8, 1, 30000), (128, 1, 8, 2, 12345),   # parts of single tokens
                                           (128, 1, 8, 16, 20000), (64, 1, 40, 5, 16385)])  # of prompts, one tile empty
def test_attention_of_few_heads_over_many_blocks(b200, D, H, group, q, n):
    """Segments that a hundred blocks share, of fewer rows than a block has, beside a short sequence."""
    c = Case(b200, [q, 1], [n, 40], H, group, D, 64, seed=n)
    first = c.check()
    for _ in range(3):
        assert np.array_equal(_down(c.run(), c.q.shape), first.astype(F))


def test_attention_many_sequences(b200):
    """More sequences than a block has threads."""
    n = 700
    rng = np.random.default_rng(6)
    Case(b200, list(rng.integers(0, 3, n)), list(rng.integers(0, 40, n)), 1, 4, 64, 16, seed=6).check()


@pytest.mark.parametrize("size,bias", [(30.0, 1.0), (1e-4, 0.0), (0.0, 1.0), (1.0, 300.0)])
def test_attention_of_sharp_and_flat_scores(b200, size, bias):
    c = Case(b200, [1, 20], [500, 150], 1, 4, 128, 16, seed=11, size=size, bias=bias)
    c.check()
    c.check(scale=0.0)
    c.check(scale=-0.05)


@pytest.mark.parametrize("power", [-100, -30, 30, 90])
def test_attention_of_values_of_any_size(b200, power):
    """Keys, values and queries far from 1: nothing overflows or vanishes on the way."""
    c = Case(b200, [1, 3], [200, 50], 1, 4, 128, 16, seed=12)
    s = F(2.0) ** F(power)
    for n in ("k", "v"):
        st = c.ref
        st.step[n] = st.step[n] * s
        st.offset[n] = st.offset[n] * s
        img = dtypes.f32_to_bf16_bits(st.scale_image(n))
        dev = getattr(c.cache, n + "_scale")
        _lib.check(_lib.lib().fopt_h2d(b200.ctx, dev.ptr, img.ctypes.data, img.nbytes), b200.ctx)
        b200.sync()
    c.q = (c.q / s).astype(F)
    c.dev["q"] = _up(b200, c.q, "bf16")
    c.check()


def test_attention_reads_no_further_than_the_lengths(b200):
    """NaN and infinities in later slots of the last page, in unused pages and in other rows' queries."""
    c = Case(b200, [1, 4, 1], [33, 20, 16], 2, 4, 128, 16, seed=14)
    want = c.check()
    q = c.q.copy()
    q[2, 3, 5], q[0, 1, 0] = np.nan, np.inf  # one row each
    c.dev["q"] = _up(b200, q, "bf16")
    got = _down(c.run(), q.shape)
    clean = np.ones(q.shape[:2], bool)
    clean[2, 3] = clean[0, 1] = False
    assert np.array_equal(got[clean], want.astype(F)[clean])
    assert np.isnan(got[2, 3]).all()


def test_attention_reports_bad_tables_and_lengths(b200):
    c = Case(b200, [1, 1, 1], [40, 20, 64], 1, 4, 128, 16, seed=15)
    good = c.check()
    table = c.table.copy()
    table[1, 0] = c.cache.pages
    bad = dict(table=(table, "page number", 1), kv_len=([40, 16 * c.width + 1, 64], "length", 1),
               q_start=([0, 1, 0, 3], "query starts", 2))
    for name, (a, text, hurt) in bad.items():
        keep, c.dev[name] = c.dev[name], _up(b200, a, "i32")
        if name == "kv_len":  # the pages past its own must exist for the cut length
            t = c.table.copy()
            t[1] = t[0, 0]
            c.dev["table"] = _up(b200, t, "i32")
        got = c.run()
        with pytest.raises(fb._lib.FoptError, match=text):
            b200.sync()
        if name != "q_start":
            ok = [i for i in range(3) if i != hurt]
            assert np.array_equal(_down(got, c.q.shape)[ok], good.astype(F)[ok])
        c.dev[name] = keep
        c.dev["table"] = _up(b200, c.table, "i32")
    c.check()


def test_attention_replays_over_growing_sequences(b200):
    """A captured append and attention, replayed while the host only rewrites the step's arrays; a second
    graph over the same cache, launched in turn with it, keeps its own workspace."""
    be = b200
    H, group, D, page, pages = 2, 4, 128, 16, 12
    rng = np.random.default_rng(21)
    ref, cache = R.Cache(pages, page, H, D), fb.PagedCache(be, pages, page, H, D)
    mine = [[3, 5, 1, 7], [0, 9, 2, 11]]
    lens = [30, 1]
    f = _freqs(D)
    rope = fb.Rope(f)
    k0 = _bf(rng.standard_normal((31, H, D)))
    fill = fb.CacheBatch(be, cache, lens, lens, mine)
    be.cache_append(cache, _up(be, k0, "bf16"), _up(be, -k0, "bf16"), fill.slots, positions=fill.positions, rope=rope)
    pos0 = np.concatenate([np.arange(30), [0]])
    ref.append(R.rotate(k0, pos0, f), -k0, fill.slots.to_numpy())
    step = fb.CacheBatch(be, cache, [1, 1], [31, 2], mine, tokens=3)
    q, k, v = (_up(be, np.zeros((3, n, D)), "bf16") for n in (H * group, H, H))
    o1, o2 = (be.from_vec(_m(3 * H * group * D), np.zeros(3 * H * group * D, F), "bf16") for _ in range(2))

    def one(o):
        be.cache_append(cache, k, v, step.slots, positions=step.positions, rope=rope)
        return be.cache_attention(q, cache, step.table, step.q_start, step.kv_len, H * group, out=o)

    one(o1)
    be.sync()
    graphs = [be.capture(lambda o=o: one(o)) for o in (o1, o2)]
    for it in range(20):
        lens = [lens[0] + 1, lens[1] + 1]
        step.rewrite([1, 1], lens, mine)
        hq, hk, hv = (_bf(rng.standard_normal((3, n, D))) for n in (H * group, H, H))
        for s, a in ((q, hq), (k, hk), (v, hv)):
            bits = dtypes.f32_to_bf16_bits(a).reshape(-1)
            _lib.check(_lib.lib().fopt_h2d(be.ctx, s.ptr, bits.ctypes.data, bits.nbytes), be.ctx)
            be.sync()
        for g in graphs:
            g.launch()
        be.sync()
        slots = step.slots.to_numpy()
        ref.append(R.rotate(hk, step.positions.to_numpy(), f), hv, slots)
        want, weight = R.attention(hq, ref, np.array(mine), [0, 1, 2], lens, D ** -0.5)
        for o in (o1, o2):
            got = _down(o, hq.shape)
            assert np.all(np.abs(got[:2] - want[:2]) <= 2.0 ** -8 * np.abs(want[:2]) + 2.0 ** -8 * weight[:2]), it
        assert np.array_equal(o1.to_numpy(), o2.to_numpy())
    for g in graphs:
        g._h and _lib.lib().fopt_graph_destroy(be.ctx, g._h)
        g._h = C.c_void_p()


def test_attention_on_two_streams(b200):
    """Calls on two streams of one backend at once: each has a workspace of its own."""
    import torch
    a = Case(b200, [1, 1], [4000, 900], 2, 4, 128, 64, seed=31)
    b = Case(b200, [1], [7000], 2, 4, 128, 64, seed=32)
    wa, wb = a.check().astype(F), b.check().astype(F)
    b200.sync()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    oa, ob = (fb.Storage(b200, "bf16", c.q.size) for c in (a, b))
    b200.sync()
    try:
        for _ in range(10):
            for s, c, o in ((s1, a, oa), (s2, b, ob)):
                b200.set_stream(s.cuda_stream)
                outs.append(c.run(out=o))
        torch.cuda.synchronize()
    finally:
        b200.set_stream(None)
    assert np.array_equal(_down(oa, a.q.shape), wa) and np.array_equal(_down(ob, b.q.shape), wb)


def test_attention_of_prompts_and_tokens_in_graphs(b200):
    """Both kernels' work in two captured graphs, replayed in turn and each followed by a copy of its output."""
    cases = [Case(b200, [1, 130, 1, 40], [700, 900, 5, 40], 2, 7, 64, 16, seed=35, wide=WIDE),
             Case(b200, [60, 1, 1], [2000, 3000, 1], 1, 8, 128, 64, seed=36, wide=WIDE)]
    want = [c.check().astype(F) for c in cases]
    outs = [fb.Storage(b200, "bf16", c.q.size) for c in cases]
    b200.sync()
    graphs = [b200.capture(lambda c=c, o=o: c.run(out=o)) for c, o in zip(cases, outs)]
    for _ in range(10):
        for g in graphs:
            g.launch()
    b200.sync()
    for o, w in zip(outs, want):
        assert np.array_equal(_down(o, w.shape), w)
    for g in graphs:
        g._h and _lib.lib().fopt_graph_destroy(b200.ctx, g._h)
        g._h = C.c_void_p()


def test_attention_in_a_capture_of_another_library(b200):
    """Two graphs that torch captures on one stream and replays on two at once: neither shares a workspace."""
    import torch
    cases = [Case(b200, [1, 1], [4000, 900], 2, 4, 128, 64, seed=37), Case(b200, [70, 1], [800, 7000], 2, 4, 128, 64, seed=38, wide=WIDE)]
    want = [c.check().astype(F) for c in cases]
    outs = [fb.Storage(b200, "bf16", c.q.size) for c in cases]
    b200.sync()
    graphs, streams, side = [], [torch.cuda.Stream() for _ in cases], torch.cuda.Stream()
    try:
        for c, o in zip(cases, outs):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                b200.set_stream(torch.cuda.current_stream().cuda_stream)
                c.run(out=o)
            graphs.append(g)
    finally:
        b200.set_stream(None)
    torch.cuda.synchronize()
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert np.array_equal(_down(o, w.shape), w)


def test_attention_on_the_legacy_stream(b200):
    """Both kernels on the stream that others wait for."""
    c = Case(b200, [1, 130, 1], [700, 900, 5], 2, 4, 128, 16, seed=39, wide=WIDE)
    want = c.check().astype(F)
    o = fb.Storage(b200, "bf16", c.q.size)
    b200.sync()
    try:
        b200.set_stream(0)
        for _ in range(10):
            c.run(out=o)
        got = _down(o, want.shape)
    finally:
        b200.set_stream(None)
    assert np.array_equal(got, want)


def test_attention_past_32_bit_offsets(b200):
    """A cache whose images pass 2^32 bytes: pages at its far end are read and written where they are."""
    H, D, page, pages = 8, 256, 1024, 4200
    cache = fb.PagedCache(b200, pages, page, H, D)
    assert cache.k.nbytes > 2 ** 32
    rng = np.random.default_rng(41)
    n = 40
    k, v = _bf(rng.standard_normal((n, H, D))), _bf(rng.standard_normal((n, H, D)))
    far, near = pages - 1, 0
    for p, sign in ((far, 1), (near, -1)):
        b200.cache_append(cache, _up(b200, sign * k, "bf16"), _up(b200, sign * v, "bf16"),
                          _up(b200, p * page + np.arange(n), "i32"))
    ref = R.Cache(1, page, H, D)
    ref.append(k, v, np.arange(n))
    q = _bf(rng.standard_normal((1, H * 2, D)))
    got = _down(b200.cache_attention(_up(b200, q, "bf16"), cache, _up(b200, [far], "i32"), _up(b200, [0, 1], "i32"),
                                     _up(b200, [n], "i32"), H * 2), q.shape)
    want, weight = R.attention(q, ref, [[0]], [0, 1], [n], D ** -0.5)
    assert np.all(np.abs(got - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -8 * weight)
    kk, _ = b200.cache_read(cache, _up(b200, [far * page + 3, near + 3], "i32"), "f32")
    kk = _down(kk, (2, H, D))
    assert np.array_equal(kk[0], ref.values("k")[0, :, 3].astype(F))


# ---------------------------------------------------------------------------------------------
# a run of them together: the decoder block as a server runs it
# ---------------------------------------------------------------------------------------------
def test_decoder_block_steps_against_the_oracle(b200):
    """Two prompts, then single tokens and a piece, through `DecoderBlockW8A8.step`, against the oracle block
    with rotary positions and the 4-bit cache; the tolerance is the block test's (3 % of max |out|, 0.3 % on
    average), for the same reason: a bf16 ulp of an activation can move its int8 code."""
    be = b200
    Hq, Hkv, FF, page = 4, 2, 1024, 16
    H = Hq * 128
    blk = W.DecoderBlockW8A8(be, 128, H, Hq, Hkv, FF, 1, 128, seed=3)
    rope = fb.Rope.scaled(128, base=500000.0, scaling="by_parts", factor=8.0, original_length=64)
    cache, ref = fb.PagedCache(be, 16, page, Hkv, 128), R.Cache(16, page, Hkv, 128)
    pages = [[4, 9, 0, 7, 8, 1], [3, 2, 15, 6, 5]]
    rng = np.random.default_rng(5)
    held = [0, 0]
    for q_lens, tokens in (([70, 50], 128), ([1, 1], 2), ([9, 1], 12), ([1, 1], 2)):
        held = [n + q for n, q in zip(held, q_lens)]
        b = blk if tokens == 128 else blk.with_tokens(tokens)
        batch = fb.CacheBatch(be, cache, q_lens, held, pages, tokens=tokens)
        x = fb.dtypes.f32_to_bf16_bits(rng.standard_normal(tokens * H).astype(F))
        got = _down(b.step(be.from_vec(b.m("[T, H]"), x, "bf16"), cache, batch, rope), (tokens, H))

        def attend(Q, K, V):
            Q, K, V = (dtypes.bf16_bits_to_f32(a).reshape(tokens, -1, 128) for a in (Q, K, V))
            pos = batch.positions.to_numpy()
            ref.append(R.rotate(K, pos, rope.inv_freq), V, batch.slots.to_numpy())
            q = R.bf16_round(R.rotate(Q, pos, rope.inv_freq))
            o, _ = R.attention(q, ref, batch.table.to_numpy().reshape(2, -1), batch.q_start.to_numpy(), held, 128 ** -0.5)
            return dtypes.f32_to_bf16_bits(np.nan_to_num(o).astype(F))

        want = dtypes.bf16_bits_to_f32(WR.decoder_ref(x, blk.host, tokens, H, Hq, Hkv, FF, 1, tokens, attend=attend))
        n = sum(q_lens)
        err, scale = np.abs(got - want.reshape(tokens, H))[:n], np.abs(want).max()
        assert err.max() <= 0.03 * scale and err.mean() <= 0.003 * scale, (err.max(), err.mean(), scale)


def test_decoder_block_forward_is_what_it_was(b200):
    """`forward` and a `with_tokens` block give the same bits."""
    blk = W.DecoderBlockW8A8(b200, 128, 256, 2, 1, 512, 1, 128, seed=9)
    x = fb.dtypes.f32_to_bf16_bits(np.random.default_rng(1).standard_normal(128 * 256).astype(F))
    xs = b200.from_vec(blk.m("[T, H]"), x, "bf16")
    other = blk.with_tokens(128)
    assert blk.forward(xs).to_bytes() == other.forward(xs).to_bytes()
