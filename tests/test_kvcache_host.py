"""Rotary positions and the paged 4-bit cache without a GPU: the oracle's own pins, the scalings, and what
the entry points refuse before they touch a context."""
import ctypes as C
import math

import numpy as np
import pytest

import furiosa_opt_b200 as fb
from furiosa_opt_b200 import _lib
from oracle import cache_ref as R

F = np.float32


# ---- the oracle ----
def test_rotation_is_a_rotation():
    """Pairs keep their length, position 0 turns nothing, and q . k depends on the distance alone."""
    rng = np.random.default_rng(0)
    f = [10000.0 ** (-2 * p / 64) for p in range(32)]
    x = rng.standard_normal((4, 1, 80)).astype(F)
    for layout, a, b in (("half", slice(0, 32), slice(32, 64)), ("interleaved", slice(0, 64, 2), slice(1, 64, 2))):
        y = R.rotate(x, [0, 3, 10 ** 6, -5], f, layout)
        assert np.array_equal(y[0], x[0]) and np.array_equal(y[..., 64:], x[..., 64:])
        assert np.allclose(y[..., a] ** 2 + y[..., b] ** 2, x[..., a] ** 2 + x[..., b] ** 2, rtol=1e-5)
        q, k = x[:1], x[1:2]
        dots = [float((R.rotate(q, [p + 7], f, layout)[..., :64] * R.rotate(k, [p], f, layout)[..., :64]).sum())
                for p in (0, 1, 1000, 100000)]
        assert np.ptp(dots) < 1e-4


def test_quantiser_pins():
    """A group that fills the codes exactly, a constant one, and the largest error of any: half a step,
    and at the ends what rounding the step and the offset to bf16 (2^-8 of each) can add."""
    x = np.concatenate([np.arange(16), np.arange(16)]).astype(F)
    c, s, z = R.quantise(x)
    assert s == 1 and z == 8 and np.array_equal(c, np.tile(np.arange(-8, 8), 2))
    c, s, z = R.quantise(np.full(32, F(-2.5)))
    assert s == 0 and z == F(-2.5) and not c.any()
    c, _, z = R.quantise(np.tile(np.array([0, 15, 7.5, 8.5], F), 8))
    assert c[2] == np.rint(7.5 - 8) and c[3] == np.rint(8.5 - 8)  # halves go to even
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1000, 64)).astype(F) * 10
    c, s, z = R.quantise(x)
    err = np.abs(R.values(c, s, z) - x).reshape(1000, 2, 32)
    assert np.all(err <= (0.5 * s + 15 * s * 2.0 ** -8 + np.abs(z) * 2.0 ** -8 + 8 * s * 2.0 ** -8)[..., None])


def test_oracle_attention_is_softmax():
    rng = np.random.default_rng(2)
    cache = R.Cache(2, 16, 1, 64)
    k, v = rng.standard_normal((20, 1, 64)).astype(F), rng.standard_normal((20, 1, 64)).astype(F)
    cache.append(k, v, np.arange(20))
    q = rng.standard_normal((1, 2, 64)).astype(F)
    o, _ = R.attention(q, cache, [[0, 1]], [0, 1], [20], 0.125)
    K, V = (cache.values(n)[:, 0].reshape(-1, 64)[:20] for n in "kv")
    e = np.exp(0.125 * q[0].astype(np.float64) @ K.T)
    assert np.allclose(o[0], e @ V / e.sum(-1, keepdims=True))


# ---- scalings ----
def test_scaled_frequencies():
    plain = fb.Rope.scaled(128, base=500000.0).inv_freq
    assert plain[0] == 1.0 and math.isclose(plain[-1], 500000.0 ** (-126 / 128))
    assert np.allclose(np.array(fb.Rope.scaled(128, 500000.0, scaling="linear", factor=4).inv_freq) * 4, plain)
    ntk = fb.Rope.scaled(128, 500000.0, scaling="ntk", factor=4).inv_freq
    assert ntk[0] == 1.0 and math.isclose(ntk[-1] * 4, plain[-1])
    parts = fb.Rope.scaled(128, 500000.0, scaling="by_parts", factor=8, original_length=8192).inv_freq
    turns = 8192 * np.array(plain) / (2 * math.pi)
    kept, cut = turns >= 32, turns <= 1
    assert kept.any() and cut.any() and (~kept & ~cut).any()
    assert np.array_equal(np.array(parts)[kept], np.array(plain)[kept])
    assert np.allclose(np.array(parts)[cut] * 8, np.array(plain)[cut])
    assert np.all(np.diff(parts) < 0)


@pytest.mark.parametrize("kw", [dict(rot_dim=7), dict(rot_dim=0), dict(rot_dim=8, scaling="other"),
                                dict(rot_dim=8, scaling="by_parts"), dict(rot_dim=8, factor=0.0),
                                dict(rot_dim=8, scaling="by_parts", original_length=10, low=4, high=4)])
def test_scaled_refusals(kw):
    with pytest.raises(ValueError):
        fb.Rope.scaled(**kw)


def test_rope_refusals():
    with pytest.raises(ValueError, match="layout"):
        fb.Rope([1.0], layout="other")
    for f in ([], [1.0] * 129, [math.inf], [math.nan]):
        with pytest.raises(_lib.FoptError):
            fb.Rope(f)
    with pytest.raises(_lib.FoptError, match="magnitude"):
        fb.Rope([1.0], magnitude=math.nan)


# ---- refusals of the entry points (no context: they are checked first) ----
A = 4096  # an aligned address that nothing dereferences


def _desc(**kw):
    return _lib.PagedCacheDesc(**{**dict(k=A, v=A, k_scale=A, v_scale=A, pages=4, page_size=16, heads=2, head_dim=128), **kw})


BAD_CACHE = [(dict(k=0), "null"), (dict(v_scale=0), "null"), (dict(k=A + 8), "aligned"), (dict(head_dim=96), "head_dim"),
             (dict(head_dim=0), "head_dim"), (dict(heads=0), "empty"), (dict(pages=-1), "empty"),
             (dict(page_size=8), "page_size"), (dict(page_size=0), "page_size"), (dict(page_size=-16), "page_size"),
             (dict(page_size=65552), "page_size"), (dict(pages=2 ** 20, page_size=4096), "2\\^31")]


def _append(cache=None, k=A, v=A, dtype=3, ks=256, vs=256, slots=A, positions=A, rope=None, tokens=3):
    return _lib.lib().fopt_cache_append(None, C.byref(cache if cache is not None else _desc()), k, v, dtype, ks, vs, slots,
                                        positions, rope, tokens)


def _read(cache=None, k=A, v=A, dtype=3, slots=A, n=3):
    return _lib.lib().fopt_cache_read(None, k, v, dtype, C.byref(cache if cache is not None else _desc()), slots, n)


def _attend(cache=None, o=A, q=A, table=A, q_start=A, kv_len=A, batch=2, tokens=2, width=3, hq=8, scale=0.1, causal=1):
    return _lib.lib().fopt_cache_attention(None, o, q, C.byref(cache if cache is not None else _desc()), table, q_start,
                                           kv_len, batch, tokens, width, hq, C.c_float(scale), causal)


def _rotary(out=A, x=A, dtype=3, positions=A, rope=True, tokens=3, heads=2, dim=128, xs=256, os=256):
    r = fb.Rope([1.0] * 64)
    return _lib.lib().fopt_rotary(None, out, x, dtype, positions, r.handle if rope else None, tokens, heads, dim, xs, os)


def _says(status, text):
    import re
    msg = _lib.lib().fopt_last_error(None).decode()
    assert status == 1 and re.search(text, msg), (status, msg)


@pytest.mark.parametrize("call", [_append, _read, _attend])
def test_caches_refused(call):
    for kw, text in BAD_CACHE:
        _says(call(_desc(**kw)), text)
    _says(call(), "null context")


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=0), "bf16 or f32"), (dict(tokens=-1), "negative"), (dict(ks=255), "stride"), (dict(vs=0), "stride"),
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(slots=None), "null")])
def test_append_refusals(kw, text):
    _says(_append(**kw), text)


def test_append_refuses_a_rotation_it_cannot_do():
    wide = fb.Rope([1.0] * 65)
    _says(_append(rope=wide.handle), "more rotated channels")
    _says(_append(rope=fb.Rope([1.0] * 4).handle, positions=None), "null")


@pytest.mark.parametrize("kw,text", [(dict(dtype=2), "bf16 or f32"), (dict(n=-1), "negative"), (dict(k=None), "null"),
                                     (dict(slots=None), "null"), (dict(v=A + 4), "aligned"), (dict(n=2 ** 31 - 1), "past 2\\^31")])
def test_read_refusals(kw, text):
    _says(_read(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(batch=-1), "negative"), (dict(tokens=-1), "negative"), (dict(width=0), "empty page table"),
    (dict(hq=7), "multiple"), (dict(hq=0), "multiple"), (dict(scale=math.inf), "finite"), (dict(scale=math.nan), "finite"),
    (dict(o=None), "null"), (dict(q=None), "null"), (dict(table=None), "null"), (dict(q_start=None), "null"),
    (dict(kv_len=None), "null"), (dict(q=A + 2), "aligned"), (dict(o=A + 16), "aligned"), (dict(tokens=2 ** 30, hq=8), "too many")])
def test_attention_refusals(kw, text):
    _says(_attend(**kw), text)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=0), "bf16 or f32"), (dict(tokens=-1), "empty"), (dict(heads=0), "empty"), (dict(dim=126, xs=252, os=252), "more rotated"),
    (dict(xs=255), "stride"), (dict(os=255), "stride"), (dict(xs=300), "in place"), (dict(out=None), "null"),
    (dict(x=A + 16, out=A, positions=None), "null"), (dict(rope=False), "null"), (dict(heads=2 ** 25), "2\\^31")])
def test_rotary_refusals(kw, text):
    _says(_rotary(**kw), text)


# ---- the Python side ----
class _FakeBackend:
    """Storages without memory."""
    ctx = None

    def sync(self):
        pass


@pytest.fixture
def fake(monkeypatch):
    from furiosa_opt_b200 import backend as B
    be = B.B200.__new__(B.B200)
    be.ctx = None
    monkeypatch.setattr(B.Storage, "_alloc", lambda self, zero: setattr(self, "_ptr", C.c_void_p(A)))
    monkeypatch.setattr(B.Storage, "__del__", lambda self: None)
    monkeypatch.setattr(B.B200, "__del__", lambda self: None)
    monkeypatch.setattr(B.B200, "sync", lambda self: None)
    yield be


def _s(be, dtype, n):
    return fb.Storage(be, dtype, n)


def test_python_refusals(fake):
    be = fake
    rope = fb.Rope([1.0] * 64)
    c = fb.PagedCache(be, 4, 16, 2, 128)
    assert c.slots == 64 and c.k_map.size == c.k.n == 4 * 16 * 2 * 128 and c.scale_map.size == c.k_scale.n
    i32 = lambda n: _s(be, "i32", n)  # noqa: E731
    bad = [
        lambda: be.rotary(_s(be, "i8", 768), i32(3), rope, 2),
        lambda: be.rotary(_s(be, "bf16", 768), _s(be, "f32", 3), rope, 2),
        lambda: be.rotary(_s(be, "bf16", 767), i32(3), rope, 2),
        lambda: be.rotary(_s(be, "bf16", 768), i32(3), rope, 2, x_offset=1),
        lambda: be.rotary(_s(be, "bf16", 768), i32(3), rope, 2, x_offset=-1),
        lambda: be.rotary(_s(be, "bf16", 768), i32(3), rope, 2, x_stride=255),
        lambda: be.rotary(_s(be, "bf16", 768), i32(3), rope, 2, out=_s(be, "f32", 768)),
        lambda: be.rotary(_s(be, "bf16", 768), i32(3), rope, 2, out=_s(be, "bf16", 769)),
        lambda: be.cache_append(c, _s(be, "bf16", 768), _s(be, "f32", 768), i32(3)),
        lambda: be.cache_append(c, _s(be, "bf16", 768), _s(be, "bf16", 767), i32(3)),
        lambda: be.cache_append(c, _s(be, "bf16", 768), _s(be, "bf16", 768), i32(3), rope=rope),
        lambda: be.cache_append(c, _s(be, "bf16", 768), _s(be, "bf16", 768), i32(3), positions=i32(2), rope=rope),
        lambda: be.cache_read(c, _s(be, "f32", 3)),
        lambda: be.cache_read(c, i32(3), "i32"),
        lambda: be.cache_read(c, i32(3), out=(_s(be, "bf16", 768), _s(be, "bf16", 700))),
        lambda: be.cache_attention(_s(be, "f32", 2048), c, i32(4), i32(3), i32(2), 8),
        lambda: be.cache_attention(_s(be, "bf16", 2047), c, i32(4), i32(3), i32(2), 8),
        lambda: be.cache_attention(_s(be, "bf16", 2048), c, i32(4), i32(2), i32(2), 8),
        lambda: be.cache_attention(_s(be, "bf16", 2048), c, i32(5), i32(3), i32(2), 8),
        lambda: be.cache_attention(_s(be, "bf16", 2048), c, i32(0), i32(1), i32(0), 8),
        lambda: be.cache_attention(_s(be, "bf16", 2048), c, i32(4), i32(3), i32(2), 8, out=_s(be, "bf16", 1024)),
        lambda: fb.PagedCache(be, 4, 24, 2, 128),
        lambda: fb.PagedCache(be, 4, 16, 2, 96),
        lambda: fb.PagedCache(be, 0, 16, 2),
    ]
    for n, call in enumerate(bad):
        with pytest.raises(ValueError):
            call()
            pytest.fail(f"call {n} was not refused")
    q = _s(be, "bf16", 2048)
    with pytest.raises(ValueError):
        be.cache_attention(q, c, i32(4), i32(3), i32(2), 8, out=q)


def test_cache_batch_arrays(fake):
    c = fb.PagedCache(fake, 8, 16, 1, 64)
    b = fb.CacheBatch.__new__(fb.CacheBatch)
    b.be, b.cache, b.batch, b.tokens, b.table_width = fake, c, 3, 8, 3
    h = b._arrays([3, 0, 2], [18, 5, 2], [[4, 2], [7], [0]])
    assert list(h["positions"]) == [15, 16, 17, 0, 1, 0, 0, 0]
    assert list(h["slots"]) == [4 * 16 + 15, 2 * 16, 2 * 16 + 1, 0, 1, -1, -1, -1]
    assert list(h["q_start"]) == [0, 3, 3, 5] and list(h["kv_len"]) == [18, 5, 2]
    assert h["table"].reshape(3, 3).tolist() == [[4, 2, -1], [7, -1, -1], [0, -1, -1]]
    for q, n, p in (([9, 0, 0], [9, 0, 0], [[0], [], []]),      # more tokens than rows
                    ([3, 0, 0], [2, 0, 0], [[0], [], []]),      # fewer keys than new tokens
                    ([1, 0, 0], [17, 0, 0], [[0], [], []]),     # keys past the pages
                    ([1, 0, 0], [1, 0, 0], [[8], [], []]),      # no such page
                    ([1, 0, 0], [1, 0, 0], [[0, 1, 2, 3], [], []]),
                    ([1, 1, 0], [1, 1, 0], [[3], [3], []]),     # one slot for two tokens
                    ([1, 0], [1, 0], [[0], []])):
        with pytest.raises(ValueError):
            b._arrays(q, n, p)
