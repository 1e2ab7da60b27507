"""What a device-side error leaves behind, what streams hold, and calls of nothing. The expired wait is made on the host: its code is written where a kernel would
write it, and arrivals are left in a workspace as a kernel that gave up would leave them; no wait runs out."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import furiosa_opt_b200 as fb
from furiosa_opt_b200 import _lib
from test_gpu_kvcache import WIDE, Case, _down, _up

pytestmark = pytest.mark.gpu

HERE = os.path.dirname(os.path.abspath(__file__))
SOURCE = """
#include "ctx.hpp"
extern "C" void* expired(fopt_ctx* c) { return c->dev_err; }
extern "C" void* workspace(fopt_ctx* c) { return c->cache_ws.begin()->second.p; }
"""


@pytest.fixture(scope="module")
def inside(tmp_path_factory):
    """The addresses of a context's word for expired waits and of its only workspace."""
    d = tmp_path_factory.mktemp("inside")
    (d / "inside.cu").write_text(SOURCE)
    csrc = os.path.join(os.path.dirname(HERE), "furiosa-opt_b200", "csrc")
    nvcc = shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc"
    subprocess.run([nvcc, "-std=c++17", "-arch=sm_100a", "-shared", "-Xcompiler", "-fPIC", "-I", csrc, "-o", str(d / "inside.so"),
                    str(d / "inside.cu")], check=True)
    lib = C.CDLL(str(d / "inside.so"))
    for f in (lib.expired, lib.workspace):
        f.restype, f.argtypes = C.c_void_p, [C.c_void_p]
    return lib


def _write(be, address, words):
    a = np.asarray(words, np.int32)
    _lib.check(_lib.lib().fopt_h2d(be.ctx, address, a.ctypes.data, a.nbytes), be.ctx)


def test_a_bad_index_does_not_hide_an_expired_wait(inside):
    """Both are reported, once, and the arrivals that the wait left behind are gone for the next call."""
    be = fb.B200(0)
    c = Case(be, [1, 1], [9001, 40], 2, 4, 128, 64, seed=51)
    good = c.check()
    past = _up(be, [c.cache.slots], "i32")  # a slot past the cache
    out = fb.Storage(be, "bf16", 256), fb.Storage(be, "bf16", 256)
    _write(be, inside.expired(be.ctx), [401])
    be.cache_read(c.cache, past, out=out)
    with pytest.raises(fb._lib.FoptError, match="wait expired.*slot past") as e:
        be.sync()
    assert e.value.status == 5
    be.sync()
    be.cache_read(c.cache, past, out=out)
    with pytest.raises(fb._lib.FoptError, match="slot past") as e:
        be.sync()
    assert e.value.status == 1
    assert np.array_equal(_down(c.run(), c.q.shape), good)


def test_an_expired_wait_leaves_no_arrivals(inside):
    """Arrivals in the workspace of one stream, the wait reported on another."""
    import torch
    be = fb.B200(0)
    c = Case(be, [1, 1], [9001, 40], 2, 4, 128, 64, seed=52)
    side = torch.cuda.Stream()
    be.sync()
    be.set_stream(side.cuda_stream)  # the only stream that attention runs on, so that its workspace is the only one
    want = _down(c.run(), c.q.shape)
    graph = be.capture(lambda: c.run())
    ws = inside.workspace(be.ctx)
    be.set_stream(None)
    for _ in range(2):
        _write(be, ws, [1] * 1024)
        _write(be, inside.expired(be.ctx), [401])
        with pytest.raises(fb._lib.FoptError, match="wait expired"):
            be.sync()
        be.set_stream(side.cuda_stream)
        for _ in range(2):
            assert np.array_equal(_down(c.run(), c.q.shape), want)
        assert np.array_equal(_down(graph.launch(), c.q.shape), want)
        be.set_stream(None)
    graph.close()


def test_many_streams_hold_few_workspaces():
    """A program that takes another stream for each request: what the context keeps for them is bounded."""
    import torch
    be = fb.B200(0)
    c = Case(be, [70, 1], [800, 3000], 2, 4, 128, 64, seed=53, wide=WIDE)
    want = c.check()
    streams = [torch.cuda.Stream() for _ in range(28)]
    assert len({s.cuda_stream for s in streams}) == 28
    out = fb.Storage(be, "bf16", c.q.size)
    be.sync()
    before = torch.cuda.mem_get_info()[0]
    for s in streams + streams[:3]:
        be.set_stream(s.cuda_stream)
        c.run(out=out)
        be.sync()
    be.set_stream(None)
    held = before - torch.cuda.mem_get_info()[0]
    assert np.array_equal(_down(out, want.shape), want)
    assert held <= 16 * 48 * 2 ** 20, held


def test_empty_calls():
    """No tokens, no slots, no queries: nothing is read, written or reported."""
    be = fb.B200(0)
    c = Case(be, [1, 1], [40, 20], 2, 4, 128, 16, seed=54)
    want = c.check()
    images = [s.to_bytes() for s in (c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale)]
    none, zero = fb.Storage(be, "bf16", 0), fb.Storage(be, "i32", 0)
    rope = fb.Rope([1.0] * 64)
    assert be.rotary(none, zero, rope, 2).n == 0
    be.cache_append(c.cache, none, none, zero, positions=zero, rope=rope)
    assert [s.n for s in be.cache_read(c.cache, zero)] == [0, 0]
    d = c.dev
    assert be.cache_attention(none, c.cache, d["table"], _up(be, [0, 0, 0], "i32"), d["kv_len"], 8).n == 0
    be.sync()
    assert images == [s.to_bytes() for s in (c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale)]
    assert np.array_equal(_down(c.run(), c.q.shape), want)


def test_a_bad_start_leaves_other_sequences_alone():
    """A start past the tokens: the sequences before it are what they are without it."""
    be = fb.B200(0)
    c = Case(be, [1, 1, 1], [40, 20, 64], 1, 4, 128, 16, seed=55)
    good = c.check()
    c.dev["q_start"] = _up(be, [0, 1, 5, 3], "i32")
    got = c.run()
    with pytest.raises(fb._lib.FoptError, match="query starts"):
        be.sync()
    assert np.array_equal(_down(got, c.q.shape)[0], good[0])


def test_forward_is_what_it_was_before_the_cached_step():
    """`DecoderBlockW8A8.forward` gives the bits that it gave before `step` came beside it."""
    import hashlib
    be = fb.B200(0)
    for shape, digest in (((128, 256, 2, 1, 512, 1, 128), "811494477c50f9293115cca434eb574a80e8ff96f18e7c81c6e09cd9479271c2"),
                          ((256, 512, 4, 2, 1024, 2, 128), "85bfc8c21782b66ae849c6e88f167df57835970b4c65ba51655290a4ee749b90")):
        blk = fb.workloads.DecoderBlockW8A8(be, *shape, seed=9)
        x = fb.dtypes.f32_to_bf16_bits(np.random.default_rng(1).standard_normal(shape[0] * shape[1]).astype(np.float32))
        y = blk.forward(be.from_vec(blk.m("[T, H]"), x, "bf16")).to_bytes()
        assert hashlib.sha256(bytes(y)).hexdigest() == digest
