"""Calls of the tree and beam operators that are refused, on the CPU: a context
that holds a configuration and nothing else (no device, no buffers) reaches the
entry points' checks, and every case returns before anything is launched."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import mockbird_amd as mb

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

SOURCE = """
#include "mb_internal.h"
extern "C" mb_ctx* fake(const mb_config* c) {
  mb_ctx* x = new mb_ctx();
  x->cfg = *c;
  x->device = -1;
  return x;
}
extern "C" void drop(mb_ctx* x) { delete x; }
"""


@pytest.fixture(scope="module")
def helper(tmp_path_factory):
    d = tmp_path_factory.mktemp("fake")
    (d / "fake.cc").write_text(SOURCE)
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    subprocess.run(["g++", "-std=c++17", "-shared", "-fPIC", "-w", "-D__HIP_PLATFORM_AMD__",
                    "-I", os.path.join(rocm, "include"), "-I", os.path.join(ROOT, "include"),
                    "-I", os.path.join(ROOT, "mockbird_amd", "csrc"), str(d / "fake.cc"),
                    "-o", str(d / "fake.so")], check=True)
    mb.load()
    L = C.CDLL(str(d / "fake.so"))
    L.fake.argtypes, L.fake.restype = [C.POINTER(mb.Config)], C.c_void_p
    L.drop.argtypes = [C.c_void_p]
    return L


@pytest.fixture
def bare(helper):
    made = []

    def make(**kw):
        c = dict(n_layers=4, vocab=16, capacity=100, max_seqs=8, max_rows=32, kv_dtype=mb.MB_KV_F32,
                 wrap=1, device=0)
        c.update(kw)
        h = helper.fake(C.byref(mb.Config(*c.values())))
        made.append(h)
        return h

    yield make
    for h in made:
        helper.drop(h)


def _refused(h, rc, code, words):
    assert rc == code, rc
    msg = mb.load().mb_last_error(h).decode()
    assert words in msg, msg


P = 1 << 12  # a pointer that is never followed, 16-byte aligned


def tree_dev(h, layer=0, B=1, rows=8, qkv=P, dtype=0, stride=2304, parent=P, pos0=P, n=P, max_pos=50,
             out=P, out_stride=768, work=P, work_bytes=1 << 40):
    return mb.load().mb_tree_attention_dev(h, layer, B, rows, qkv, dtype, stride, parent, pos0, n,
                                           max_pos, out, out_stride, work, work_bytes)


@pytest.mark.parametrize("kw,words", [
    (dict(layer=-1), "layer"), (dict(layer=4), "layer"), (dict(B=9), "B 9"), (dict(B=-1), "B -1"),
    (dict(rows=0), "rows_max"), (dict(rows=65), "rows_max"), (dict(dtype=2), "dtype"),
    (dict(stride=2303), "stride"), (dict(out_stride=767), "stride"), (dict(max_pos=-1), "max_pos"),
    (dict(qkv=None), "null"), (dict(parent=None), "null"), (dict(pos0=None), "null"),
    (dict(out=None), "null"), (dict(qkv=P + 8), "16 bytes"), (dict(stride=2306), "16 bytes"),
    (dict(dtype=1, stride=2308), "16 bytes"), (dict(out_stride=770), "16 bytes"), (dict(out=P + 4), "16 bytes"),
    (dict(max_pos=5000, work=None), "workspace"), (dict(max_pos=5000, work_bytes=100), "workspace"),
    (dict(max_pos=5000, work=P + 8), "workspace"),
    (dict(), "out overlaps"), (dict(out=P + 8 * 2304 * 4 - 16), "out overlaps"),
    (dict(stride=3084, out_stride=3084, out=P + 2304 * 4 - 16), "out overlaps"),
    (dict(stride=3068, out_stride=3068, out=P + 2304 * 4), "out overlaps"),
])
def test_tree_attention_dev_refuses(bare, kw, words):
    _refused(h := bare(capacity=5000), tree_dev(h, **kw), mb.MB_ERR_ARG, words)


def test_tree_attention_beyond_a_non_wrapping_ring(bare):
    h = bare(wrap=0)
    _refused(h, tree_dev(h, max_pos=100), mb.MB_ERR_RANGE, "exceeds the KV ring")
    assert tree_dev(h, B=0, qkv=None) == mb.MB_OK


def test_work_queries(bare):
    lib, n = mb.load(), C.c_int64(-1)
    h = bare(capacity=4096)
    assert lib.mb_tree_attention_work(h, 0, 8, 100, C.byref(n)) == 0 and n.value == 0
    assert lib.mb_tree_attention_work(h, 1, 8, 4000, C.byref(n)) == 0 and n.value > 0
    assert lib.mb_tree_attention_work(h, 8, 64, 2 ** 31 - 1, C.byref(n)) == 0 and n.value > 0
    _refused(h, lib.mb_tree_attention_work(h, 1, 8, -1, C.byref(n)), mb.MB_ERR_ARG, "max_pos")
    _refused(h, lib.mb_tree_attention_work(h, 1, 65, 1, C.byref(n)), mb.MB_ERR_ARG, "rows_max")
    _refused(h, lib.mb_tree_attention_work(h, 1, 8, 1, None), mb.MB_ERR_ARG, "null")
    assert lib.mb_beam_select_work(h, 4, 8, 1024, 8, C.byref(n)) == 0 and n.value == 0
    assert lib.mb_beam_select_work(h, 4, 8, 1 << 30, 8, C.byref(n)) == 0 and 0 < n.value < 1 << 20
    _refused(h, lib.mb_beam_select_work(h, 4, 33, 10, 8, C.byref(n)), mb.MB_ERR_ARG, "beams")
    _refused(h, lib.mb_beam_select_work(h, 4, 8, 10, 8, None), mb.MB_ERR_ARG, "null")


def _p(a):
    return a.ctypes.data


@pytest.mark.parametrize("change,words,code", [
    (dict(n=-1), "nodes", mb.MB_ERR_ARG), (dict(n=5), "nodes", mb.MB_ERR_ARG),
    (dict(pos0=-1), "position", mb.MB_ERR_ARG), (dict(pos0=2 ** 31 - 64), "position", mb.MB_ERR_ARG),
    (dict(parent=[0, -1, -1, -1]), "no earlier node", mb.MB_ERR_ARG),
    (dict(parent=[-1, 2, -1, -1]), "no earlier node", mb.MB_ERR_ARG),
    (dict(parent=[-2, -1, -1, -1]), "no earlier node", mb.MB_ERR_ARG),
    (dict(pos0=98, parent=[-1, 0, 1, 2]), "exceeds the KV ring", mb.MB_ERR_RANGE),
])
def test_tree_attention_refuses(bare, change, words, code):
    h = bare(wrap=0)
    a = dict(n=4, pos0=10, parent=[-1, 0, 0, 1])
    a.update(change)
    qkv, out = np.zeros((1, 4, 2304), np.float32), np.zeros((1, 4, 768), np.float32)
    par, pos, n = (np.array(x, np.int32).reshape(1, -1) for x in (a["parent"], a["pos0"], a["n"]))
    rc = mb.load().mb_tree_attention(h, 0, 1, 4, _p(qkv), _p(par), _p(pos), _p(n), _p(out))
    _refused(h, rc, code, words)


def commit_dev(h, layer0=0, L=2, B=2, rows=8, qkv=P, dtype=0, stride=2304, layer_stride=2 * 8 * 2304,
               pos0=P, path_max=4, path=P, n=P):
    return mb.load().mb_tree_commit_dev(h, layer0, L, B, rows, qkv, dtype, stride, layer_stride, pos0,
                                        path_max, path, n)


@pytest.mark.parametrize("kw,words", [
    (dict(layer0=4), "layer"), (dict(layer0=3), "layers"), (dict(L=-1), "layers"), (dict(B=9), "B 9"),
    (dict(rows=65), "rows_max"), (dict(dtype=3), "dtype"), (dict(stride=2000), "stride"),
    (dict(path_max=-1), "path_max"), (dict(qkv=None), "null"), (dict(pos0=None), "null"),
    (dict(path=None), "null"), (dict(layer_stride=2304), "layer stride"),
    (dict(layer_stride=2 * 8 * 2304 + 2), "16 bytes"), (dict(qkv=P + 4), "16 bytes"),
])
def test_tree_commit_dev_refuses(bare, kw, words):
    h = bare()
    _refused(h, commit_dev(h, **kw), mb.MB_ERR_ARG, words)
    assert commit_dev(h, path_max=0, qkv=None) == mb.MB_OK
    assert commit_dev(h, L=0, qkv=None) == mb.MB_OK


@pytest.mark.parametrize("change,words,code", [
    (dict(pos0=-1), "negative", mb.MB_ERR_ARG), (dict(n=4), "path of", mb.MB_ERR_ARG),
    (dict(n=-1), "path of", mb.MB_ERR_ARG), (dict(path=[0, 4, 1]), "path node", mb.MB_ERR_ARG),
    (dict(path=[-1, 0, 1]), "path node", mb.MB_ERR_ARG),
    (dict(pos0=2 ** 31 - 2), "overflow", mb.MB_ERR_ARG),
    (dict(pos0=98), "exceeds the KV ring", mb.MB_ERR_RANGE),
])
def test_tree_commit_refuses(bare, change, words, code):
    h = bare(wrap=0)
    a = dict(n=3, pos0=10, path=[0, 1, 3])
    a.update(change)
    qkv = np.zeros((1, 1, 4, 2304), np.float32)
    path, pos, n = (np.array(x, np.int32).reshape(1, -1) for x in (a["path"], a["pos0"], a["n"]))
    rc = mb.load().mb_tree_commit(h, 0, 1, 1, 4, _p(qkv), _p(pos), 3, _p(path), _p(n))
    _refused(h, rc, code, words)


Q = 1 << 40


def beam_dev(h, B=2, W=4, V=100, n=4, logits=P, dtype=0, stride=100, scores=P, done=P, end=7, seen=P,
             penalty=1.2, scores_out=Q, parent=P, token=P, done_out=Q, seen_out=Q, work=P,
             work_bytes=1 << 40):
    return mb.load().mb_beam_select_dev(h, B, W, V, n, logits, dtype, stride, scores, done, end, seen,
                                        penalty, scores_out, parent, token, done_out, seen_out, work,
                                        work_bytes)


@pytest.mark.parametrize("kw,words", [
    (dict(B=-1), "voices"), (dict(W=0), "beams"), (dict(W=33), "beams"), (dict(n=0), "chosen"),
    (dict(n=33), "chosen"), (dict(V=0), "vocab"), (dict(V=(1 << 30) + 1), "vocab"),
    (dict(dtype=2), "dtype"), (dict(stride=99), "stride"), (dict(end=-1), "end_id"),
    (dict(end=100), "end_id"), (dict(end=-2, done=None), "end_id"), (dict(seen=None), "seen_out"),
    (dict(penalty=0.0), "penalty"), (dict(penalty=-1.0), "penalty"),
    (dict(penalty=float("nan")), "penalty"), (dict(penalty=float("inf")), "penalty"),
    (dict(scores_out=P), "its input"), (dict(done_out=P), "its input"), (dict(seen_out=P), "its input"),
    (dict(scores_out=P + 28), "its input"), (dict(done=Q + 28), "its input"), (dict(seen=Q + 124), "its input"),
    (dict(penalty=1e-60), "penalty"), (dict(penalty=1e300), "penalty"),
    (dict(logits=None), "null"), (dict(scores=None), "null"), (dict(scores_out=None), "null"),
    (dict(parent=None), "null"), (dict(token=None), "null"),
    (dict(V=5000, stride=5000, work=None), "workspace"),
    (dict(V=5000, stride=5000, work_bytes=64), "workspace"),
    (dict(V=5000, stride=5000, work=P + 8), "workspace"),
    (dict(B=2 ** 31 - 1, scores_out=1 << 60, done_out=1 << 60, seen_out=1 << 60), "too many rows"),
])
def test_beam_select_dev_refuses(bare, kw, words):
    h = bare()
    _refused(h, beam_dev(h, **kw), mb.MB_ERR_ARG, words)
    assert beam_dev(h, B=0, logits=None) == mb.MB_OK


def test_beam_select_refuses(bare):
    h, lib = bare(), mb.load()
    x = np.zeros((1, 2, 10), np.float32)
    s, o, i = np.zeros(2, np.float32), np.zeros(2, np.float32), np.zeros(2, np.int32)
    call = lambda W=2, sc=s, so=o, par=i, end=-1, done=None: lib.mb_beam_select(  # noqa: E731
        h, 1, W, 10, 2, _p(x), _p(sc), done, end, None, 1.0, _p(so), par if par is None else _p(par),
        _p(i), None, None)
    _refused(h, call(W=0), mb.MB_ERR_ARG, "beams")
    _refused(h, call(so=s), mb.MB_ERR_ARG, "its input")
    _refused(h, call(end=10), mb.MB_ERR_ARG, "end_id")
    _refused(h, call(done=_p(i)), mb.MB_ERR_ARG, "end_id")
    _refused(h, call(par=None), mb.MB_ERR_ARG, "null")


def reorder_dev(h, layer0=0, L=4, B=8, W=4, parent=P, a=P, z=P, most=10):
    return mb.load().mb_ring_reorder_dev(h, layer0, L, B, W, parent, a, z, most)


@pytest.mark.parametrize("kw,words", [
    (dict(layer0=-1), "layer"), (dict(L=5), "layers"), (dict(B=9), "B 9"), (dict(W=0), "width"),
    (dict(W=33), "width"), (dict(W=3), "divisor"), (dict(a=None), "together"), (dict(z=None), "together"),
    (dict(most=-1), "max_rows"), (dict(parent=None), "null"),
])
def test_ring_reorder_dev_refuses(bare, kw, words):
    h = bare()
    _refused(h, reorder_dev(h, **kw), mb.MB_ERR_ARG, words)
    assert reorder_dev(h, B=0, parent=None) == mb.MB_OK
    assert reorder_dev(h, most=0, parent=None) == mb.MB_OK


def test_ring_reorder_of_more_rings_than_a_launch_takes(bare):
    h = bare(n_layers=64, max_seqs=65535)
    _refused(h, reorder_dev(h, L=64, B=65535, W=1), mb.MB_ERR_ARG, "too many rings")


@pytest.mark.parametrize("a,z,code", [(-1, 5, mb.MB_ERR_ARG), (6, 5, mb.MB_ERR_ARG), (90, 101, mb.MB_ERR_RANGE)])
def test_ring_reorder_refuses(bare, a, z, code):
    h = bare(wrap=0)
    par = np.zeros(2, np.int32)
    x, y = np.array([a], np.int32), np.array([z], np.int32)
    rc = mb.load().mb_ring_reorder(h, 0, 1, 2, 2, _p(par), _p(x), _p(y))
    _refused(h, rc, code, "positions")


def test_python_shapes_are_checked(bare):
    ctx = object.__new__(mb.Context)
    ctx.lib, ctx.h = mb.load(), None
    z = np.zeros
    with pytest.raises(ValueError):
        ctx.tree_attention(0, z((2, 3, 2304)), z((2, 4)), z(2), z(2))
    with pytest.raises(ValueError):
        ctx.tree_attention(0, z((2, 3, 2304)), z((2, 3)), z(2), z(2), out=z((2, 3, 768)))
    with pytest.raises(ValueError):
        ctx.tree_commit(0, z((1, 2, 3, 2304)), z(2), z((3, 2)), z(2))
    with pytest.raises(ValueError):
        ctx.beam_select(z((1, 2, 70)), z((1, 2)), 2, seen=z((1, 2, 2)))
    with pytest.raises(ValueError):
        ctx.ring_reorder(0, 1, z((2, 3)), z(3), z(2))
