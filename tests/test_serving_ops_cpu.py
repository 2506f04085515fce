"""Refusals of the beam and scan entry points, and the host-side checks, without a GPU."""
import ctypes

import pytest
import torch

from tesm_b200 import _lib, ops

P = ctypes.c_void_p(1 << 20)  # never dereferenced: the checks come first


def status(name, *args):
    return getattr(_lib.load(), name)(*args)


def beam(dtype=0, G=1, W=4, V=100, K=4, logits=P, scores=P, lengths=None, alpha=0.0, pad=0, ws=P, ws_bytes=1 << 30):
    return status("tesm_b200_beam_select", logits, dtype, 400, 100, G, W, V, K, scores, None, lengths, -1, pad, alpha, P, P,
                  P, P, P, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,want", [(dict(dtype=2), 2), (dict(W=0), 1), (dict(W=33), 1), (dict(K=0), 1), (dict(K=33), 1),
                                     (dict(V=0), 1), (dict(V=1 << 31), 1), (dict(G=-1), 1), (dict(G=1 << 23), 1),
                                     (dict(logits=None), 1), (dict(scores=None), 1), (dict(alpha=1.0), 1),
                                     (dict(alpha=float("nan"), lengths=P), 1), (dict(pad=-1), 1), (dict(ws=None), 1),
                                     (dict(ws_bytes=15), 1), (dict(ws=ctypes.c_void_p((1 << 20) + 8)), 1), (dict(G=0), 0)])
def test_beam_select_refuses(kw, want):
    assert beam(**kw) == want
    if want:
        assert "beam_select" in _lib.last_error()


def test_beam_workspace():
    n = ctypes.c_int64(-1)
    assert status("tesm_b200_beam_select_workspace", 0, 2, 4, 32000, 4, ctypes.addressof(n)) == 0 and n.value > 0
    assert status("tesm_b200_beam_select_workspace", 1, 0, 4, 32000, 4, ctypes.addressof(n)) == 0 and n.value == 0
    assert status("tesm_b200_beam_select_workspace", 0, 2, 33, 32000, 4, ctypes.addressof(n)) == 1
    assert status("tesm_b200_beam_select_workspace", 0, 2, 4, 32000, 4, None) == 1


def rows(*entries):
    t = (_lib.StateRows * len(entries))()
    for e, (src, dst, n, s, d) in zip(t, entries):
        e.src, e.dst, e.row_bytes, e.src_stride, e.dst_stride = src, dst, n, s, d
    return t


@pytest.mark.parametrize("entry,G,Win,Wout,parents,want", [
    ((4096, 4096, 64, 64, 64), 2, 4, 33, P, 1), ((4096, 4096, 64, 64, 64), 2, 4, 0, P, 1),
    ((4096, 4096, 64, 64, 64), 2, 0, 4, P, 1), ((4096, 4096, 64, 64, 64), -1, 4, 4, P, 1),
    ((4096, 4096, 64, 64, 64), 2, 4, 4, None, 1), ((None, 4096, 64, 64, 64), 2, 4, 4, P, 1),
    ((4096, None, 64, 64, 64), 2, 4, 4, P, 1), ((4096, 4096, 64, 32, 64), 2, 4, 4, P, 1),
    ((4096, 4096, 64, 64, 32), 2, 4, 4, P, 1), ((4096, 4096, -1, 64, 64), 2, 4, 4, P, 1),
    ((4096, 4096, 64, 64, 64), 2, 1, 4, P, 1), ((4096, 4096, 64, 64, 128), 2, 4, 4, P, 1),
    ((4096, 4096, 1 << 36, 1 << 36, 1 << 36), 2, 4, 4, ctypes.c_void_p(1 << 60), 5), ((4096, 4096, 64, 64, 64), 0, 4, 4, P, 0),
    ((4096, 4096, 0, 0, 0), 2, 4, 4, P, 0)])
def test_reorder_refuses(entry, G, Win, Wout, parents, want):
    t = rows(entry)
    assert status("tesm_b200_reorder_states", ctypes.addressof(t), 1, G, Win, Wout, parents, None) == want


@pytest.mark.parametrize("parents", [4096, 4096 + 60, 4096 + 7 * 64 + 63, 4096 - 4])
def test_reorder_refuses_parents_inside_a_state(parents):
    t = rows((4096, 4096, 64, 64, 64))
    assert status("tesm_b200_reorder_states", ctypes.addressof(t), 1, 2, 4, 4, ctypes.c_void_p(parents), None) == 1
    assert "parents" in _lib.last_error()


def test_reorder_checks_every_state_before_the_first_launch():
    """200 states take two launches; a size that only the last one refuses refuses the call."""
    good, bad = (4096, 4096, 64, 64, 64), (4096, 4096, 1 << 36, 1 << 36, 1 << 36)
    t = rows(*[good] * 199, bad)
    assert status("tesm_b200_reorder_states", ctypes.addressof(t), 200, 2, 4, 4, ctypes.c_void_p(1 << 60), None) == 5


def test_reorder_refuses_no_table():
    assert status("tesm_b200_reorder_states", None, 1, 2, 4, 4, P, None) == 1
    assert status("tesm_b200_reorder_states", None, 0, 2, 4, 4, P, None) == 0


def conv(dtype=0, B=1, L=4, D=8, K=4, x=P, w=P, out=P):  # checks that come before the ones on shared memory
    return status("tesm_b200_causal_conv", x, dtype, 32, 8, B, L, D, K, w, None, None, None, 1, out, 32, 8, None)


@pytest.mark.parametrize("kw,want", [(dict(dtype=3), 2), (dict(B=-1), 1), (dict(L=-1), 1), (dict(D=1 << 31), 1),
                                     (dict(K=1), 5), (dict(K=9), 5), (dict(x=None), 1), (dict(w=None), 1),
                                     (dict(out=None), 1), (dict(B=1 << 29, L=64, D=1024), 1), (dict(L=0), 0), (dict(B=0), 0)])
def test_conv_refuses(kw, want):
    assert conv(**kw) == want


def scan(dtype=0, B=1, L=4, D=8, N=16, x=P, A=P, out=P, strides=True, ws=None, ws_bytes=0):
    s = (ctypes.c_int64 * 12)(*[64] * 12)
    return status("tesm_b200_ssm_scan", x, P, P, P, None, out, ctypes.addressof(s) if strides else None, dtype, B, L, D, N,
                  A, None, None, 1, None, None, ws, ws_bytes, None)


@pytest.mark.parametrize("kw,want", [(dict(dtype=3), 2), (dict(B=-1), 1), (dict(B=1 << 62), 1), (dict(L=1 << 30), 1), (dict(N=0), 5),
                                     (dict(N=129), 5), (dict(x=None), 1), (dict(A=None), 1), (dict(out=None), 1),
                                     (dict(strides=False), 1), (dict(B=1 << 29, D=64), 1), (dict(L=0), 0), (dict(D=0), 0)])
def test_scan_refuses(kw, want):
    assert scan(**kw) == want


def test_scan_workspace():
    """Long sequences of few channels need one; the call checks it before anything else runs."""
    n = ctypes.c_int64(-1)
    assert status("tesm_b200_ssm_scan_workspace", 1, 4096, 64, 16, ctypes.addressof(n)) == 0 and n.value > 0
    need = n.value
    for shape in [(1, 1, 64, 16), (1, 100, 64, 16), (0, 4096, 64, 16), (1, 4096, 0, 16), (64, 4096, 8192, 16)]:
        assert status("tesm_b200_ssm_scan_workspace", *shape, ctypes.addressof(n)) == 0 and n.value == 0
    assert status("tesm_b200_ssm_scan_workspace", 1, 4096, 64, 129, ctypes.addressof(n)) == 1
    assert status("tesm_b200_ssm_scan_workspace", 1, 4096, 64, 16, None) == 1
    s = (ctypes.c_int64 * 12)(*[64 * 4096, 64, 64 * 4096, 64, 16 * 4096, 16, 16 * 4096, 16, 0, 0, 64 * 4096, 64])
    at = [ctypes.c_void_p((i + 1) << 30) for i in range(8)]
    for ws, size in [(None, need), (at[6], need - 1), (ctypes.c_void_p((7 << 30) + 8), need)]:
        assert status("tesm_b200_ssm_scan", at[0], at[1], at[2], at[3], None, at[4], ctypes.addressof(s), 0, 1, 4096, 64, 16,
                      at[5], None, None, 1, None, None, ws, size, None) == 1
        assert "workspace" in _lib.last_error()
    for i in range(6):  # a workspace inside an input, A or out
        assert status("tesm_b200_ssm_scan", at[0], at[1], at[2], at[3], None, at[4], ctypes.addressof(s), 0, 1, 4096, 64, 16,
                      at[5], None, None, 1, None, None, at[i], need, None) == 1


def test_rows_disjoint():
    """Sets of rows (pointer, bytes, stride, rows): apart, interleaved in one buffer, overlapping."""
    d = ops._rows_disjoint
    assert d((0, 8, 8, 4), (32, 8, 8, 4)) and not d((0, 8, 8, 4), (24, 8, 8, 4))
    assert d((0, 8, 16, 4), (8, 8, 16, 4)) and d((8, 8, 16, 4), (0, 8, 16, 4))
    assert not d((0, 8, 16, 4), (4, 8, 16, 4)) and not d((0, 8, 16, 4), (12, 8, 16, 4))
    assert not d((0, 8, 16, 4), (8, 8, 24, 4)) and not d((0, 8, 8, 1), (0, 8, 8, 1))
    assert d((0, 0, 8, 4), (0, 8, 8, 4)) and d((0, 8, 8, 0), (0, 8, 8, 4))
    # by brute force
    g = torch.Generator().manual_seed(0)
    for _ in range(300):
        a, b = ([int(v) for v in torch.randint(0, 20, (4,), generator=g)] for _ in range(2))
        for t in (a, b):
            t[2] = max(t[1], 1) + t[2] % 5
            t[3] = t[3] % 4
        if int(torch.randint(0, 2, (1,), generator=g)):
            b[2] = max(a[2], b[1])
        cover = [set(p + r * s + i for r in range(k) for i in range(n)) for p, n, s, k in (a, b)]
        if ops._rows_disjoint(tuple(a), tuple(b)):
            assert not (cover[0] & cover[1]), (a, b)


def vp(n):
    return None if n is None else ctypes.c_void_p(n)


@pytest.mark.parametrize("x,w,state,lengths,out,ldo", [
    (4096, 1 << 16, None, None, 4096, (32, 8)), (4096, 1 << 16, None, None, 4096 + 4, (32, 8)),
    (4096, 1 << 16, None, None, 4096 + 252, (32, 8)), (4096, 1 << 16, 8192, None, 8192 + 188, (32, 8)),
    (4096, 1 << 16, 4096 + 255, None, 1 << 17, (32, 8)), (4096, 8192, None, None, 8192 + 124, (32, 8)),
    (4096, 8192, None, 1 << 17, (1 << 17) + 4, (32, 8)), (4096, 8192, None, None, 1 << 17, (32, 7)),
    (4096, 8192, None, None, 1 << 17, (8, 8)), (4096, 8192, None, None, 1 << 17, (0, 8)),
    (4096, 8192, None, None, 1 << 17, (15, 22)), (4096, 8192, None, None, 1 << 17, (-32, 8))])
def test_conv_refuses_shared_memory(x, w, state, lengths, out, ldo):
    """x (2, 4, 8) float32, weight (8, 4): out or state over an input, over each other or over itself."""
    assert status("tesm_b200_causal_conv", vp(x), 0, 32, 8, 2, 4, 8, 4, vp(w), None, vp(state), vp(lengths), 1, vp(out), *ldo,
                  None) == 1
    assert "causal_conv" in _lib.last_error()


@pytest.mark.parametrize("which", ["x", "dt", "bm", "cm", "z", "A", "skip", "bias", "lengths", "state", "self", "negative"])
@pytest.mark.parametrize("written", ["out", "state"])
def test_scan_refuses_shared_memory(which, written):
    at = {n: (i + 1) << 16 for i, n in enumerate(["x", "dt", "bm", "cm", "z", "out", "A", "skip", "bias", "state", "lengths"])}
    s = [32, 8] * 2 + [64, 16] * 2 + [32, 8] * 2
    if which == "self":
        s[10] = 24
    elif which == "negative":
        s[1] = -8
    elif which == "state":
        at["out"] = at["state"] + 4
    else:
        at[written] = at[which] + 4
    t = (ctypes.c_int64 * 12)(*s)
    assert status("tesm_b200_ssm_scan", *(vp(at[n]) for n in ("x", "dt", "bm", "cm", "z", "out")), ctypes.addressof(t), 0, 2, 4,
                  8, 16, vp(at["A"]), vp(at["skip"]), vp(at["bias"]), 1, vp(at["state"]), vp(at["lengths"]), None, 0,
                  None) == 1


def test_cpu_tensors_are_refused():
    z = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        ops.beam_select(z(1, 2, 8), z(1, 2))
    with pytest.raises(ValueError, match="CUDA"):
        ops.StateReorder([z(4, 3)], 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.causal_conv(z(1, 2, 8), z(8, 4))
    with pytest.raises(ValueError, match="CUDA"):
        ops.ssm_scan(z(1, 2, 8), z(1, 2, 8), z(8, 4), z(1, 2, 4), z(1, 2, 4))
