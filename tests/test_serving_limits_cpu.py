"""Serving operators at the limits of their entry points: sizes whose products leave 64 bits, and what
the checks on the host let through.  Without a GPU."""
import ctypes
import pathlib
import re

import pytest
import torch

from tesm_b200 import _lib

P = ctypes.c_void_p(1 << 20)  # never dereferenced: the checks come first


def status(name, *args):
    return getattr(_lib.load(), name)(*args)


@pytest.mark.parametrize("G,W", [(1 << 62, 4), (1 << 59, 32), (1 << 60, 16), ((1 << 62) + 1, 4), (1 << 24, 1),
                                 (((1 << 24) - 1) // 3 + 1, 3)])
def test_beam_prompts_whose_rows_leave_64_bits(G, W):
    """A product G * W that wraps to 0 would divide by 0, which ends the process: refused instead."""
    n = ctypes.c_int64(-1)
    assert status("tesm_b200_beam_select_workspace", 0, G, W, 100, 4, ctypes.addressof(n)) == 1 and n.value == -1
    assert status("tesm_b200_beam_select", P, 0, 400, 100, G, W, 100, 4, P, None, None, -1, 0, 0.0, P, P, P, P, P, P, 1 << 30,
                  None) == 1
    assert "bad shape" in _lib.last_error()


def test_beam_prompts_up_to_the_limit():
    n = ctypes.c_int64(-1)
    for W in (1, 3, 32):
        assert status("tesm_b200_beam_select_workspace", 1, ((1 << 24) - 1) // W, W, 1 << 30, 32, ctypes.addressof(n)) == 0
        assert n.value > 0
    assert status("tesm_b200_beam_select_workspace", 1, 1, 1, (1 << 30) + 1, 32, ctypes.addressof(n)) == 1


@pytest.mark.parametrize("B,L,D", [((1 << 62) + 1, 1, 512), (1 << 62, 1, 512), ((1 << 40) + 1, 1 << 29, 1 << 29), (1 << 31, 1, 1),
                                   ((1 << 30) + 1, 1 << 29, 1 << 29)])
def test_conv_sequences_whose_blocks_leave_64_bits(B, L, D):
    """The number of blocks wraps to a small one, and (int)B with it: only a part would be computed."""
    x, w, out = (ctypes.c_void_p(1 << k) for k in (41, 43, 45))
    assert status("tesm_b200_causal_conv", x, 0, 0, 0, B, L, D, 4, w, None, None, None, 1, out, D, 0, None) == 1
    assert "bad shape" in _lib.last_error() or "blocks" in _lib.last_error()


def test_memory_that_a_kernel_writes_is_not_read_through_the_read_only_path():
    """``__ldg`` is defined for memory that nobody writes while the kernel runs; the convolution shifts its
    window of inputs in place, so the window's rows come through ordinary loads."""
    text = (pathlib.Path(__file__).parents[1] / "tesm_b200" / "csrc" / "ssm.cu").read_text()
    pack = text[text.index("struct alignas"):text.index("\n};", text.index("struct alignas"))]
    bodies = re.split(r"__device__ __forceinline__ void (?=\w+\()", pack)[1:]
    read_only = [b.split("(")[0] for b in bodies if "__ldg" in b]
    assert read_only, "the test no longer finds the loads"
    calls = re.findall(r"\.(\w+)\((?:st|state|a\.state|ahead)\b", text)
    assert "load" in calls and not set(calls) & set(read_only), (calls, read_only)


def test_memory_written_while_a_kernel_waits_is_not_declared_read_only():
    """The selection's second kernel is resident while the first writes its statistics and lists: declared
    const __restrict__ they would count as constant for the kernel's life, and the compiler could load
    them before the wait."""
    text = (pathlib.Path(__file__).parents[1] / "tesm_b200" / "csrc" / "beam.cu").read_text()
    head = re.search(r"k_beam_pick\((.*?)\) \{", text, re.S).group(1)
    params = [" ".join(p.split()) for p in head.split(",")]
    for name in ("stat", "cval", "cidx"):
        (p,) = [p for p in params if re.search(rf"\b{name}$", p)]
        assert "*" in p and "__restrict__" not in p, p


@pytest.mark.skipif(torch.cuda.is_available(), reason="what the checks let through must find no device to run on")
def test_shared_memory_by_brute_force():
    """x and out (2, 3, n) float32 at strides and distances drawn at random: refused wherever a byte is
    shared, and let through as columns of one buffer."""
    g = torch.Generator().manual_seed(1)
    r = lambda lo, hi: int(torch.randint(lo, hi, (1,), generator=g))  # noqa: E731
    w = ctypes.c_void_p(1 << 40)
    passed = interleaved = 0
    for i in range(3000):
        n, base = r(1, 5), 1 << 20
        shape = [(r(1, 4), r(1, 4), n)] * 2
        if i % 2:  # columns of one buffer
            wide = 2 * n + r(0, 4)
            ld = [(wide * shape[0][1], wide) if i % 4 == 1 else (wide, wide * shape[0][0])] * 2
        else:
            ld = [(r(0, 40), r(0, 16)) for _ in range(2)]
        off = r(-12, 60)
        x, out = (set(4 * (o + b * lb + t * lt + c) + k for b in range(B) for t in range(T) for c in range(n) for k in range(4))
                  for (B, T, n), (lb, lt), o in zip(shape, ld, (0, off)))
        B, T, _ = shape[0]
        rc = status("tesm_b200_causal_conv", ctypes.c_void_p(base), 0, *ld[0], B, T, n, 2, w, None, None, None, 1,
                    ctypes.c_void_p(base + 4 * off), *ld[1], None)
        assert rc in (1, 3)
        if x & out or len(out) < 4 * B * T * n:
            assert rc == 1, (shape, ld, off)
        elif i % 2:
            # the rows as a whole lie apart, or between one another without a common byte modulo the buffer's width
            at = off % wide if off >= 0 else wide - (-off) % wide
            between = n <= at and at + n <= wide
            apart = max(x) < min(out) or max(out) < min(x)
            assert rc == 3 or not (between or apart), (shape, ld, off)
            interleaved += between and not apart
        passed += rc == 3
    assert passed > 300 and interleaved > 50


def segments(B, L, D, N):
    """Into how many segments a scan is cut: the workspace holds the states at each one's start and all sums
    of steps but the last."""
    n = ctypes.c_int64(-1)
    assert status("tesm_b200_ssm_scan_workspace", B, L, D, N, ctypes.addressof(n)) == 0
    s, rest = divmod(n.value // 4 + B * D, B * D * (N + 1))
    assert n.value == 0 or rest == 0
    return s if n.value else 1


@pytest.mark.parametrize("B,L,D,N,want", [
    # a block holds 128 channels of up to 4 states, an SM 4 blocks: 3 blocks per SM are no few channels
    (1, 4096, 3 * 148 * 128, 1, 1), (8, 4096, 8192, 1, 1), (1, 4096, 74 * 128, 1, 16), (1, 8192, 2048, 1, 32),
    # above 16 states an SM holds 2 blocks
    (1, 2048, 128 * 16, 32, 1), (1, 1024, 111 * 8, 64, 1), (1, 2048, 37 * 8, 64, 8), (1, 2048, 74 * 4, 128, 4),
    (1, 4096, 18 * 4, 128, 16), (3, 777, 771, 24, 1),
    # 4 to 16 states
    (1, 8192, 2048, 16, 16), (1, 4096, 4096, 16, 16), (1, 8192, 8192, 16, 1), (1, 512, 2048, 16, 4), (1, 511, 2048, 16, 1)])
def test_scan_is_cut_where_few_blocks_run(B, L, D, N, want):
    assert segments(B, L, D, N) == want
