"""Serving operators on the GPU where the documentation allows a call and a special case begins."""
import threading

import pytest
import torch

from tesm_b200 import _lib, ops
from test_beam_gpu import check as check_beam
from test_ssm_gpu import DT, check_conv, check_scan, conv64, cuda, inputs, rand, scan64

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ out between the columns of its inputs
@DT
@pytest.mark.parametrize("L", [1, 3, 37])
@pytest.mark.parametrize("D", [16, 9])
def test_conv_into_other_columns_of_its_projection(L, D, dtype):
    B = 3
    x, w, s = rand(1, B, L, D, dtype=dtype), rand(2, D, 4), rand(3, B, 3, D, dtype=dtype)
    y, tol, new = conv64(x, w, None, s)
    for order in ((0, 1), (1, 0)):
        proj = torch.full((B, L, 2 * D + 16), 7.0, dtype=dtype, device="cuda")
        proj[..., order[0] * D:][..., :D] = x.cuda()
        st = s.cuda()
        out = proj[..., order[1] * D:][..., :D]
        assert ops.causal_conv(proj[..., order[0] * D:][..., :D], w.cuda(), state=st, out=out) is out
        assert ((out.cpu().double() - y).abs() <= tol).all() and torch.equal(st.cpu(), new)
        assert torch.equal(proj[..., order[0] * D:][..., :D].cpu(), x) and (proj[..., 2 * D:] == 7).all()
        with pytest.raises(_lib.TesmError):  # one column too far
            ops.causal_conv(proj[..., :D], w.cuda(), out=proj[..., D - 1:2 * D - 1])


@DT
@pytest.mark.parametrize("L", [1, 45, 560])
def test_scan_into_other_columns_of_its_projection(L, dtype):
    B, C, N = 2, 24, 8
    kw = inputs(9, B, L, C, N, dtype)
    ref, tol, h, eh = scan64(**kw)
    proj = torch.full((B, L, 4 * C + 2 * N), 7.0, dtype=dtype, device="cuda")
    at, cols = 0, {}
    for name, n in (("x", C), ("Bm", N), ("out", C), ("dt", C), ("z", C), ("Cm", N)):
        cols[name] = proj[..., at:at + n]
        if name != "out":
            cols[name].copy_(kw[name])
        at += n
    before = {n: c.clone() for n, c in cols.items()}
    a = cuda(kw)
    ops.ssm_scan(cols["x"], cols["dt"], a["A"], cols["Bm"], cols["Cm"], D=a["D"], z=cols["z"], dt_bias=a["dt_bias"],
                 state=a["state"], out=cols["out"])
    assert ((cols["out"].cpu().double() - ref).abs() <= tol).all() and ((a["state"].cpu().double() - h).abs() <= eh).all()
    assert all(torch.equal(c, before[n]) for n, c in cols.items() if n != "out")
    with pytest.raises(_lib.TesmError):
        ops.ssm_scan(cols["x"], cols["dt"], a["A"], cols["Bm"], cols["Cm"], out=proj[..., C:2 * C])


# ------------------------------------------------------------------ both sides of the cut into segments
def segments(B, L, C, N):
    """As cut by the scan: its workspace holds the states at the segments' starts and all sums of steps but one."""
    n = ops._scan_workspace(B, L, C, N) // 4
    return (n + B * C) // (B * C * (N + 1)) if n else 1


@pytest.mark.parametrize("L,dtype", [(512, torch.bfloat16), (700, torch.float32), (1100, torch.bfloat16)])
@pytest.mark.parametrize("N", [1, 2, 16, 24])
def test_scan_on_both_sides_of_the_cut(N, L, dtype):
    """The most channels that are cut and the fewest that are not, by what the workspace says."""
    lo, hi = 1, 1 << 17
    assert segments(1, L, lo, N) > 1 and segments(1, L, hi, N) == 1
    while hi - lo > 1:
        mid = (lo + hi) // 2
        lo, hi = (mid, hi) if segments(1, L, mid, N) > 1 else (lo, mid)
    for C in (lo, hi):
        check_scan(inputs(L + C, 1, L, C, N, dtype, gate=L == 700, skip=L != 700))


# ------------------------------------------------------------------ decode batches
@DT
@pytest.mark.parametrize("L", [1, 3])
@pytest.mark.parametrize("kind", ["aligned", "odd"])
def test_conv_several_sequences_per_thread(kind, L, dtype):
    """Batches of short sequences so large that a thread takes four of them: blocks of 128 threads times 16 bytes
    (rows of odd width: one channel) of channels, 8 per SM or more.  A batch that is no multiple of four, sequences
    of length 0 and shorter than the window."""
    B, D, K = 301, {"odd": 505}.get(kind, 51200 // (8 * dtype.itemsize)), 4
    lengths = torch.randint(0, L + 1, (B,), generator=torch.Generator().manual_seed(3), dtype=torch.int32)
    assert 0 in lengths and L in lengths
    x = rand(1, B, L, D, dtype=dtype)
    for b, n in enumerate(lengths):
        x[b, n:] = float("nan")
    got = check_conv(x, rand(2, D, K), rand(3, D), rand(4, B, K - 1, D, dtype=dtype), lengths)
    assert torch.isfinite(got.float()).all()
    check_conv(torch.nan_to_num(x), rand(2, D, K), None, rand(4, B, K - 1, D, dtype=dtype))


@DT
@pytest.mark.parametrize("N", [1, 4, 6, 16, 128])
@pytest.mark.parametrize("B", [17, 33, 259])
def test_scan_tokens_of_many_sequences(B, N, dtype):
    """Single tokens beyond the 16 sequences that a thread takes, with remainders of the groups it takes at a time,
    and sequences without a token in all places of a group."""
    kw = inputs(B + N, B, 1, 19, N, dtype)
    lengths = torch.randint(0, 2, (B,), generator=torch.Generator().manual_seed(B), dtype=torch.int32)
    for name in ("x", "dt", "Bm", "Cm", "z"):
        kw[name][lengths == 0] = float("nan")
    got = check_scan(kw, lengths=lengths)
    assert torch.isfinite(got.float()).all() and (got[(lengths == 0).cuda()] == 0).all()
    for name in ("x", "dt", "Bm", "Cm", "z"):
        kw[name] = torch.nan_to_num(kw[name])
    check_scan(kw)


# ------------------------------------------------------------------ values that are not finite
@pytest.mark.parametrize("name,bad", [("x", float("inf")), ("x", float("nan")), ("dt", float("inf")), ("dt", float("nan"))])
@pytest.mark.parametrize("N", [1, 3, 16, 24])
@pytest.mark.parametrize("L", [1, 40, 600])
def test_scan_keeps_what_is_not_finite_in_its_channel(L, N, name, bad):
    """From the token on the channel's outputs and states are inf or NaN; other channels, and the outputs before,
    do not change."""
    B, C, at = 2, 9, L // 2
    kw = inputs(31, B, L, C, N, torch.float32)
    a = cuda(kw)
    clean = a["state"].clone()
    args = lambda k: (k["x"], k["dt"], k["A"], k["Bm"], k["Cm"])  # noqa: E731
    want = ops.ssm_scan(*args(a), D=a["D"], dt_bias=a["dt_bias"], state=clean)
    a[name][1, at, 4] = bad
    got = ops.ssm_scan(*args(a), D=a["D"], dt_bias=a["dt_bias"], state=a["state"])
    hit = torch.zeros(B, L, C, dtype=torch.bool, device="cuda")
    hit[1, at:, 4] = True
    assert not torch.isfinite(got[hit]).any() and torch.equal(got[~hit], want[~hit])
    rows = torch.zeros(B, C, dtype=torch.bool, device="cuda")
    rows[1, 4] = True
    assert not torch.isfinite(a["state"][rows]).any() and torch.equal(a["state"][~rows], clean[~rows])


# ------------------------------------------------------------------ beams
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("G,W,K,V", [(75, 8, 8, 1000), (19, 32, 4, 4999), (149, 4, 4, 8200)])
def test_select_more_rows_than_blocks_at_once(G, W, K, V, dtype):
    """Rows beyond the 592 blocks that 148 SMs hold, one part each."""
    check_beam(rand(G, G, W, V, dtype=dtype, scale=3.0), rand(V, G, W), K)


def test_select_from_several_threads():
    """Calls at once from host threads, each on a stream of its own."""
    G, W, V = 3, 4, 5000
    logits = [rand(i, G, W, V).cuda() * 3 for i in range(4)]
    scores = [rand(10 + i, G, W).cuda() for i in range(4)]
    want = [ops.beam_select(l, s) for l, s in zip(logits, scores)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            got = [ops.beam_select(logits[i], scores[i]) for _ in range(30)]
        stream.synchronize()
        wrong.extend(i for g in got for n in ("tokens", "parents", "scores", "finished", "lengths")
                     if not torch.equal(getattr(g, n), getattr(want[i], n)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not wrong
