"""Serving operators on the GPU where the documentation allows a call and a special case begins."""
import pytest
import torch

from tesm_b200 import _lib, ops
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
