"""Causal convolution and selective scan on the GPU against plain 64-bit recurrences.

Tolerances: the error of every step is bounded from the operations' own error bounds (rounding
2^-24 in fp32, 2^-22 relative for the hardware exponential and reciprocal) and carried through
the recurrence beside the values, so each element has its own bound.
"""
import pytest
import torch

from tesm_b200 import _lib, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def rand(seed, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def cuda(kw):
    return {k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()}


def silu64(x, err):
    """x sigmoid(x) and its error: |d/dx| <= 1.1; the exponential's argument is off by |x| 2^-23 and
    its value, the sum and the reciprocal by about 2^-21 together."""
    y = x * torch.sigmoid(x)
    return y, 1.1 * err + y.abs() * (x.abs() * 2 * U + 2.0 ** -20)


# ------------------------------------------------------------------ convolution
def conv64(x, weight, bias=None, state=None, lengths=None, silu=True):
    """y, its error bound and the new state."""
    B, L, D = x.shape
    K = weight.shape[1]
    y = torch.zeros(B, L, D, dtype=torch.float64)
    tol = torch.zeros_like(y)
    old = torch.zeros(B, K - 1, D, dtype=x.dtype) if state is None else state
    new = old.clone()
    for b in range(B):
        n = L if lengths is None else min(max(int(lengths[b]), 0), L)
        seq = torch.cat([old[b], x[b, :n]])
        new[b] = seq[n:]
        s = seq.double()
        for t in range(n):
            terms = s[t:t + K].t() * weight.double()
            b0 = bias.double() if bias is not None else torch.zeros(D, dtype=torch.float64)
            acc, mag = b0 + terms.sum(1), b0.abs() + terms.abs().sum(1)
            err = K * U * mag
            y[b, t], tol[b, t] = silu64(acc, err) if silu else (acc, err)
    return y, tol + y.abs() * half_step(x.dtype), new


def check_conv(x, weight, bias=None, state=None, lengths=None, silu=True, view=None):
    y, tol, new = conv64(x, weight, bias, state, lengths, silu)
    a = cuda(dict(x=x, weight=weight, bias=bias, state=state, lengths=lengths))
    if view is not None:
        a["x"] = view(a["x"])
    got = ops.causal_conv(a["x"], a["weight"], a["bias"], state=a["state"], lengths=a["lengths"], silu=silu)
    assert got.dtype == x.dtype
    off = (got.cpu().double() - y).abs()
    assert (off <= tol).all(), f"{(off / tol.clamp(min=1e-300)).max():.3g} times the bound"
    if state is not None:
        assert torch.equal(a["state"].cpu(), new)
    return got


DT = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])


@DT
@pytest.mark.parametrize("K", [2, 3, 4, 5, 6, 7, 8])
def test_conv_widths(K, dtype):
    x = rand(K, 2, 21, 40, dtype=dtype)
    check_conv(x, rand(K + 1, 40, K), rand(K + 2, 40), rand(K + 3, 2, K - 1, 40, dtype=dtype))


@DT
@pytest.mark.parametrize("B,L,D", [(1, 1, 1), (3, 1, 64), (2, 2, 7), (1, 3, 1030), (2, 64, 16), (1, 65, 24), (2, 130, 33),
                                   (1, 1000, 8)])
def test_conv_sizes(B, L, D, dtype):
    x = rand(L, B, L, D, dtype=dtype)
    check_conv(x, rand(1, D, 4), None, rand(2, B, 3, D, dtype=dtype), silu=False)
    check_conv(x, rand(1, D, 4), rand(3, D), None)


@DT
def test_conv_lengths_and_garbage_behind_them(dtype):
    B, L, D, K = 6, 19, 32, 4
    lengths = torch.tensor([0, 1, 2, 3, 19, 11], dtype=torch.int32)
    x = rand(1, B, L, D, dtype=dtype)
    for b, n in enumerate(lengths):
        x[b, n:] = float("nan")
        x[b, n + 1:] = float("inf")
    check_conv(x, rand(2, D, K), rand(3, D), rand(4, B, K - 1, D, dtype=dtype), lengths)
    # lengths outside 0 .. L count as the nearer end
    clipped = torch.tensor([-5, 1, 2, 3, 99, 11], dtype=torch.int32)
    a = ops.causal_conv(x.cuda(), rand(2, D, K).cuda(), lengths=lengths.cuda())
    b = ops.causal_conv(x.cuda(), rand(2, D, K).cuda(), lengths=clipped.cuda())
    assert torch.equal(a, b)


@DT
@pytest.mark.parametrize("D", [48, 20, 6])
@pytest.mark.parametrize("off", [0, 1, 4, 8])
def test_conv_strided_rows(off, D, dtype):
    """x and out as slices of wider buffers, at every alignment, batch innermost of the two; channels
    that end inside a 16-byte access."""
    B, L = 3, 37
    pad = 16 + -D % 8

    def wide(x):
        buf = torch.full((L, B, D + pad), float("nan"), dtype=dtype, device="cuda")
        v = buf[:, :, off:off + D].transpose(0, 1)
        v.copy_(x)
        return v

    x, w, s = rand(1, B, L, D, dtype=dtype), rand(2, D, 4), rand(3, B, 3, D, dtype=dtype)
    a = check_conv(x, w, None, s, view=wide)
    buf = torch.full((B, L, D + pad), 7.0, dtype=dtype, device="cuda")
    st = s.cuda()
    r = ops.causal_conv(x.cuda(), w.cuda(), state=st, out=buf[:, :, off:off + D])
    assert r.data_ptr() == buf[:, :, off:off + D].data_ptr() and torch.equal(r, a)
    rest = torch.ones(D + pad, dtype=torch.bool)
    rest[off:off + D] = False
    assert (buf[:, :, rest.cuda()] == 7).all()


@DT
def test_conv_prompt_in_pieces_gives_the_same_bits(dtype):
    B, L, D, K = 2, 90, 24, 4
    x, w, b = rand(1, B, L, D, dtype=dtype).cuda(), rand(2, D, K).cuda(), rand(3, D).cuda()
    s1 = torch.zeros(B, K - 1, D, dtype=dtype, device="cuda")
    whole = ops.causal_conv(x, w, b, state=s1)
    for cuts in ([1] * 90, [2, 1, 40, 47], [89, 1]):
        s2 = torch.zeros_like(s1)
        at, parts = 0, []
        for n in cuts:
            parts.append(ops.causal_conv(x[:, at:at + n], w, b, state=s2))
            at += n
        assert torch.equal(torch.cat(parts, 1), whole) and torch.equal(s1, s2)


def test_conv_empty():
    w = torch.zeros(8, 4, device="cuda")
    s = torch.ones(2, 3, 8, device="cuda")
    assert ops.causal_conv(torch.empty(2, 0, 8, device="cuda"), w, state=s).shape == (2, 0, 8)
    assert (s == 1).all()
    assert ops.causal_conv(torch.empty(0, 5, 8, device="cuda"), w).shape == (0, 5, 8)


def test_conv_refusals():
    x, w = torch.zeros(2, 5, 8, device="cuda"), torch.zeros(8, 4, device="cuda")
    st = torch.zeros(2, 3, 8, device="cuda")
    for a in [(x[0], w), (x.cpu(), w), (x, w[:, :1]), (x, torch.zeros(8, 9, device="cuda")), (x, w.bfloat16()),
              (x, w[:4]), (x.transpose(1, 2), torch.zeros(5, 4, device="cuda")), (x, w.cpu()), (x, w, w[:, 0])]:
        with pytest.raises(ValueError):
            ops.causal_conv(*a)
    for kw in [dict(state=st.bfloat16()), dict(state=st[:, :2]), dict(lengths=torch.zeros(2, device="cuda")),
               dict(out=torch.zeros(2, 5, 7, device="cuda")), dict(out=x.bfloat16()),
               dict(lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))]:
        with pytest.raises(ValueError):
            ops.causal_conv(x, w, **kw)
    both = torch.zeros(2 * 5 * 8 + 48, device="cuda")
    for kw in [dict(out=x), dict(out=torch.zeros(1, 5, 8, device="cuda").expand(2, 5, 8))]:
        with pytest.raises(_lib.TesmError):
            ops.causal_conv(x, w, **kw)
    with pytest.raises(_lib.TesmError):
        ops.causal_conv(both[:80].view(2, 5, 8), w, state=both[60:108].view(2, 3, 8))
    with pytest.raises(_lib.TesmError):
        ops.causal_conv(x.half(), w)
    with torch.enable_grad(), pytest.raises(RuntimeError):
        ops.causal_conv(x.clone().requires_grad_(), w)


# ------------------------------------------------------------------ scan
def scan64(x, dt, A, Bm, Cm, D=None, z=None, dt_bias=None, softplus=True, state=None, lengths=None):
    """out and the new state with an error bound for each."""
    B, L, C = x.shape
    N = A.shape[1]
    d64 = lambda t: t.double()  # noqa: E731
    h = torch.zeros(B, C, N, dtype=torch.float64) if state is None else state.double()
    H, E = h.abs(), torch.zeros_like(h)
    out = torch.zeros(B, L, C, dtype=torch.float64)
    tol = torch.zeros_like(out)
    n = torch.full((B,), L) if lengths is None else lengths.clamp(0, L)
    for t in range(L):
        on = (t < n)[:, None]
        raw = torch.where(on, d64(dt[:, t]), 0.0) + (0 if dt_bias is None else dt_bias.double())
        xt = torch.where(on, d64(x[:, t]), 0.0)
        bt, ct = torch.where(on, d64(Bm[:, t]), 0.0), torch.where(on, d64(Cm[:, t]), 0.0)
        if softplus:
            d = torch.nn.functional.softplus(raw, threshold=1e9)
            # raw is rounded; e^-|raw| is off by |raw| 2^-23 + 2^-22, the series by a few roundings
            ed = d * (2.0 ** -20 + raw.abs() * 2 * U) + raw.abs() * U * torch.sigmoid(raw)
        else:
            d, ed = raw, raw.abs() * U
        a = torch.exp(d[..., None] * A.double())
        arg = (d[..., None] * A.double()).abs()
        ra = 2.0 ** -22 + 3 * U * arg + ed[..., None] * A.double().abs()   # relative error of a
        u = (d * xt)[..., None] * bt[:, None, :]
        eu = u.abs() * 3 * U + (ed * xt.abs())[..., None] * bt.abs()[:, None, :]
        E1 = a * E + a * H * ra * 1.01 + eu
        H1 = a * H + u.abs()
        h1 = a * h + u
        E1 = E1 + 2 * U * H1
        k = on[..., None]
        h, H, E = torch.where(k, h1, h), torch.where(k, H1, H), torch.where(k, E1, E)
        y = (h * ct[:, None, :]).sum(-1)
        ey = (E * ct[:, None, :].abs()).sum(-1) + (N + 4) * U * (H * ct[:, None, :].abs()).sum(-1)
        if D is not None:
            y, ey = y + D.double() * xt, ey + 2 * U * (D.double() * xt).abs()
        if z is not None:
            g, eg = silu64(torch.where(on, d64(z[:, t]), 0.0), 0.0)
            ey = ey * g.abs() + y.abs() * eg + 2 * U * (y * g).abs()
            y = y * g
        out[:, t], tol[:, t] = torch.where(on, y, 0.0), torch.where(on, ey, 0.0)
    return out, tol + out.abs() * half_step(x.dtype), h, E + U * h.abs()


def inputs(seed, B, L, C, N, dtype, gate=True, state=True, skip=True):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    kw = dict(x=r(B, L, C).to(dtype), dt=(0.5 * r(B, L, C)).to(dtype),
              A=-torch.rand(C, N, generator=g) * N - 0.01, Bm=r(B, L, N).to(dtype), Cm=r(B, L, N).to(dtype),
              dt_bias=-4 + 2 * torch.rand(C, generator=g))
    if skip:
        kw["D"] = r(C)
    if gate:
        kw["z"] = r(B, L, C).to(dtype)
    if state:
        kw["state"] = r(B, C, N)
    return kw


def check_scan(kw, **change):
    kw = {**kw, **change}
    out, tol, h, eh = scan64(**kw)
    a = cuda(kw)
    got = ops.ssm_scan(a.pop("x"), a.pop("dt"), a.pop("A"), a.pop("Bm"), a.pop("Cm"), **a)
    assert got.dtype == kw["x"].dtype
    off = (got.cpu().double() - out).abs()
    assert (off <= tol).all(), f"out: {(off / tol.clamp(min=1e-300)).max():.3g} times the bound"
    if kw.get("state") is not None:
        off = (a["state"].cpu().double() - h).abs()
        assert (off <= eh).all(), f"state: {(off / eh.clamp(min=1e-300)).max():.3g} times the bound"
    return got


@DT
@pytest.mark.parametrize("N", [1, 2, 3, 4, 5, 8, 13, 16, 24, 32, 64, 100, 128])
@pytest.mark.parametrize("L", [1, 70])
def test_scan_state_sizes(N, L, dtype):
    check_scan(inputs(N, 2, L, 19, N, dtype))


@DT
@pytest.mark.parametrize("B,L,C,N", [(1, 1, 1, 16), (1, 2, 1, 16), (9, 1, 600, 16), (1, 33, 8, 16), (1, 300, 3, 4),
                                     (2, 129, 40, 8), (1, 64, 700, 2)])
def test_scan_sizes(B, L, C, N, dtype):
    check_scan(inputs(L, B, L, C, N, dtype))


@pytest.mark.parametrize("N", [2, 4, 8, 16, 32, 64, 128])
@pytest.mark.parametrize("C", [300, 2400, 19200])
def test_scan_lane_splits(N, C):
    """Numbers of channels at which the states of a channel are spread over fewer lanes."""
    check_scan(inputs(C + N, 1, 3, C, N, torch.float32))


@DT
@pytest.mark.parametrize("L", [127, 128, 255, 256, 257, 700])
@pytest.mark.parametrize("C,N", [(8, 16), (4, 3), (40, 1), (16, 17), (24, 33), (8, 128)])
def test_scan_few_channels(C, N, L, dtype):
    """Few channels and many tokens."""
    check_scan(inputs(L + N, 2, L, C, N, dtype))


@DT
@pytest.mark.parametrize("B,L,C,N", [(1, 511, 5, 16), (1, 512, 5, 16), (2, 1025, 9, 7), (1, 2100, 3, 128), (3, 640, 17, 24),
                                     (1, 1300, 1, 1), (1, 1100, 700, 2)])
def test_scan_in_segments(B, L, C, N, dtype):
    """Sequences of few channels are cut into segments from 512 tokens on."""
    check_scan(inputs(L, B, L, C, N, dtype))


@DT
@pytest.mark.parametrize("state", [True, False])
def test_scan_in_segments_ragged(state, dtype):
    lengths = torch.tensor([0, 1, 128, 129, 600, 900, 1023], dtype=torch.int32)
    kw = inputs(22, 7, 1023, 6, 16, dtype, state=state)
    for name in ("x", "dt", "Bm", "Cm", "z"):
        for b, n in enumerate(lengths):
            kw[name][b, n:] = float("nan")
    got = check_scan(kw, lengths=lengths)
    assert torch.isfinite(got.float()).all()


@pytest.mark.parametrize("A", [-0.01, -50.0])
def test_scan_in_segments_keeps_an_infinite_state(A):
    """A state that has overflowed stays infinite and does not turn into NaN, not by a decay that is 0
    over a segment either."""
    kw = inputs(23, 1, 1024, 4, 8, torch.float32)
    kw["dt"], kw["dt_bias"] = torch.full_like(kw["dt"], 0.1), torch.zeros(4)
    kw["A"] = torch.full_like(kw["A"], A)
    kw["state"][0, 1, 2] = float("inf")
    a = cuda(kw)
    ops.ssm_scan(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], dt_bias=a["dt_bias"], state=a["state"])
    assert a["state"][0, 1, 2] == float("inf") and torch.isfinite(a["state"]).sum() == 31


@pytest.mark.parametrize("first", [0, 300, 1020])
def test_scan_in_segments_growth(first):
    """Decays above 1 whose product over a segment leaves fp32's range, in front of the first input: the
    states are 0 until then."""
    kw = inputs(25, 1, 1024, 4, 8, torch.float32, state=False)
    kw["dt"], kw["dt_bias"] = torch.full_like(kw["dt"], 2.0), torch.zeros(4)
    kw["A"] = torch.full_like(kw["A"], 3.0 if first == 1020 else -3.0)
    kw["x"][:, :first] = 0
    check_scan(kw)


@pytest.mark.parametrize("lengths", [(9, 4), (1, 1)])
def test_scan_infinite_A(lengths):
    """A = -inf forgets at every token, and only there: not at the padding behind the end."""
    L = max(lengths)
    kw = inputs(26, 2, L, 5, 4, torch.float32)
    kw["A"][:] = float("-inf")
    a = cuda(kw)
    ops.ssm_scan(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], dt_bias=a["dt_bias"], state=a["state"],
                 lengths=torch.tensor(lengths, dtype=torch.int32, device="cuda"))
    for b, n in enumerate(lengths):
        dt = torch.nn.functional.softplus(kw["dt"][b, n - 1].double() + kw["dt_bias"].double())
        h = (dt * kw["x"][b, n - 1].double())[:, None] * kw["Bm"][b, n - 1].double()
        # softplus as in scan64: (1 + |raw| (2^-3 + 2^-4)) 2^-20 with |raw| < 8, two products
        assert ((a["state"][b].cpu().double() - h).abs() <= h.abs() * 3 * 2.0 ** -20).all()
    a["dt"].zero_()
    before = a["state"].clone()
    ops.ssm_scan(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], softplus=False, state=a["state"])
    assert torch.equal(a["state"], before)


def test_scan_in_segments_captured():
    """The two launches and their workspace in a graph, replayed beside eager calls."""
    kw = cuda(inputs(24, 1, 1500, 12, 16, torch.bfloat16))
    args = (kw["x"], kw["dt"], kw["A"], kw["Bm"], kw["Cm"])
    st, first = kw["state"].clone(), kw["state"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.ssm_scan(*args, z=kw["z"], state=st)
    for _ in range(3):
        want = ops.ssm_scan(*args, z=kw["z"], state=first)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(st, first)


@DT
@pytest.mark.parametrize("gate,state,skip", [(False, True, False), (True, False, True), (False, False, False)])
def test_scan_few_channels_ragged(gate, state, skip, dtype):
    lengths = torch.tensor([0, 1, 300, 256, 8, 257], dtype=torch.int32)
    kw = inputs(20, 6, 300, 24, 18, dtype, gate, state, skip)
    for name in ("x", "dt", "Bm", "Cm", "z"):
        for b, n in enumerate(lengths):
            if name in kw:
                kw[name][b, n:] = float("nan")
    got = check_scan(kw, lengths=lengths)
    assert torch.isfinite(got.float()).all()


@DT
def test_scan_few_channels_in_pieces_and_strided(dtype):
    """The kernels for prompts and tokens continue one another; rows inside wider buffers."""
    B, L, C, N = 2, 600, 16, 16
    kw = inputs(21, B, L, C, N, dtype)
    out, tol, h, eh = scan64(**kw)
    a = cuda(kw)
    proj = torch.full((B, L, 3 * C + 2 * N + 16), float("nan"), dtype=dtype, device="cuda")
    at = 8
    for name, n in (("x", C), ("dt", C), ("z", C), ("Bm", N), ("Cm", N)):
        proj[..., at:at + n] = a[name]
        a[name] = proj[..., at:at + n]
        at += n
    buf = torch.full((B, L, C + 16), 7.0, dtype=dtype, device="cuda")
    for cuts in ([600], [300, 1, 128, 171], [40, 560]):
        st, at = a["state"].clone(), 0
        for n in cuts:
            s = slice(at, at + n)
            ops.ssm_scan(a["x"][:, s], a["dt"][:, s], a["A"], a["Bm"][:, s], a["Cm"][:, s], D=a["D"], z=a["z"][:, s],
                         dt_bias=a["dt_bias"], state=st, out=buf[:, s, 8:8 + C])
            at += n
        assert ((buf[..., 8:8 + C].cpu().double() - out).abs() <= tol).all()
        assert ((st.cpu().double() - h).abs() <= eh).all()
        assert (buf[..., :8] == 7).all() and (buf[..., 8 + C:] == 7).all()


@DT
@pytest.mark.parametrize("gate,state,skip,bias,softplus", [(False, True, True, True, True), (True, False, False, False, True),
                                                           (False, False, False, False, False),
                                                           (True, True, True, True, False)])
@pytest.mark.parametrize("L", [1, 40])
def test_scan_optional_arguments(gate, state, skip, bias, softplus, L, dtype):
    kw = inputs(5, 2, L, 33, 16, dtype, gate, state, skip)
    if not softplus:
        kw["dt"] = kw["dt"].float().abs().mul(0.1).to(dtype)
        kw["dt_bias"] = kw["dt_bias"].abs() * 0.01
    if not bias:
        kw["dt_bias"] = None
    check_scan(kw, softplus=softplus)


@DT
def test_scan_lengths_and_garbage_behind_them(dtype):
    lengths = torch.tensor([0, 1, 70, 33, 64, 69], dtype=torch.int32)
    kw = inputs(6, 6, 70, 21, 16, dtype)
    for name in ("x", "dt", "Bm", "Cm", "z"):
        for b, n in enumerate(lengths):
            kw[name][b, n:] = float("nan")
            kw[name][b, n + 1:] = float("inf")
    got = check_scan(kw, lengths=lengths)
    assert torch.isfinite(got.float()).all()
    one = inputs(7, 6, 1, 21, 16, dtype)
    one["x"][0] = float("nan")
    check_scan(one, lengths=torch.tensor([0, 1, 5, 0, 1, -3], dtype=torch.int32))


def test_scan_extreme_steps():
    """Steps of 0, tiny and huge steps, decays that are 0 and 1, growth (A > 0)."""
    kw = inputs(8, 1, 24, 6, 4, torch.float32)
    kw["dt_bias"] = torch.zeros(6)
    kw["dt"] = torch.tensor([-200.0, -60.0, -20.0, 0.0, 30.0, 90.0]).expand(1, 24, 6).contiguous()
    kw["A"] = torch.tensor([-0.5, -1e-6, -1e6, 1e-3]).expand(6, 4).contiguous()
    check_scan(kw)


@pytest.mark.parametrize("L", [1, 2, 100, 700])
@pytest.mark.parametrize("N", [1, 2, 7, 16])
def test_scan_step_of_zero_keeps_the_state(N, L):
    """exp(0) is 1: not a bit of a state changes, in front of the end or behind it."""
    kw = inputs(L, 3, L, 11, N, torch.float32)
    kw["dt"].zero_()
    a = cuda(kw)
    ops.ssm_scan(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], softplus=False, state=a["state"],
                 lengths=torch.tensor([L, 1, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(a["state"].cpu(), kw["state"])


@DT
@pytest.mark.parametrize("B,L,C,N", [(10, 73, 1166, 4), (2, 200, 70, 16), (1, 700, 60, 16), (1, 700, 30, 1)])
def test_scan_errors_do_not_add_up(B, L, C, N, dtype):
    """The states' error over all channels, with steps of 0.001 to 0.1.  A decay of that size is rounded
    in its 24th bit (at random: 3e-8 root mean square), and a state remembers the last L of them at
    most: with errors of one sign, e each, the norm would be off by up to L e, at random by sqrt(L) 3e-8, to
    which the state's own roundings, the step and its product with A add as much: 2 sqrt(L) 6e-8."""
    g = torch.Generator().manual_seed(L + N)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    step = torch.exp(torch.rand(C, generator=g) * 4.6 - 6.9)
    kw = dict(x=r(B, L, C).to(dtype), dt=(0.5 * r(B, L, C)).to(dtype), Bm=r(B, L, N).to(dtype), Cm=r(B, L, N).to(dtype),
              A=-(torch.arange(1, N + 1).float() * torch.exp(0.1 * r(C, N))), dt_bias=step + torch.log(-torch.expm1(-step)),
              state=r(B, C, N))
    h = scan64(**kw)[2]
    a = cuda(kw)
    ops.ssm_scan(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], dt_bias=a["dt_bias"], state=a["state"])
    assert (a["state"].cpu().double() - h).norm() <= h.norm() * 2 * L ** 0.5 * 6e-8


@DT
@pytest.mark.parametrize("off", [0, 1, 4, 8])
@pytest.mark.parametrize("L,C,N", [(45, 24, 8), (1, 24, 8), (560, 24, 8), (1, 20, 6)])
def test_scan_strided_inputs(L, C, N, off, dtype):
    """All inputs as slices of one projection, at every alignment; out inside a wider buffer."""
    B = 2
    kw = inputs(9, B, L, C, N, dtype)
    a = cuda(kw)
    want_state = a["state"].clone()
    want = ops.ssm_scan(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], D=a["D"], z=a["z"], dt_bias=a["dt_bias"],
                        state=want_state)
    proj = torch.full((L, B, off + 3 * C + 2 * N + 8), float("nan"), dtype=dtype, device="cuda").transpose(0, 1)
    at = off
    for name, n in (("x", C), ("dt", C), ("z", C), ("Bm", N), ("Cm", N)):
        proj[..., at:at + n] = a[name]
        a[name] = proj[..., at:at + n]
        at += n
    buf = torch.full((B, L, C + 16), 7.0, dtype=dtype, device="cuda")
    out = buf[..., off:off + C]
    got = ops.ssm_scan(a["x"], a["dt"], a["A"], a["Bm"], a["Cm"], D=a["D"], z=a["z"], dt_bias=a["dt_bias"],
                       state=a["state"], out=out)
    assert got is out and torch.equal(got, want) and torch.equal(a["state"], want_state)
    ref, tol, h, eh = scan64(**kw)
    assert ((got.cpu().double() - ref).abs() <= tol).all() and ((a["state"].cpu().double() - h).abs() <= eh).all()
    rest = torch.ones(C + 16, dtype=torch.bool)
    rest[off:off + C] = False
    assert (buf[:, :, rest.cuda()] == 7).all()


def test_scan_broadcast_inputs():
    kw = inputs(10, 3, 20, 16, 16, torch.float32)
    kw["Bm"] = kw["Bm"][:1].expand(3, -1, -1)
    kw["dt"] = kw["dt"][:, :1].expand(-1, 20, -1)
    check_scan(kw)


@DT
def test_scan_prompt_in_pieces(dtype):
    """A prompt in pieces, down to single tokens, against the whole and the same bounds."""
    B, L, C, N = 2, 70, 40, 16
    kw = inputs(11, B, L, C, N, dtype)
    out, tol, h, eh = scan64(**kw)
    a = cuda(kw)
    for cuts in ([1] * L, [1, 30, 39], [69, 1]):
        st = a["state"].clone()
        parts, at = [], 0
        for n in cuts:
            s = slice(at, at + n)
            parts.append(ops.ssm_scan(a["x"][:, s], a["dt"][:, s], a["A"], a["Bm"][:, s], a["Cm"][:, s], D=a["D"],
                                      z=a["z"][:, s], dt_bias=a["dt_bias"], state=st))
            at += n
        assert ((torch.cat(parts, 1).cpu().double() - out).abs() <= tol).all()
        assert ((st.cpu().double() - h).abs() <= eh).all()


@pytest.mark.parametrize("L", [1, 50])
def test_scan_twice_gives_the_same_bits(L):
    kw = cuda(inputs(12, 4, L, 200, 16, torch.bfloat16))
    run = lambda st: ops.ssm_scan(kw["x"], kw["dt"], kw["A"], kw["Bm"], kw["Cm"], D=kw["D"], z=kw["z"],  # noqa: E731
                                  dt_bias=kw["dt_bias"], state=st)
    s1, s2 = kw["state"].clone(), kw["state"].clone()
    assert torch.equal(run(s1), run(s2)) and torch.equal(s1, s2)


def test_scan_in_a_graph_and_on_a_stream():
    kw = cuda(inputs(13, 2, 40, 64, 16, torch.float32))
    args = (kw["x"], kw["dt"], kw["A"], kw["Bm"], kw["Cm"])
    st = kw["state"].clone()
    first = kw["state"].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.ssm_scan(*args, state=st)
        cv = ops.causal_conv(kw["x"], torch.ones(64, 3, device="cuda"))
    for _ in range(2):
        want = ops.ssm_scan(*args, state=first)
        graph.replay()
        assert torch.equal(out, want) and torch.equal(st, first)
    assert torch.equal(cv, ops.causal_conv(kw["x"], torch.ones(64, 3, device="cuda")))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.ssm_scan(*args, state=st)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, ops.ssm_scan(*args, state=first))


def test_scan_empty():
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    st = torch.ones(2, 4, 8, device="cuda")
    assert ops.ssm_scan(z(2, 0, 4), z(2, 0, 4), z(4, 8), z(2, 0, 8), z(2, 0, 8), state=st).shape == (2, 0, 4)
    assert (st == 1).all()
    assert ops.ssm_scan(z(0, 3, 4), z(0, 3, 4), z(4, 8), z(0, 3, 8), z(0, 3, 8)).shape == (0, 3, 4)


def test_scan_refusals():
    z = lambda *s: torch.zeros(*s, device="cuda")  # noqa: E731
    good = dict(x=z(2, 5, 4), dt=z(2, 5, 4), A=z(4, 8), Bm=z(2, 5, 8), Cm=z(2, 5, 8), D=z(4), z=z(2, 5, 4),
                dt_bias=z(4), state=z(2, 4, 8), lengths=torch.zeros(2, dtype=torch.int32, device="cuda"))
    call = lambda k: ops.ssm_scan(k.pop("x"), k.pop("dt"), k.pop("A"), k.pop("Bm"), k.pop("Cm"), **k)  # noqa: E731
    call(dict(good))
    for name, bad in [("x", z(2, 5)), ("x", good["x"].cpu()), ("dt", z(2, 5, 3)), ("dt", good["dt"].bfloat16()),
                      ("A", z(4)), ("A", z(4, 0)), ("A", z(4, 129)), ("A", z(8, 4).t()), ("A", z(4, 8).double()),
                      ("Bm", z(2, 5, 7)), ("Cm", z(2, 8, 5).transpose(1, 2)), ("D", z(5)), ("z", z(2, 4, 5).transpose(1, 2)),
                      ("dt_bias", z(8)[::2]), ("state", z(2, 4, 8).double()), ("state", z(2, 8, 4).transpose(1, 2)),
                      ("state", z(1, 4, 8).expand(2, 4, 8)), ("lengths", z(2)), ("out", z(2, 5, 4).bfloat16())]:
        with pytest.raises(ValueError):
            call({**good, name: bad})
    for bad in (good["x"], good["z"], z(1, 5, 4).expand(2, 5, 4)):
        with pytest.raises(_lib.TesmError):
            call({**good, "out": bad})
    with pytest.raises(_lib.TesmError):
        call({**good, "x": good["x"].half()})
    with torch.enable_grad(), pytest.raises(RuntimeError):
        call({**good, "A": z(4, 8).requires_grad_()})
