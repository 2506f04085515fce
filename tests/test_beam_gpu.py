"""Beam search selection and state reordering on the GPU against plain 64-bit forms."""
import math

import numpy as np
import pytest
import torch

from tesm_b200 import _lib, ops

pytestmark = pytest.mark.gpu
NEG = float("-inf")


def pick64(logits, scores, K, finished=None, lengths=None, eos=None, pad=0, alpha=0.0):
    """The definition: every candidate's key in 64 bits, sorted by (-key, beam, token)."""
    G, W, V = logits.shape
    l = logits.double().cpu().numpy()
    l = np.where(np.isnan(l), NEG, np.minimum(l, float(torch.finfo(torch.float32).max)))
    sc = scores.double().cpu().numpy()
    fin = np.zeros((G, W), bool) if finished is None else finished.cpu().numpy()
    ln = np.zeros((G, W), np.int64) if lengths is None else lengths.cpu().numpy().astype(np.int64)
    out = dict(tokens=np.full((G, K), pad), parents=np.zeros((G, K), int), scores=np.full((G, K), NEG),
               finished=np.ones((G, K), bool), lengths=np.zeros((G, K), int))
    gaps = []
    for g in range(G):
        cand = []
        for w in range(W):
            n = ln[g, w] + (0 if fin[g, w] else 1)
            div = float(max(n, 1)) ** alpha
            if fin[g, w]:
                cand.append((sc[g, w] / div, w, pad, sc[g, w], n))
                continue
            m = l[g, w].max()
            if m == NEG:
                continue
            d = l[g, w] - m
            tot = np.exp(d).sum()
            c = sc[g, w] + (d - math.log(tot))
            for v in np.argsort(-l[g, w], kind="stable")[:K]:
                cand.append((c[v] / div, w, int(v), c[v], n))
        cand = [c for c in cand if c[0] > NEG]
        cand.sort(key=lambda c: (-c[0], c[1], c[2]))
        for a, b in zip(cand[:K], cand[1:K + 1]):
            if a[1] != b[1] and a[0] != b[0]:  # within a beam the logits decide, without rounding
                gaps.append(abs(a[0] - b[0]))
        for k in range(K):
            p = cand[k][1] if k < len(cand) else min(k, W - 1)
            out["parents"][g, k] = p
            out["lengths"][g, k] = ln[g, p]
            if k < len(cand):
                out["tokens"][g, k], out["scores"][g, k], out["lengths"][g, k] = cand[k][2], cand[k][3], cand[k][4]
                out["finished"][g, k] = fin[g, p] or (eos is not None and cand[k][2] == eos)
    return out, min(gaps, default=math.inf)


def score_tol(V, ref):
    """Bound on a score's error.  An exponential is off by 2^-22 (ex2.approx) and three roundings, a
    thread's 16 terms add 16 roundings, each of its steps two more, the joins (exponentials
    again) a dozen: relative to the sum, hence absolute on its logarithm.  One rounding of the
    result."""
    steps = -(-V // 4096)
    with np.errstate(invalid="ignore"):
        return (16 + 2 * steps + 24) * 2.0 ** -24 + np.where(np.isfinite(ref), np.abs(ref), 0) * 2.0 ** -24


def check(logits, scores, K=None, **kw):
    K = K or logits.shape[1]
    names = dict(finished="finished", lengths="lengths", eos="eos_token_id", pad="pad_token_id", alpha="length_penalty")
    ref, gap = pick64(logits, scores, K, **kw)
    V = logits.shape[2]
    # keys of different beams lie far enough apart for the order to be a matter of arithmetic
    assert gap > 4 * (40 + 2 * -(-V // 4096)) * 2.0 ** -24 + 1e-6, f"the inputs have a near tie ({gap})"
    before = ops.device_status()
    r = ops.beam_select(logits.cuda(), scores.cuda(), K, **{names[k]: v.cuda() if torch.is_tensor(v) else v
                                                            for k, v in kw.items()})
    assert r.tokens.dtype == torch.int64 and r.parents.dtype == torch.int32 and before == 0
    for name in ("tokens", "parents", "finished", "lengths"):
        np.testing.assert_array_equal(getattr(r, name).cpu().numpy(), ref[name], err_msg=name)
    got = r.scores.double().cpu().numpy()
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(ref["scores"]))
    ok = np.isfinite(got)
    assert (np.abs(got - ref["scores"])[ok] <= score_tol(V, ref["scores"])[ok]).all()
    return r


def rand(seed, *shape, dtype=torch.float32, scale=3.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("G,W,K,V", [(1, 1, 1, 1), (1, 1, 4, 7), (2, 3, 3, 33), (1, 4, 4, 4096), (3, 4, 4, 4097),
                                     (2, 5, 10, 8191), (1, 32, 32, 515), (5, 2, 32, 9000), (1, 7, 7, 151936),
                                     (40, 8, 8, 1000), (1, 32, 1, 12289)])
def test_select_sizes(G, W, K, V, dtype):
    check(rand(10 * V + W, G, W, V, dtype=dtype), rand(V, G, W), K)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("alpha", [0.0, 0.7, 1.0, -0.5])
def test_select_finished_and_penalty(dtype, alpha):
    G, W, V = 6, 5, 2000
    g = torch.Generator().manual_seed(3)
    fin = torch.rand(G, W, generator=g) < 0.5
    fin[0] = True  # a prompt whose beams have all ended
    ln = torch.randint(0, 50, (G, W), generator=g, dtype=torch.int32)
    logits = rand(4, G, W, V, dtype=dtype)
    scores = -rand(5, G, W).abs() * 4
    eos = int(logits[3, 0].float().argmax())
    check(logits, scores, finished=fin, lengths=ln, eos=eos, pad=11, alpha=alpha)


def test_ties_go_to_the_lowest_beam_and_token():
    # bf16 multiples of 1/4: hundreds of equal logits in a row; two beams with the same rows and scores
    V = 5003
    logits = (torch.round(rand(1, 2, 4, V) * 4 / 3) / 4).bfloat16()
    logits[:, 2] = logits[:, 1]
    scores = torch.tensor([[-1.0, -0.5, -0.5, -2.0], [0.0, 0.0, 0.0, 0.0]])
    scores[1] = torch.tensor([-3.0, -0.25, -0.25, -7.0])
    check(logits, scores, 32)
    check(torch.zeros(1, 3, V).bfloat16(), torch.tensor([[NEG, 0.0, NEG]]), 32)  # a flat row


@pytest.mark.parametrize("order", ["up", "down"])
def test_sorted_rows(order):
    # every logit (or none after the first) enters the candidate lists
    v = torch.arange(20000, dtype=torch.float32) / 1000
    v = v if order == "up" else v.flip(0)
    check(torch.stack([v, v + 0.0003]).view(1, 2, -1), torch.tensor([[0.0, -0.3704]]), 32)


def test_masked_values():
    V = 6000
    big = torch.finfo(torch.float32).max
    l = rand(2, 1, 8, V)
    l[0, 0, 5:] = NEG                      # five tokens left
    l[0, 1] = NEG                          # nothing left
    l[0, 2] = -big                         # masked by the type's lowest value: a flat row
    l[0, 3, ::2] = float("nan")            # NaN counts as -inf
    l[0, 4, 17] = float("inf")             # takes the whole mass
    l[0, 5, :] = float("nan")
    l[0, 6, 4096:] = -big
    l[0, 7, [3, 5000]] = float("inf")
    check(l, torch.tensor([[-0.1, 0.0, 9.1, -0.3, -12.3, 0.0, -0.6, -7.7]]), 32)


def test_dead_beams_and_empty_slots():
    V = 9
    l = rand(8, 3, 4, V)
    scores = torch.tensor([[0.0, NEG, NEG, NEG], [NEG] * 4, [float("nan"), -1.0, NEG, float("nan")]])
    l[0, 0, 2:] = NEG
    l[2, 1, 1:] = NEG
    r = check(l, scores, 6, eos=3, pad=5)
    assert torch.isinf(r.scores[1]).all() and r.finished[1].all() and (r.tokens[1] == 5).all()
    # the next step keeps them dead
    r2 = ops.beam_select(rand(9, 3, 6, V).cuda(), r.scores, finished=r.finished, lengths=r.lengths, pad_token_id=5)
    assert torch.isinf(r2.scores[1]).all() and r2.finished[1].all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("off", [0, 1, 3, 8])
def test_strided_logits_give_the_same_bits(dtype, off):
    """Row strides and unaligned rows change the loads, not the sums."""
    G, W, V = 3, 4, 4999
    base = rand(11, G, W, V, dtype=dtype).cuda()
    scores = rand(12, G, W).cuda()
    a = ops.beam_select(base, scores)
    wide = torch.full((W, G, V + 16 + off), float("nan"), dtype=dtype, device="cuda")  # beams outermost
    view = wide[:, :, off:off + V].transpose(0, 1)
    view.copy_(base)
    b = ops.beam_select(view, scores)
    for name in ("tokens", "parents", "scores", "finished", "lengths"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name
    # one beam over the same row again and again: a stride of zero
    c = ops.beam_select(base[:1, :1].expand(1, W, V), scores[:1])
    d = ops.beam_select(base[:1, :1].expand(1, W, V).contiguous(), scores[:1])
    assert torch.equal(c.tokens, d.tokens) and torch.equal(c.parents, d.parents) and torch.equal(c.scores, d.scores)


def test_no_prompts():
    r = ops.beam_select(torch.empty(0, 4, 100, device="cuda"), torch.empty(0, 4, device="cuda"))
    assert r.tokens.shape == (0, 4)


def test_select_on_a_stream_and_in_a_graph():
    G, W, V = 4, 4, 5000
    l, s = rand(20, G, W, V).cuda(), rand(21, G, W).cuda()
    want = ops.beam_select(l, s)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.beam_select(l, s)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got.tokens, want.tokens) and torch.equal(got.scores, want.scores)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        r = ops.beam_select(l, s)
    l2, s2 = rand(22, G, W, V).cuda(), rand(23, G, W).cuda()
    want2 = ops.beam_select(l2, s2)
    l.copy_(l2), s.copy_(s2)
    graph.replay()
    assert torch.equal(r.tokens, want2.tokens) and torch.equal(r.scores, want2.scores)


def test_select_refusals():
    l, s = torch.zeros(2, 3, 10, device="cuda"), torch.zeros(2, 3, device="cuda")
    f, n = torch.zeros(2, 3, dtype=torch.bool, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    for bad in [dict(logits=l.cpu()), dict(logits=l[0]), dict(scores=s.double()), dict(scores=s[:, :2]),
                dict(beams=0), dict(beams=33), dict(logits=l.transpose(1, 2).contiguous().transpose(1, 2)),
                dict(finished=f.int()), dict(lengths=n.long()), dict(length_penalty=1.0), dict(pad_token_id=10),
                dict(pad_token_id=-1), dict(scores=s.cpu()), dict(logits=torch.zeros(2, 3, 0, device="cuda")),
                dict(logits=torch.zeros(2, 33, 10, device="cuda"), scores=torch.zeros(2, 33, device="cuda"))]:
        kw = dict(logits=l, scores=s)
        kw.update(bad)
        with pytest.raises(ValueError):
            ops.beam_select(kw.pop("logits"), kw.pop("scores"), **kw)
    with pytest.raises(_lib.TesmError):
        ops.beam_select(l.half(), s)
    with torch.enable_grad(), pytest.raises(RuntimeError):
        ops.beam_select(l.requires_grad_(), s)


# ------------------------------------------------------------------ states
def moved(t, parents, W):
    G, K = parents.shape
    rows = (torch.arange(G)[:, None] * W + parents.cpu()).reshape(-1).to(t.device)
    return t[rows]


def bytes_like(seed, *shape, dtype):
    """Random bits (NaN patterns among them): the rows are copied as bits."""
    n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
    raw = torch.randint(0, 256, (n,), generator=torch.Generator().manual_seed(seed), dtype=torch.uint8).cuda()
    return raw.view(dtype).view(*shape)


def same_bits(a, b):
    return torch.equal(a.contiguous().view(torch.uint8), b.contiguous().view(torch.uint8))


@pytest.mark.parametrize("G,W", [(1, 1), (1, 2), (3, 4), (2, 5), (7, 8), (2, 13), (1, 16), (2, 17), (3, 32)])
def test_reorder_in_place(G, W):
    rows = G * W
    states = [bytes_like(1, rows, 37, dtype=torch.float64), bytes_like(2, rows, 5, 8, dtype=torch.float32),
              bytes_like(3, rows, 3, 11, dtype=torch.bfloat16), bytes_like(4, rows, 7, dtype=torch.uint8),
              bytes_like(5, rows, dtype=torch.int64), bytes_like(6, rows, 4096, dtype=torch.float32),
              torch.empty(rows, 0, device="cuda")]
    parents = torch.randint(0, W, (G, W), generator=torch.Generator().manual_seed(W), dtype=torch.int32).cuda()
    want = [moved(s, parents, W) for s in states]
    plan = ops.StateReorder(states, W)
    out = plan(parents)
    assert all(o is s and same_bits(s, w) for o, s, w in zip(out, states, want))
    # the plan again, with other parents, one beam taking all, and no move at all
    for p in (parents.flip(1).contiguous(), torch.full_like(parents, W - 1),
              torch.arange(W, dtype=torch.int32, device="cuda").expand(G, W).contiguous()):
        want = [moved(s, p, W) for s in states]
        plan(p)
        assert all(same_bits(s, w) for s, w in zip(states, want))
    assert ops.device_status() == 0


@pytest.mark.parametrize("off", [0, 1, 2, 4, 8])
def test_reorder_strides_and_what_lies_between(off):
    """Rows inside wider buffers, at every alignment; the bytes between the rows stay."""
    G, W, n = 3, 4, 48
    buf = bytes_like(9, G * W, n + 32, dtype=torch.uint8)
    keep = buf.clone()
    view = buf[:, off:off + n]
    parents = torch.randint(0, W, (G, W), generator=torch.Generator().manual_seed(1), dtype=torch.int32).cuda()
    want = moved(view, parents, W).clone()
    ops.reorder_states([view], parents)
    assert same_bits(view, want)
    keep[:, off:off + n] = want
    assert same_bits(buf, keep)


def test_reorder_layers_of_one_buffer_and_many_states():
    # (rows, layers, D): interleaved rows of 150 layers, more than one launch takes
    G, W = 2, 4
    base = bytes_like(10, G * W, 150, 6, dtype=torch.float32)
    want = moved(base, torch.tensor([[1, 1, 0, 3], [2, 0, 0, 0]]), W).clone()
    parents = torch.tensor([[1, 1, 0, 3], [2, 0, 0, 0]], dtype=torch.int32, device="cuda")
    ops.reorder_states([base[:, i] for i in range(150)], parents)
    assert same_bits(base, want)


@pytest.mark.parametrize("Win,Wout", [(1, 4), (1, 32), (8, 3), (3, 8), (4, 4)])
def test_reorder_into_other_tensors(Win, Wout):
    G = 3
    src = [bytes_like(1, G * Win, 33, dtype=torch.float32), bytes_like(2, G * Win, 2, 64, dtype=torch.float64)]
    dst = [torch.empty(G * Wout, *s.shape[1:], dtype=s.dtype, device="cuda") for s in src]
    parents = torch.randint(0, Win, (G, Wout), generator=torch.Generator().manual_seed(7), dtype=torch.int32).cuda()
    keep = [s.clone() for s in src]
    ops.reorder_states(src, parents, out=dst)
    for s, k, d in zip(src, keep, dst):
        assert same_bits(s, k) and same_bits(d, moved(s, parents, Win))


def test_parent_out_of_range_is_reported_and_moves_nothing():
    G, W = 2, 4
    s = bytes_like(3, G * W, 100, dtype=torch.float32)
    parents = torch.tensor([[1, 4, -1, 0], [3, 2, 1, 0x7fffffff]], dtype=torch.int32, device="cuda")
    ok = torch.tensor([[1, 1, 2, 0], [3, 2, 1, 3]])
    want = moved(s, ok, W)
    assert ops.device_status() == 0
    ops.reorder_states([s], parents)
    assert same_bits(s, want)
    assert ops.device_status() == 1 and ops.device_status() == 0


def test_reorder_refusals():
    s = torch.zeros(8, 16, device="cuda")
    p = torch.zeros(2, 4, dtype=torch.int32, device="cuda")
    t = torch.zeros(16, 8, device="cuda").t()
    for states, kw in [([], {}), ([s, s], {}), ([s, s[:, 4:]], {}), ([s[:4]], {}), ([t[:8]], {}),
                       ([s, torch.zeros(4, 3, device="cuda")], {}), ([s.cpu()], {}), ([s.t()], {}),
                       ([s[:1].expand(8, 16)], {}), ([s], dict(out=[s[:, :8]])), ([s], dict(out=[s.double()])),
                       ([s], dict(out=[s, s]))]:
        if states and states[0] is not None and kw == {} and len(states) == 1 and states[0].shape[0] == 4:
            p4 = torch.zeros(3, 4, dtype=torch.int32, device="cuda")
            with pytest.raises(ValueError):
                ops.reorder_states(states, p4)
            continue
        with pytest.raises(ValueError):
            ops.reorder_states(states, p, **kw)
    plan = ops.StateReorder([s], 4)
    for bad in (p.long(), p.cpu(), p[:1], p.t()):
        with pytest.raises(ValueError):
            plan(bad)
    with pytest.raises(ValueError):
        ops.StateReorder([s], 33)
    with pytest.raises(ValueError):
        ops.StateReorder([s], 3)
    with pytest.raises(ValueError):
        ops.StateReorder([s], 4, beams_in=2)


def test_reorder_in_a_graph_and_on_a_stream():
    G, W = 4, 4
    s = bytes_like(3, G * W, 1000, dtype=torch.float32)
    parents = torch.randint(0, W, (G, W), dtype=torch.int32, device="cuda")
    plan = ops.StateReorder([s], W)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        plan(parents)
    for seed in range(3):
        parents.copy_(torch.randint(0, W, (G, W), generator=torch.Generator().manual_seed(seed), dtype=torch.int32))
        want = moved(s, parents, W)
        graph.replay()
        assert same_bits(s, want)
    side = torch.cuda.Stream()
    want = moved(s, parents, W)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plan(parents)
    torch.cuda.current_stream().wait_stream(side)
    assert same_bits(s, want)
