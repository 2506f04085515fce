"""Beam search end to end on the GPU: TESMLMHeadModel.beam_search against a plain beam search over
the model's own eager decode steps, and the serving operators together in a small recurrent
language model (convolution, scan, selection, reordering; prompt, single tokens, captured)."""
import math

import pytest
import torch

from helpers import build_model
from tesm_b200 import ops
from tesm_b200._lib import TesmError

pytestmark = pytest.mark.gpu

TINY = dict(n_layer=2, d_model=64, d_state=32, ent_rank=16, d_intermediate=96, vocab_size=128, max_seq_len=64,
            entanglement_window=8)
CFGS = {"siso": TINY, "mimo": dict(TINY, use_mimo=True, n_heads=2, d_state=16, ent_rank=8)}
STATES = ("state", "ent_k_cache", "ent_v_cache")


# A log-probability over at most 1024 words is off by at most 14 roundings: two hardware exponentials
# (2^-22 each, a word's and its thread's maximum's), their arguments (differences below 1 in size or
# exponentials that make up for it) and three additions in fp32; the rest is in fp64.
LOGP = 14 * 2.0 ** -24


def pick(logits, beams, K, eos, pad, alpha, off=0.0):
    """One plain selection step in 64 bits.  A beam is (key, score, parent, token, ended, length, error),
    the last a bound on how far the operator's fp32 score may be off (``off``: how far its logits are).  Returns the chosen beams of every
    prompt, and how often the bounds fit into the smallest gap between neighbouring keys."""
    G, W, V = logits.shape
    lp = torch.log_softmax(logits.double().cpu(), -1)
    res, room = [], math.inf
    for g in range(G):
        cand = []
        for w, (_, s, _, _, ended, n, err) in enumerate(beams[g]):
            if ended:
                cand.append((s / max(n, 1) ** alpha, s, w, pad, True, n, err))
                continue
            for v in torch.topk(lp[g, w], min(K, V)).indices.tolist():
                c = s + float(lp[g, w, v])
                cand.append((c / (n + 1) ** alpha, c, w, v, v == eos, n + 1, err + LOGP + 2 * off + abs(c) * 2.0 ** -24))
        cand.sort(key=lambda c: (-c[0], c[2], c[3]))
        for a, b in zip(cand[:K], cand[1:K + 1]):
            if a[2] != b[2]:  # within a beam the logits decide, without rounding
                room = min(room, (a[0] - b[0]) / (a[6] / max(a[5], 1) ** alpha + b[6] / max(b[5], 1) ** alpha))
        res.append(cand[:K])
    return res, room


START = (0.0, 0.0, 0, 0, False, 0, 0.0)


def plain_search(m, ids, W, steps, alpha, eos, pad):
    G, L = ids.shape
    ip = {"state_cache": m.backbone.allocate_inference_cache(G, 64)}
    logits = m(ids, inference_params=ip)[0].logits[:, -1:, :]
    beams, room = pick(logits, [[START]] * G, W, eos, pad, alpha)
    caches = m.backbone.allocate_inference_cache(G * W, 64)
    for i, c in ip["state_cache"].items():
        for n in STATES:
            caches[i][n].copy_(c[n].repeat_interleave(W, 0))
        caches[i]["seq_pos"], caches[i]["cache_idx"] = c["seq_pos"], c["cache_idx"]
    hyps = [[[b[3]] for b in beams[g]] for g in range(G)]
    for _ in range(1, steps):
        if all(b[4] for g in beams for b in g):
            break
        tok = torch.tensor([[h[-1]] for g in hyps for h in g], device="cuda")
        logits = m(tok, inference_params={"state_cache": caches})[0].logits[:, -1, :].view(G, W, -1)
        new, d = pick(logits, beams, W, eos, pad, alpha)
        room = min(room, d)
        rows = torch.tensor([g * W + b[2] for g in range(G) for b in new[g]], device="cuda")
        for c in caches.values():
            for n in STATES:
                c[n].copy_(c[n][rows])
        hyps = [[hyps[g][b[2]] + [b[3]] for b in new[g]] for g in range(G)]
        beams = new
    return hyps, beams, room


@pytest.mark.parametrize("kind", ["siso", "mimo"])
@pytest.mark.parametrize("G,W,L,alpha,use_graph", [(1, 2, 12, 0.0, False), (3, 4, 12, 1.0, True), (2, 5, 1, 0.7, True),
                                                   (1, 32, 5, 1.0, False)])
def test_model_beam_search(kind, G, W, L, alpha, use_graph):
    m = build_model(CFGS[kind]).cuda()
    ids = torch.randint(0, 128, (G, L), generator=torch.Generator().manual_seed(G), device="cpu").cuda()
    with torch.no_grad():
        hyps, beams, room = plain_search(m, ids, W, 10, alpha, None, 0)
        assert room > 1, "the plain search has a near tie"
        seq, score = m.beam_search(ids, num_beams=W, max_new_tokens=10, length_penalty=alpha, num_return_sequences=W,
                                   use_graph=use_graph)
    assert seq.shape == (G, W, L + 10) and (seq[:, :, :L] == ids[:, None]).all()
    assert seq[:, :, L:].tolist() == hyps
    want = torch.tensor([[b[0] for b in g] for g in beams], dtype=torch.float64)
    tol = torch.tensor([[b[6] / b[5] ** alpha for b in g] for g in beams]) + want.abs() * 2.0 ** -23
    assert ((score.double().cpu() - want).abs() <= tol).all()
    assert ops.device_status() == 0


@pytest.mark.parametrize("use_graph", [False, True])
def test_model_beam_search_with_eos(use_graph):
    m = build_model(CFGS["siso"]).cuda()
    ids = torch.randint(0, 128, (2, 9), generator=torch.Generator().manual_seed(5)).cuda()
    with torch.no_grad():
        free, _, _ = plain_search(m, ids, 3, 12, 1.0, None, 0)
        eos = free[0][0][2]  # a token that the best hypothesis takes early
        m.tesm_config.eos_token_id, m.tesm_config.pad_token_id = eos, 7
        hyps, _, room = plain_search(m, ids, 3, 12, 1.0, eos, 7)
        assert room > 1 and any(eos in h for g in hyps for h in g)
        seq, score = m.beam_search(ids, num_beams=3, max_new_tokens=12, num_return_sequences=3, use_graph=use_graph)
    got = seq[:, :, 9:].tolist()
    assert got == [[h + [7] * (len(got[0][0]) - len(h)) for h in g] for g in hyps]


def test_one_beam_is_greedy_and_caches_can_be_reused():
    m = build_model(CFGS["siso"]).cuda()
    ids = torch.randint(0, 128, (3, 8), generator=torch.Generator().manual_seed(2)).cuda()
    with torch.no_grad():
        want = m.generate(ids, max_new_tokens=9, temperature=0.0)
        for _ in range(2):
            seq, _ = m.beam_search(ids, num_beams=1, max_new_tokens=9)
            assert torch.equal(seq[:, 0], want)
        seq, _ = m.beam_search(ids, num_beams=4, max_new_tokens=1)
        assert torch.equal(seq[:, 0], want[:, :9])


def test_more_beams_than_words():
    """A vocabulary of 3: the first step fills 3 of 8 beams, the others start dead."""
    m = build_model(dict(TINY, vocab_size=3)).cuda()
    ids = torch.zeros(2, 4, dtype=torch.int64, device="cuda")
    with torch.no_grad():
        seq, score = m.beam_search(ids, num_beams=8, max_new_tokens=3, num_return_sequences=8)
        one, s1 = m.beam_search(ids, num_beams=8, max_new_tokens=1, num_return_sequences=8)
    assert torch.isfinite(score).all() and len({tuple(r) for r in seq[0].tolist()}) == 8
    assert torch.isfinite(s1[:, :3]).all() and torch.isinf(s1[:, 3:]).all()


def test_beam_search_refusals():
    m = build_model(CFGS["siso"]).cuda()
    ids = torch.zeros(1, 4, dtype=torch.int64, device="cuda")
    for kw in [dict(num_beams=0), dict(num_beams=33), dict(num_beams=2, num_return_sequences=3), dict(max_new_tokens=0),
               dict(max_new_tokens=62)]:
        with pytest.raises(ValueError):
            m.beam_search(ids, **kw)
    with pytest.raises(ValueError):
        m.beam_search(ids[0])
    m.backbone.layers[0].mlp.__dict__["_b200_tp"] = type("TP", (), {"world": 2})()
    with pytest.raises(TesmError):
        m.beam_search(ids, max_new_tokens=4)


# ------------------------------------------------------------------ the operators together
class RecurrentLM:
    """One selective state space layer between an embedding and an output matrix, on the serving
    operators or (plain=True) in 64 bits on the CPU."""

    def __init__(self, seed, V=97, D=24, N=8, K=4, plain=False):
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.p = dict(emb=r(V, 2 * D), conv=r(D, K) * 0.5, cb=r(D) * 0.1, bc=r(D, 2 * N) * 0.3, dtw=r(D, D) * 0.1,
                      A=-torch.rand(D, N, generator=g) * 4 - 0.1, skip=r(D), db=-2 + r(D), out=r(D, V))
        self.plain, self.V, self.D, self.N, self.K = plain, V, D, N, K
        self.p = {k: v.double() if plain else v.cuda() for k, v in self.p.items()}

    def states(self, rows):
        z = dict(dtype=torch.float64) if self.plain else dict(device="cuda")
        return [torch.zeros(rows, self.K - 1, self.D, **z), torch.zeros(rows, self.D, self.N, **z)]

    def __call__(self, ids, states):
        """Logits of the last token; the states move on."""
        p, cs, hs = self.p, *states
        e = p["emb"][ids]
        x, z = e[..., :self.D], e[..., self.D:]
        if not self.plain:
            x = ops.causal_conv(x, p["conv"], p["cb"], state=cs)
            bc = x @ p["bc"]
            y = ops.ssm_scan(x, x @ p["dtw"], p["A"], bc[..., :self.N], bc[..., self.N:], D=p["skip"], z=z,
                             dt_bias=p["db"], state=hs)
            return y[:, -1] @ p["out"]
        full = torch.cat([cs, x], 1)
        acc = sum(full[:, j:j + ids.shape[1]] * p["conv"][:, j] for j in range(self.K)) + p["cb"]
        cs.copy_(full[:, -(self.K - 1):])
        x = acc * torch.sigmoid(acc)
        bc, dt = x @ p["bc"], torch.nn.functional.softplus(x @ p["dtw"] + p["db"])
        for t in range(ids.shape[1]):
            hs.copy_(torch.exp(dt[:, t, :, None] * p["A"]) * hs +
                     (dt[:, t] * x[:, t])[..., None] * bc[:, t, None, :self.N])
            y = (hs * bc[:, t, None, self.N:]).sum(-1) + p["skip"] * x[:, t]
        y = y * z[:, -1] * torch.sigmoid(z[:, -1])
        # an fp32 logit lies behind some 128 roundings: the products with bc, dtw and out (24 terms each),
        # the convolution, the step, its exponentials and the sum over the states
        self.off = 128 * 2.0 ** -24 * float((y.abs() @ p["out"].abs()).max())
        return y @ p["out"]


@pytest.mark.parametrize("G,W,steps,seed", [(1, 4, 12, 21), (3, 5, 8, 39)])
def test_operators_together(G, W, steps, seed):
    """Prompt -> beams -> single tokens, the whole step captured in a graph and replayed, against the
    same search in 64 bits."""
    eos = 3
    ids = torch.randint(0, 97, (G, 11), generator=torch.Generator().manual_seed(W))
    ref = RecurrentLM(seed, plain=True)
    st = ref.states(G)
    beams, room = pick(ref(ids, st)[:, None], [[START]] * G, W, eos, 0, 1.0, ref.off)
    st = [s.repeat_interleave(W, 0) for s in st]
    hyps = [[[b[3]] for b in beams[g]] for g in range(G)]
    for _ in range(steps):
        tok = torch.tensor([[h[-1]] for g in hyps for h in g])
        beams, d = pick(ref(tok, st).view(G, W, -1), beams, W, eos, 0, 1.0, ref.off)
        room = min(room, d)
        rows = torch.tensor([g * W + b[2] for g in range(G) for b in beams[g]])
        st = [s[rows] for s in st]
        hyps = [[hyps[g][b[2]] + [b[3]] for b in beams[g]] for g in range(G)]
    assert room > 1, "the plain search has a near tie"

    lm = RecurrentLM(seed)
    kw = dict(eos_token_id=eos, length_penalty=1.0)
    with torch.no_grad():
        prompt = lm.states(G)
        step = ops.beam_select(lm(ids.cuda(), prompt)[:, None], torch.zeros(G, 1, device="cuda"), W,
                               lengths=torch.zeros(G, 1, dtype=torch.int32, device="cuda"), **kw)
        states = lm.states(G * W)
        ops.reorder_states(prompt, step.parents, out=states)
        seqs = torch.zeros(G * W, steps + 1, dtype=torch.int64, device="cuda")
        seqs[:, 0] = step.tokens.view(-1)
        plan = ops.StateReorder(states + [seqs], W)
        cur = step

        def one():
            logits = lm(cur.tokens.view(-1, 1), states).view(G, W, -1)
            new = ops.beam_select(logits, cur.scores, finished=cur.finished, lengths=cur.lengths, **kw)
            plan(new.parents)
            for name in ("tokens", "parents", "scores", "finished", "lengths"):
                getattr(cur, name).copy_(getattr(new, name))

        keep = [t.clone() for t in states + [seqs, cur.tokens, cur.parents, cur.scores, cur.finished, cur.lengths]]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            one()  # warm-up: the matrix products' workspaces
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one()
        for t, k in zip(states + [seqs, cur.tokens, cur.parents, cur.scores, cur.finished, cur.lengths], keep):
            t.copy_(k)
        for i in range(1, steps + 1):
            graph.replay()
            seqs[:, i] = cur.tokens.view(-1)
    assert seqs.view(G, W, -1).tolist() == hyps
    want = torch.tensor([[b[1] for b in g] for g in beams], dtype=torch.float64)
    assert ((cur.scores.cpu().double() - want).abs() <= torch.tensor([[b[6] for b in g] for g in beams])).all()
    for a, b in zip(states, st):
        # states behind the same roundings as a logit, less the last product
        assert ((a.cpu().double() - b).abs() <= 128 * 2.0 ** -24 * (1 + b.abs().max())).all()
    assert ops.device_status() == 0
