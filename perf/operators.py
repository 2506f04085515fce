"""The operators of serving with recurrent states, as cases that can be timed and compared.

Four operators: ``beam_select`` (one step of beam search over beams and vocabulary),
``reorder_states`` (the recurrent caches follow the chosen beams), ``causal_conv`` (the short
depthwise convolution in front of a selective scan) and ``ssm_scan`` (h_t = a_t * h_{t-1} + B_t x_t,
y_t = C_t . h_t with input-dependent a, B and C), the last two for prompts and for single tokens.

``run`` computes a case in plain torch operations where ``own`` is false and with the framework's
operators where it is true.  Sizes follow the framework's configurations (d_model 2048 / 4096 with
expand 2, d_state 256, ent_rank 64, window 16, 32 layers, vocabularies 32000 and 151936, batch 256
decode) or are generic.
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ESIZE = {"bf16": 2, "f32": 4}
EOS, PAD = 2, 0


# ------------------------------------------------------------------ cases
def listed():
    return [
        # one prompt, four beams: the smallest step of a chat turn, where latency counts
        dict(name="beam one prompt", op="beam", G=1, W=4, V=32000, dtype="bf16", alpha=0.0, done=0),
        # the batch-256 decode step: 64 prompts of four beams, a quarter of the beams ended
        dict(name="beam decode batch", op="beam", G=64, W=4, V=32000, dtype="bf16", alpha=1.0, done=64),
        # wide beams over the default (large) vocabulary with fp32 logits
        dict(name="beam wide f32", op="beam", G=8, W=32, V=151936, dtype="f32", alpha=0.6, done=16),
        # the decode caches of 32 layers follow four beams of one prompt
        dict(name="reorder one prompt", op="reorder", kind="tesm", layers=32, G=1, W=4, D=256, R=64, win=16),
        # the same for the batch-256 decode step
        dict(name="reorder decode batch", op="reorder", kind="tesm", layers=32, G=64, W=4, D=256, R=64, win=16),
        # a batch of four prompts of 4096 tokens at d_model 4096, expand 2
        dict(name="conv prompt", op="conv", B=4, L=4096, D=8192, K=4, dtype="bf16", ragged=False, bias=True),
        # padded prompts of odd lengths and an odd width that go on from an earlier window
        dict(name="conv ragged f32", op="conv", B=5, L=1021, D=1537, K=3, dtype="f32", ragged=True, bias=False),
        # one token for each of 256 sequences
        dict(name="conv token", op="conv", B=256, L=1, D=8192, K=4, dtype="bf16", ragged=False, bias=True),
        # one prompt of 4096 tokens at d_model 4096, expand 2
        dict(name="scan prompt", op="scan", B=1, L=4096, D=8192, N=16, dtype="bf16", ragged=False, gate=True),
        # a long prompt with few channels: work only along the sequence
        dict(name="scan long", op="scan", B=1, L=8192, D=2048, N=16, dtype="bf16", ragged=False, gate=True),
        # padded prompts of odd lengths, odd width, a state size that is no power of two
        dict(name="scan ragged f32", op="scan", B=3, L=777, D=771, N=24, dtype="f32", ragged=True, gate=False),
        # one token for each of 256 sequences: the state is read and written once
        dict(name="scan token", op="scan", B=256, L=1, D=8192, N=16, dtype="bf16", ragged=False, gate=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["beam", "reorder", "conv", "scan", "conv token", "scan token"])
    dtype = rng.choice(["bf16", "f32"])
    if op == "beam":
        W = rng.randint(1, 32)
        V = _log(rng, 500, 151936)
        G = _log(rng, 1, max(1, min(64, 38_000_000 // (W * V))))
        return dict(op="beam", G=G, W=W, V=V, dtype=dtype, alpha=rng.choice([0.0, 0.6, 1.0]),
                    done=rng.randint(0, G * W // 2))
    if op == "reorder":
        W = rng.randint(2, 32)
        return dict(op="reorder", kind=rng.choice(["tesm", "ssm"]), layers=rng.randint(1, 32),
                    G=_log(rng, 1, max(1, 256 // W)), W=W, D=_log(rng, 33, 512), R=_log(rng, 8, 128),
                    win=rng.randint(2, 24))
    if op.startswith("conv"):
        D = _log(rng, 64, 8192)
        L = 1 if op.endswith("token") else _log(rng, 2, 4096)
        B = _log(rng, 1, max(1, min(256, 120_000_000 // (L * D))))
        return dict(op="conv", B=B, L=L, D=D, K=rng.randint(2, 8), dtype=dtype,
                    ragged=L > 1 and rng.random() < 0.5, bias=rng.random() < 0.5)
    D = _log(rng, 64, 8192)
    N = rng.choice([1, 4, 8, 16, 16, 16, 21, 32, 64, 128])
    L = 1 if op.endswith("token") else _log(rng, 2, 4096)
    L = max(1, min(L, 250_000_000 // (D * N)))
    B = _log(rng, 1, max(1, min(256, 250_000_000 // (L * D * N))))
    return dict(op="scan", B=B, L=L, D=D, N=N, dtype=dtype, ragged=L > 1 and rng.random() < 0.5,
                gate=rng.random() < 0.7)


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=dev)

    def ints(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device=dev)

    s = dict(case)
    op = case["op"]
    if op == "beam":
        G, W, V, dt = case["G"], case["W"], case["V"], DTYPES[case["dtype"]]
        logits = (randn(G, W, V) * 3.0).to(dt)
        # a vocabulary padded to its size and words that a user has banned
        logits[..., V - V // 50:] = float("-inf")
        logits[..., ints(0, V, 8)] = torch.finfo(dt).min
        s["logits"] = logits
        s["scores"] = -randn(G, W).abs() * 6.0
        done = torch.zeros(G * W, dtype=torch.bool, device=dev)
        done[torch.randperm(G * W, generator=g, device=dev)[:case["done"]]] = True
        s["finished"] = done.view(G, W)
        s["lengths"] = ints(1, 200, G, W).to(torch.int32)
    elif op == "reorder":
        G, W, n, D, R, w = (case[k] for k in ("G", "W", "layers", "D", "R", "win"))
        rows = G * W
        if case["kind"] == "tesm":  # fp64 state, fp32 windows of keys and of values
            bases = [randn(n, rows, D).double(), randn(n, rows, w, R), randn(n, rows, w, D)]
        else:  # fp32 state of N = 16 per channel, bf16 window of the convolution
            bases = [randn(n, rows, 8 * D, 16), randn(n, rows, 3, 8 * D).bfloat16()]
        s["bases"] = bases
        s["parents"] = ints(0, W, G, W).to(torch.int32)
        states = [b[i] for i in range(n) for b in bases]
        if own:
            from tesm_b200 import ops
            s["plan"] = ops.StateReorder(states, W)  # kept by a program for the life of its caches
    elif op == "conv":
        B, L, D, K, dt = case["B"], case["L"], case["D"], case["K"], DTYPES[case["dtype"]]
        # x is the first half of a projection's rows, the gate is the other
        s["x"] = randn(B, L, 2 * D).to(dt)[..., :D]
        s["weight"] = randn(D, K) * K ** -0.5
        s["bias"] = randn(D) * 0.1 if case["bias"] else None
        s["state"] = randn(B, K - 1, D).to(dt)
        s["lengths"] = ints(0, L + 1, B).to(torch.int32) if case["ragged"] else None
    else:
        B, L, D, N, dt = case["B"], case["L"], case["D"], case["N"], DTYPES[case["dtype"]]
        s["x"] = randn(B, L, D).to(dt)
        s["dt"] = (randn(B, L, D) * 0.5).to(dt)
        bc = randn(B, L, 2 * N).to(dt)  # slices of one projection
        s["Bm"], s["Cm"] = bc[..., :N], bc[..., N:]
        s["A"] = -(torch.arange(1, N + 1, device=dev).float().expand(D, N) * torch.exp(randn(D, N) * 0.1))
        step = torch.exp(torch.rand(D, generator=g, device=dev) * math.log(100.0) + math.log(1e-3))
        s["dt_bias"] = step + torch.log(-torch.expm1(-step))  # softplus(dt_bias) = step in [0.001, 0.1]
        s["skip"] = 1.0 + randn(D) * 0.1
        s["z"] = randn(B, L, 2 * D).to(dt)[..., D:] if case["gate"] else None
        s["state"] = randn(B, D, N) * 0.5
        s["lengths"] = ints(0, L + 1, B).to(torch.int32) if case["ragged"] else None
    return s


# ------------------------------------------------------------------ one pass
def run(s):
    op = s["op"]
    if own:
        from tesm_b200 import ops
        if op == "beam":
            r = ops.beam_select(s["logits"], s["scores"], finished=s["finished"], lengths=s["lengths"],
                                eos_token_id=EOS, pad_token_id=PAD, length_penalty=s["alpha"])
            return {"tokens": r.tokens, "parents": r.parents, "scores": r.scores, "finished": r.finished,
                    "lengths": r.lengths}
        if op == "reorder":
            s["plan"](s["parents"])
            return s["bases"]
        if op == "conv":
            y = ops.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s["lengths"])
            return {"y": y, "state": s["state"]}
        y = ops.ssm_scan(s["x"], s["dt"], s["A"], s["Bm"], s["Cm"], D=s["skip"], z=s["z"], dt_bias=s["dt_bias"],
                         state=s["state"], lengths=s["lengths"])
        return {"y": y, "state": s["state"]}
    return {"beam": _beam, "reorder": _reorder, "conv": _conv, "scan": _scan}[op](s)


def _beam(s):
    """The keys of all beams x vocabulary in 64 bits (values next to a border decide), the best W
    of them, ties to the lowest place."""
    G, W, V = s["logits"].shape
    dev = s["logits"].device
    l = s["logits"].double()
    m = l.amax(dim=-1, keepdim=True)
    logp = (l - m) - torch.log(torch.exp(l - m).sum(dim=-1, keepdim=True))
    done, length = s["finished"], s["lengths"]
    base = s["scores"].double()
    live_len = (length + (~done).int()).double()
    total = base[..., None] + logp
    only = torch.full((), float("-inf"), dtype=torch.float64, device=dev)
    ended = torch.where(torch.arange(V, device=dev) == PAD, base[..., None], only)
    total = torch.where(done[..., None], ended, total)
    key = (total / live_len.clamp(min=1)[..., None] ** s["alpha"]).view(G, W * V)
    border = torch.topk(key, W, dim=-1).values[:, -1:]
    above, equal = key > border, key == border
    take = above | (equal & (equal.int().cumsum(-1) <= W - above.int().sum(-1, keepdim=True)))
    place = torch.arange(W * V, device=dev, dtype=torch.int32).expand(G, -1)
    place = torch.where(take, place, torch.full_like(place[:1, :1], 2 ** 31 - 1))
    place = torch.topk(place, W, dim=-1, largest=False, sorted=True).values.long()
    best, order = torch.sort(key.gather(1, place), dim=-1, descending=True, stable=True)
    place = place.gather(1, order)
    score = total.view(G, W * V).gather(1, place)
    empty = ~(best > float("-inf"))  # no live candidate is left for this slot
    slot = torch.arange(W, device=dev).expand(G, W)
    parents = torch.where(empty, slot, place // V)
    tokens = torch.where(empty, torch.full_like(place, PAD), place % V)
    was = done.gather(1, parents)
    length = length.gather(1, parents) + (~was & ~empty).int()
    return {"tokens": tokens, "parents": parents.int(), "scores": torch.where(empty, only, score).float(),
            "finished": was | empty | (tokens == EOS), "lengths": length}


def _reorder(s):
    W = s["W"]
    rows = (torch.arange(s["G"], device=s["parents"].device)[:, None] * W + s["parents"]).view(-1)
    [b.copy_(b[:, rows]) for b in s["bases"]]
    return s["bases"]


def _valid(s, B, L):
    """(B, L) truth values: the positions of each sequence's tokens."""
    n = s["lengths"]
    at = torch.arange(L, device=s["x"].device)
    return at.expand(B, L) < (L if n is None else n[:, None])


def _conv(s):
    B, L, D = s["x"].shape
    K = s["K"]
    full = torch.cat([s["state"], s["x"]], dim=1)
    taps = full.unfold(1, K, 1).float()  # (B, L, D, K)
    y = (taps * s["weight"]).sum(-1)
    if s["bias"] is not None:
        y = y + s["bias"]
    y = y / (1 + torch.exp(-y))
    ok = _valid(s, B, L)
    y = torch.where(ok[..., None], y, torch.zeros((), device=y.device))
    # the last K - 1 inputs of each sequence
    at = ok.sum(-1)[:, None] + torch.arange(K - 1, device=y.device)
    s["state"].copy_(full.gather(1, at[..., None].expand(-1, -1, D)))
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


def _scan(s):
    """The recurrence by doubling: after step i every position holds the 2^i positions before it."""
    B, L, D = s["x"].shape
    x = s["x"].float()
    dt = s["dt"].float() + s["dt_bias"]
    dt = dt.clamp(min=0) + torch.log1p(torch.exp(-dt.abs()))
    ok = _valid(s, B, L)
    dt = torch.where(ok[..., None], dt, torch.zeros((), device=x.device))
    a = torch.exp(dt[..., None] * s["A"])
    h = (dt * x)[..., None] * s["Bm"].float()[:, :, None, :]
    h[:, 0] += a[:, 0] * s["state"]
    n = 1
    while n < L:
        h = torch.cat([h[:, :n], torch.addcmul(h[:, n:], a[:, n:], h[:, :-n])], dim=1)
        if 2 * n < L:
            a = torch.cat([a[:, :n], a[:, n:] * a[:, :-n]], dim=1)
        n *= 2
    y = (h * s["Cm"].float()[:, :, None, :]).sum(-1) + s["skip"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z / (1 + torch.exp(-z))
    y = torch.where(ok[..., None], y, torch.zeros((), device=y.device))
    s["state"].copy_(h[:, -1])
    return {"y": y.to(s["x"].dtype), "state": s["state"]}


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    op = case["op"]
    if op == "beam":
        G, W, V = case["G"], case["W"], case["V"]
        rows = G * W - case["done"]  # an ended beam's logits are not needed
        return {"bytes": rows * V * ESIZE[case["dtype"]] + G * W * 30, "flops": 4 * rows * V}
    if op == "reorder":
        G, W, n, D, R, w = (case[k] for k in ("G", "W", "layers", "D", "R", "win"))
        row = 8 * D + 4 * w * (R + D) if case["kind"] == "tesm" else 8 * D * 16 * 4 + 3 * 8 * D * 2
        moved = 1 - 1 / W  # random parents: the share of rows that move, and of rows that are read
        read = min(moved, 1 - (1 - 1 / W) ** W)
        return {"bytes": int(n * G * W * row * (moved + read)), "flops": 0}
    B, L, D, e = case["B"], case["L"], case["D"], ESIZE[case["dtype"]]
    tokens = B * L // 2 if case["ragged"] else B * L  # lengths are uniform in 0..L
    if op == "conv":
        K = case["K"]
        return {"bytes": (tokens + B * L) * D * e + 2 * B * (K - 1) * D * e + D * (K + 1) * 4,
                "flops": tokens * D * (2 * K + 4)}
    N = case["N"]
    vectors = 3 if case["gate"] else 2
    return {"bytes": (tokens * vectors + B * L) * D * e + tokens * 2 * N * e + 2 * B * D * N * 4 + D * N * 4,
            "flops": tokens * D * (7 * N + 12)}


# ------------------------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"beam": _exact_beam, "reorder": _exact_reorder, "conv": _exact_conv, "scan": _exact_scan}[case["op"]](s)


def _exact_reorder(s):
    parents, W = s["parents"].tolist(), s["W"]
    rows = [g * W + p for g in range(s["G"]) for p in parents[g]]
    return [torch.stack([b[:, r] for r in rows], dim=1).double() for b in s["bases"]]


def _exact_beam(s):
    G, W, V = s["logits"].shape
    scores, done, length = (s[k].cpu().numpy() for k in ("scores", "finished", "lengths"))
    out = {"tokens": np.zeros((G, W), np.int64), "parents": np.zeros((G, W), np.int32),
           "scores": np.full((G, W), -np.inf), "finished": np.ones((G, W), bool), "lengths": length.copy()}
    for g in range(G):
        logits = s["logits"][g].double().cpu().numpy()
        found = []  # (minus key, beam, token, score, length)
        for w in range(W):
            if done[g, w]:
                n = max(int(length[g, w]), 1)
                found.append((-float(scores[g, w]) / n ** s["alpha"], w, PAD, float(scores[g, w]), int(length[g, w])))
                continue
            row = logits[w]
            top = row.max()
            lse = top + math.log(np.exp(row - top).sum())
            n = int(length[g, w]) + 1
            best = np.flatnonzero(row >= np.partition(row, V - min(W, V))[V - min(W, V)])
            for v in best:
                p = float(scores[g, w]) + float(row[v]) - lse
                found.append((-p / n ** s["alpha"], w, int(v), p, n))
        found = sorted(f for f in found if f[3] > -math.inf)[:W]
        for k in range(W):
            out["parents"][g, k] = k
        for k, (_, w, v, p, n) in enumerate(found):
            out["parents"][g, k], out["tokens"][g, k], out["scores"][g, k], out["lengths"][g, k] = w, v, p, n
            out["finished"][g, k] = done[g, w] or v == EOS
        for k in range(len(found), W):
            out["lengths"][g, k] = length[g, k]
    return {k: torch.from_numpy(v) for k, v in out.items()}


def _exact_conv(s):
    B, L, D = s["x"].shape
    K = s["K"]
    x, w = s["x"].double(), s["weight"].double()
    n = [L] * B if s["lengths"] is None else s["lengths"].tolist()
    y = torch.zeros(B, L, D, dtype=torch.float64, device=x.device)
    state = s["state"].double()
    new = state.clone()
    for b in range(B):
        seq = torch.cat([state[b], x[b, :n[b]]])
        acc = torch.zeros(n[b], D, dtype=torch.float64, device=x.device)
        for j in range(K):
            acc += w[:, j] * seq[j:j + n[b]]
        if s["bias"] is not None:
            acc += s["bias"].double()
        y[b, :n[b]] = acc * torch.sigmoid(acc)
        new[b] = seq[n[b]:]
    return {"y": y, "state": new}


def _exact_scan(s):
    B, L, D = s["x"].shape
    h = s["state"].double()
    A, bias, skip = s["A"].double(), s["dt_bias"].double(), s["skip"].double()
    n = torch.full((B,), L, device=h.device) if s["lengths"] is None else s["lengths"]
    y = torch.zeros(B, L, D, dtype=torch.float64, device=h.device)
    for t in range(L):
        x, raw = s["x"][:, t].double(), s["dt"][:, t].double() + bias
        dt = torch.nn.functional.softplus(raw, threshold=1e9)
        new = torch.exp(dt[..., None] * A) * h + (dt * x)[..., None] * s["Bm"][:, t, None, :].double()
        out = (new * s["Cm"][:, t, None, :].double()).sum(-1) + skip * x
        if s["z"] is not None:
            z = s["z"][:, t].double()
            out = out * z * torch.sigmoid(z)
        on = (t < n)[:, None]
        h = torch.where(on[..., None], new, h)
        y[:, t] = torch.where(on, out, torch.zeros_like(out))
    return {"y": y, "state": h}
