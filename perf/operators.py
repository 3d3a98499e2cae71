"""The sequence-mixer operators whose speed is watched: gated linear recurrences and the gated norm behind them.

* ``delta``  the gated delta rule of the GatedDeltaNet layers: per head a state S [dk, dv] with
  S_t = e^{g_t} S_{t-1} + k_t (x) u_t, u_t = beta_t (v_t - (e^{g_t} S_{t-1})^T k_t), o_t = S_t^T q_t, where q and k are
  L2-normalised per head and q is scaled by dk^-1/2;
* ``ssd``    the scan of the Mamba2 layers: S_t = e^{dt_t A} S_{t-1} + dt_t x_t (x) B_t, y_t = S_t C_t + D x_t, with B and C
  shared by the heads of a group;
* ``norm``   the RMS norm over column groups with its SiLU gate, before it (Mamba2) or behind it (GatedDeltaNet).

Rows are packed documents.  ``mode`` is "train" (forward, then backward from a given output gradient; gradients of every
input are returned), "score" (forward alone) or "carry" (forward from given states, final states returned: what a rank
of a sharded sequence runs on its piece, down to documents of one token).
"""
import math
import random

import torch

own = False

CHUNK = 64
EPS = 1e-6
BF = torch.bfloat16


def _delta(name, mode, tokens, docs, hk, hv, dk, dv):
    return dict(name=name, op="delta", mode=mode, tokens=tokens, docs=docs, hk=hk, hv=hv, dk=dk, dv=dv)


def _ssd(name, mode, tokens, docs, groups, heads, state, dim):
    return dict(name=name, op="ssd", mode=mode, tokens=tokens, docs=docs, hk=groups, hv=heads, dk=state, dv=dim)


def _norm(name, mode, tokens, width, group, norm_first):
    return dict(name=name, op="norm", mode=mode, tokens=tokens, width=width, group=group, norm_first=norm_first)


def listed():
    return [
        # the toy hybrid that tests and smoke runs train: heads of 8, a batch of three short documents
        _delta("delta_small_train", "train", 130, 3, 2, 4, 8, 8),
        # a training row of a hybrid layer: 16 key heads shared by 32 value heads, packed documents
        _delta("delta_train_4096", "train", 4096, 5, 16, 32, 128, 128),
        # log-probabilities of one long document
        _delta("delta_score_16384", "score", 16384, 1, 16, 32, 128, 128),
        # pieces of 48 documents of a few tokens each, with their states carried in and out
        _delta("delta_carry_48", "carry", 101, 48, 16, 32, 128, 128),
        # the toy state-space hybrid
        _ssd("ssd_small_train", "train", 130, 3, 2, 8, 16, 16),
        # a training row of a state-space layer: 128 heads of 64, 8 groups of 128 states, an odd length
        _ssd("ssd_train_4095", "train", 4095, 5, 8, 128, 128, 64),
        # one long document without gradients
        _ssd("ssd_score_16384", "score", 16384, 1, 8, 128, 128, 64),
        # a few documents' pieces with their states, a smaller layer
        _ssd("ssd_carry_777", "carry", 777, 6, 4, 64, 64, 64),
        # the norm of a small layer on a short row
        _norm("norm_gate_small", "train", 130, 256, 128, False),
        # per-head norm, then the gate: 32 value heads of 128
        _norm("norm_then_gate_4096", "train", 4096, 4096, 128, True),
        # gate, then groups of 1024: the 8192-wide state-space layer
        _norm("gate_then_norm_4095", "train", 4095, 8192, 1024, False),
        # the same without gradients on a long row
        _norm("gate_then_norm_score", "score", 16384, 8192, 1024, False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["delta", "ssd", "norm"])
    if op == "norm":
        group = rng.choice([64, 128, 256, 512, 1024])
        groups = _log(rng, 1, 8192 // group)
        return _norm("", rng.choice(["train", "score"]), _log(rng, 1, 4096), group * groups, group, rng.random() < 0.5)
    mode = rng.choice(["train", "score", "carry"])
    tokens = _log(rng, 1, 4096)
    docs = min(tokens, _log(rng, 1, 48))
    if op == "delta":
        hk = rng.choice([1, 2, 4, 8, 16])
        c = _delta("", mode, tokens, docs, hk, hk * rng.choice([1, 2]), rng.choice([64, 96, 128]), rng.choice([64, 128]))
    else:
        hk = rng.choice([1, 2, 4, 8])
        c = _ssd("", mode, tokens, docs, hk, hk * rng.choice([4, 8, 16]), rng.choice([16, 64, 128]), rng.choice([32, 64, 80]))
    return c


def _cuts(case, seed):
    """Document boundaries: ``docs`` documents of uneven lengths that fill the row."""
    r = random.Random(seed)
    T, n = case["tokens"], case["docs"]
    return [0] + sorted(r.sample(range(1, T), n - 1)) + [T]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))

    def rand(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def uniform(n):
        return torch.rand(n, generator=gen, device="cuda")

    T = case["tokens"]
    s = {"case": case}
    if case["op"] == "norm":
        W = case["width"]
        s["x"] = rand(T, W).to(BF)
        # the gate is a column slice of a wider projection where it comes first in the row's layout
        s["gate"] = rand(T, W).to(BF) if case["norm_first"] else rand(T, W + 64).to(BF)[:, :W]
        s["weight"] = (1 + 0.1 * rand(case["group"] if case["norm_first"] else W)).to(BF)
        s["dy"] = rand(T, W).to(BF)
        return s
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    s["cu"] = torch.tensor(_cuts(case, seed), dtype=torch.int32, device="cuda")
    silu = torch.nn.functional.silu
    softplus = torch.nn.functional.softplus
    # time steps log-uniform in [1e-3, 0.1] before the input moves them, as the models initialise them
    step = torch.exp(uniform(hv) * math.log(100.0) + math.log(1e-3))
    bias = step + torch.log(-torch.expm1(-step))
    dt = softplus(0.5 * rand(T, hv) + bias)
    if case["op"] == "delta":
        s["q"], s["k"] = silu(rand(T, hk, dk)).to(BF), silu(rand(T, hk, dk)).to(BF)
        s["v"] = silu(rand(T, hv, dv)).to(BF)
        s["g"] = -(1 + 15 * uniform(hv)) * dt
        s["beta"] = torch.sigmoid(rand(T, hv))
        shape = (case["docs"], hv, dk, dv)
    else:
        # x, B and C are column slices of one convolution's output
        row = silu(rand(T, hv * dv + 2 * hk * dk)).to(BF)
        s["x"] = row[:, :hv * dv].unflatten(1, (hv, dv))
        s["B"] = row[:, hv * dv:hv * dv + hk * dk].unflatten(1, (hk, dk))
        s["C"] = row[:, hv * dv + hk * dk:].unflatten(1, (hk, dk))
        s["dt"] = dt
        s["A"] = -torch.arange(1, hv + 1, dtype=torch.float32, device="cuda")
        s["D"] = 1 + 0.1 * rand(hv)
        shape = (case["docs"], hv, dv, dk)
    if case["mode"] == "carry":
        s["state"] = 0.1 * rand(*shape)
    if case["mode"] == "train":
        s["dy"] = rand(T, hv, dv).to(BF)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------
def _chunk_table(cu):
    """[docs, chunks, CHUNK] token indices (each document cut into chunks) and which of them are tokens."""
    start, end = cu[:-1].long(), cu[1:].long()
    n = int(torch.div(end - start + CHUNK - 1, CHUNK, rounding_mode="floor").max().clamp_min(1))
    idx = start.view(-1, 1, 1) + torch.arange(n * CHUNK, device=cu.device).view(1, n, CHUNK)
    ok = idx < end.view(-1, 1, 1)
    return torch.where(ok, idx, 0), ok


def _chunks(x, idx, ok):
    """[T, H, d] -> [docs, H, chunks, CHUNK, d] in fp32, zeros where there is no token."""
    return (x.float()[idx] * ok[..., None, None]).permute(0, 3, 1, 2, 4)


def _unchunk(o, idx, ok, T):
    """Back to [T, H, d]."""
    flat = o.permute(0, 2, 3, 1, 4)[ok]
    return torch.zeros(T, *flat.shape[1:], device=o.device).index_put((idx[ok],), flat)


def _decays(g, idx, ok):
    """Inclusive sums of the log decay within each chunk, and exp(G_i - G_j) for j <= i."""
    G = _chunks(g.unsqueeze(-1), idx, ok)[..., 0].double().cumsum(-1)
    tri = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=g.device).tril()
    return G, torch.exp((G.unsqueeze(-1) - G.unsqueeze(-2)).masked_fill(~tri, -math.inf).float())


def _plain_delta(q, k, v, g, beta, cu, state):
    T, hk, dk = q.shape
    rep = v.shape[1] // hk
    qf, kf = q.float(), k.float()
    qn = (qf / qf.pow(2).sum(-1, keepdim=True).sqrt().clamp_min(1e-12) * dk ** -0.5).repeat_interleave(rep, 1)
    kn = (kf / kf.pow(2).sum(-1, keepdim=True).sqrt().clamp_min(1e-12)).repeat_interleave(rep, 1)
    idx, ok = _chunk_table(cu)
    Q, K, V = _chunks(qn, idx, ok), _chunks(kn, idx, ok), _chunks(v, idx, ok)
    b = _chunks(beta.unsqueeze(-1), idx, ok)
    G, D = _decays(g, idx, ok)
    gamma, last = torch.exp(G.float()).unsqueeze(-1), torch.exp((G[..., -1:] - G).float()).unsqueeze(-1)
    M = torch.eye(CHUNK, device=q.device) + (b * D * (K @ K.transpose(-1, -2))).tril(-1)
    sol = torch.linalg.solve_triangular(M, torch.cat([b * V, b * gamma * K], -1), upper=False, unitriangular=True)
    U0, W = sol[..., :v.shape[2]], sol[..., v.shape[2]:]
    P = D * (Q @ K.transpose(-1, -2))
    S = torch.zeros(len(cu) - 1, v.shape[1], dk, v.shape[2], device=q.device) if state is None else state
    out = []
    for n in range(idx.shape[1]):                                    # the state goes from chunk to chunk
        U = U0[:, :, n] - W[:, :, n] @ S
        out.append(gamma[:, :, n] * (Q[:, :, n] @ S) + P[:, :, n] @ U)
        S = gamma[:, :, n, -1:] * S + (last[:, :, n] * K[:, :, n]).transpose(-1, -2) @ U
    return _unchunk(torch.stack(out, 2), idx, ok, T), S


def _plain_ssd(x, dt, A, B, C, D, cu, state):
    T, H, P = x.shape
    rep = H // B.shape[1]
    idx, ok = _chunk_table(cu)
    X, Bh, Ch = _chunks(x, idx, ok), _chunks(B, idx, ok).repeat_interleave(rep, 1), _chunks(C, idx, ok).repeat_interleave(rep, 1)
    U = _chunks(dt.unsqueeze(-1), idx, ok) * X
    G, L = _decays(dt * A, idx, ok)
    last = torch.exp((G[..., -1:] - G).float()).unsqueeze(-1)
    y = (L * (Ch @ Bh.transpose(-1, -2))) @ U
    S = (last * Bh).transpose(-1, -2) @ U                             # what each chunk adds: [docs, H, n, N, P]
    E = torch.nn.functional.pad(G[..., -1], (1, 0)).cumsum(-1)        # log decay up to each chunk's start
    n = idx.shape[1]
    tri = torch.ones(n + 1, n, dtype=torch.bool, device=x.device).tril(-1)
    between = torch.exp((E.unsqueeze(-1) - E[..., 1:].unsqueeze(-2)).masked_fill(~tri, -math.inf).float())
    S = (between @ S.flatten(-2)).unflatten(-1, S.shape[-2:])         # [docs, H, n + 1, N, P]
    if state is not None:
        S = S + torch.exp(E.float())[..., None, None] * state.transpose(-1, -2).unsqueeze(2)
    y = y + torch.exp(G.float()).unsqueeze(-1) * (Ch @ S[:, :, :-1])
    y = y + D.view(1, -1, 1, 1, 1) * X
    return _unchunk(y, idx, ok, T), S[:, :, -1].transpose(-1, -2)


def _plain_norm(x, gate, weight, group, norm_first):
    g = gate.float() * torch.sigmoid(gate.float())
    h = x.float() if norm_first else x.float() * g
    h = h.unflatten(-1, (-1, group))
    h = h * torch.rsqrt(h.pow(2).mean(-1, keepdim=True) + EPS)
    h = h * weight.float().view(-1, group)
    h = h.flatten(-2)
    return h * g if norm_first else h


def _plain(s, names, fn):
    """Runs ``fn`` on fp32 copies of the named inputs; returns its outputs and, in training, the inputs' gradients."""
    train = s["case"]["mode"] == "train"
    leaves = [s[n].float().requires_grad_(train) if n in s else None for n in names]
    with torch.set_grad_enabled(train):
        y, state = fn(*leaves)
    out = {"y": y.detach().to(BF)}
    if train:
        given = [(n, v) for n, v in zip(names, leaves) if v is not None]
        grads = torch.autograd.grad(y, [v for _, v in given], s["dy"].float())
        out.update({"d" + n: d.to(s[n].dtype) for (n, _), d in zip(given, grads)})
    if s["case"]["mode"] == "carry":
        out["state"] = state
    return out


# ---- the framework's calls -----------------------------------------------------------------------------------
def _own(s, names, fn):
    train = s["case"]["mode"] == "train"
    leaves = [s[n].detach().requires_grad_(train) if n in s else None for n in names]
    with torch.set_grad_enabled(train):
        y = fn(*leaves)
    out = {}
    if s["case"]["mode"] == "carry":
        y, out["state"] = y
    out["y"] = y.detach()
    if train:
        given = [(n, v) for n, v in zip(names, leaves) if v is not None]
        grads = torch.autograd.grad(y, [v for _, v in given], s["dy"])
        out.update({"d" + n: d for (n, _), d in zip(given, grads)})
    return out


def run(s):
    c = s["case"]
    if c["op"] == "norm":
        names = ("x", "gate", "weight")
        if own:
            from xorl_b200.ops.norm import gated_rms_norm
            return _own(s, names, lambda x, z, w: gated_rms_norm(x, z, w, c["group"], EPS, norm_first=c["norm_first"]))
        return _plain(s, names, lambda x, z, w: (_plain_norm(x, z, w, c["group"], c["norm_first"]), None))
    if c["op"] == "delta":
        names = ("q", "k", "v", "g", "beta", "state")
        if own:
            from xorl_b200.ops.recurrence import gated_delta_rule
            return _own(s, names, lambda q, k, v, g, b, S: gated_delta_rule(
                q, k, v, g, b, s["cu"], scale=c["dk"] ** -0.5, qk_l2norm=True, initial_state=S,
                return_final_state=c["mode"] == "carry"))
        return _plain(s, names, lambda q, k, v, g, b, S: _plain_delta(q, k, v, g, b, s["cu"], S))
    names = ("x", "dt", "A", "B", "C", "D", "state")
    if own:
        from xorl_b200.ops.recurrence import ssd_scan
        return _own(s, names, lambda x, dt, A, B, C, D, S: ssd_scan(
            x, dt, A, B, C, D, s["cu"], initial_state=S, return_final_state=c["mode"] == "carry"))
    return _plain(s, names, lambda x, dt, A, B, C, D, S: _plain_ssd(x, dt, A, B, C, D, s["cu"], S))


def work(case):
    """Each input read once and each output written once per direction (the backward pass reads the inputs again: nothing
    says that they are still on the chip); the products of the token-by-token recurrence."""
    T, train = case["tokens"], case["mode"] == "train"
    if case["op"] == "norm":
        row = T * case["width"] * 2
        return {"bytes": row * (3 + (5 if train else 0)), "flops": T * case["width"] * (30 if train else 10)}
    hk, hv, dk, dv = case["hk"], case["hv"], case["dk"], case["dv"]
    narrow = T * hv * 4 * (2 if case["op"] == "delta" else 1)
    inputs = T * (2 * hk * dk + hv * dv) * 2 + narrow
    b = inputs + T * hv * dv * 2
    cell = T * hv * dk * dv
    f = (6 if case["op"] == "delta" else 4) * cell
    if case["mode"] == "carry":
        b += 2 * case["docs"] * hv * dk * dv * 4
    if train:
        b += 2 * inputs + T * hv * dv * 2
        f += (14 if case["op"] == "delta" else 10) * cell
    return {"bytes": b, "flops": f}


# ---- the definitions in 64 bits, token by token ----------------------------------------------------------------
def _exact_recurrence(delta, q, k, v, decay, b, cuts, state, dy):
    """q, k [T, H, dk], v [T, H, dv], decay, b [T, H], all fp64 and with heads spread; returns y, the final states
    [docs, H, dk, dv] and, given dy, the gradients of q, k, v, log decay and b by the adjoint recurrence."""
    T, H, dk = q.shape
    dv = v.shape[2]
    y = torch.zeros(T, H, dv, dtype=torch.float64, device=q.device)
    a = torch.exp(decay)
    finals, kept = [], {}
    every = 64

    def step(S, t):
        S = a[t].view(H, 1, 1) * S
        r = v[t] - torch.einsum("hkv,hk->hv", S, k[t]) if delta else v[t]
        return torch.baddbmm(S, k[t].unsqueeze(-1), (b[t].unsqueeze(-1) * r).unsqueeze(1)), S, r

    for d in range(len(cuts) - 1):
        S = torch.zeros(H, dk, dv, dtype=torch.float64, device=q.device) if state is None else state[d]
        for t in range(cuts[d], cuts[d + 1]):
            if dy is not None and (t - cuts[d]) % every == 0:
                kept[t] = S
            S, _, _ = step(S, t)
            y[t] = torch.einsum("hkv,hk->hv", S, q[t])
        finals.append(S)
    finals = torch.stack(finals)
    if dy is None:
        return y, finals, None
    dq, dk_, dv_ = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    dg, db = torch.zeros_like(decay), torch.zeros_like(b)
    for d in range(len(cuts) - 1):
        dS = torch.zeros(H, dk, dv, dtype=torch.float64, device=q.device)
        for c0 in reversed(range(cuts[d], cuts[d + 1], every)):
            S, steps = kept[c0], []
            for t in range(c0, min(c0 + every, cuts[d + 1])):
                S, before, r = step(S, t)
                steps.append((t, S, before, r))
            for t, after, before, r in reversed(steps):
                dq[t] = torch.einsum("hkv,hv->hk", after, dy[t])
                dS = torch.baddbmm(dS, q[t].unsqueeze(-1), dy[t].unsqueeze(1))
                du = torch.einsum("hkv,hk->hv", dS, k[t])
                dk_[t] = torch.einsum("hkv,hv->hk", dS, b[t].unsqueeze(-1) * r)
                db[t] = (du * r).sum(-1)
                dr = b[t].unsqueeze(-1) * du
                dv_[t] = dr
                if delta:                                             # r = v - before^T k
                    dk_[t] -= torch.einsum("hkv,hv->hk", before, dr)
                    dS = torch.baddbmm(dS, k[t].unsqueeze(-1), dr.unsqueeze(1), alpha=-1)
                dg[t] = (dS * before).sum((-1, -2))
                dS = a[t].view(H, 1, 1) * dS
    return y, finals, (dq, dk_, dv_, dg, db)


def _shared(d, heads):
    """Gradients of heads that are read by several: the sum over their readers."""
    return d.unflatten(1, (heads, -1)).sum(2)


def exact(case, seed):
    s = prepare(case, seed)
    train = case["mode"] == "train"
    f = {n: v.double() for n, v in s.items() if torch.is_tensor(v)}
    if case["op"] == "norm":
        n, T = case["group"], case["tokens"]
        x, z, dy = (f[m].reshape(T, -1, n) for m in ("x", "gate", "dy"))
        w = f["weight"].reshape(1, -1, n)
        sg = 1 / (1 + torch.exp(-z))
        act, slope = z * sg, sg * (1 + z * (1 - sg))
        h = x if case["norm_first"] else x * act
        r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS)
        y = h * r * w * (act if case["norm_first"] else 1)
        out = {"y": y.reshape(T, -1)}
        if train:
            dn = dy * w * (act if case["norm_first"] else 1)            # gradient of h * r
            dh = r * dn - h * r ** 3 * (dn * h).mean(-1, keepdim=True)
            out["dx"] = dh if case["norm_first"] else dh * act
            out["dgate"] = (dy * h * r * w if case["norm_first"] else dh * x) * slope
            dw = dy * h * r * (act if case["norm_first"] else 1)
            out["dweight"] = dw.sum((0, 1)) if case["norm_first"] else dw.sum(0).reshape(-1)
            out["dx"], out["dgate"] = out["dx"].reshape(T, -1), out["dgate"].reshape(T, -1)
        return out
    cuts = _cuts(case, seed)
    hk, rep, dk = case["hk"], case["hv"] // case["hk"], case["dk"]
    spread = lambda t: t.repeat_interleave(rep, 1)  # noqa: E731
    if case["op"] == "delta":
        nq, nk = (torch.linalg.vector_norm(f[m], dim=-1, keepdim=True).clamp_min(1e-12) for m in "qk")
        qn, kn = f["q"] / nq, f["k"] / nk
        y, S, grads = _exact_recurrence(True, spread(qn * dk ** -0.5), spread(kn), f["v"], f["g"], f["beta"], cuts,
                                        f.get("state"), f.get("dy") if train else None)
        out = {"y": y}
        if train:
            dq, dkk, dv, dg, db = grads
            dq, dkk = _shared(dq, hk) * dk ** -0.5, _shared(dkk, hk)
            out["dq"] = (dq - qn * (qn * dq).sum(-1, keepdim=True)) / nq
            out["dk"] = (dkk - kn * (kn * dkk).sum(-1, keepdim=True)) / nk
            out["dv"], out["dg"], out["dbeta"] = dv, dg, db
    else:
        y, S, grads = _exact_recurrence(False, spread(f["C"]), spread(f["B"]), f["x"], f["dt"] * f["A"], f["dt"], cuts,
                                        None if "state" not in f else f["state"].transpose(-1, -2),
                                        f.get("dy") if train else None)
        out = {"y": y + f["D"].view(1, -1, 1) * f["x"]}
        S = S.transpose(-1, -2)
        if train:
            dC, dB, dx, dg, ddt = grads
            out["dx"] = dx + f["D"].view(1, -1, 1) * f["dy"]
            out["ddt"], out["dA"] = ddt + dg * f["A"], (dg * f["dt"]).sum(0)
            out["dB"], out["dC"] = _shared(dB, hk), _shared(dC, hk)
            out["dD"] = (f["dy"] * f["x"]).sum((0, 2))
    if case["mode"] == "carry":
        out["state"] = S
    return out
