"""Operators of recurrent language models, in their plain form and through the framework.

Three operators, measured by call: the gated delta rule (a matrix state per head
with decay and an error-correcting write: training, prompts, single tokens),
layer norm (forward and backward) and the choice of the next token
(temperature, top-k, top-p and min-p from given random numbers). ``run`` computes
them with elementary torch operations, or, where ``own`` is true, through
``sunnynet_amd.runtime``. ``exact`` restates each one in 64 bits from its
definition. Sizes are those of this repository's configurations (12 heads of 64,
widths 1024, 1536 and 200, vocabularies 12000, 32000 and 65536) or generic ones.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False              # True: the framework's kernels
DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CHUNK = 64               # tokens per chunk of the plain delta rule


def listed():
    return [
        # One user's next token on the 12 x 64-head model: launch and latency.
        {"name": "delta_step_b1", "kind": "delta_step", "dtype": "fp32", "B": 1, "Hk": 12, "H": 12, "K": 64,
         "V": 64},
        # A serving batch's next tokens, query and key heads shared by two value heads.
        {"name": "delta_step_b64", "kind": "delta_step", "dtype": "bf16", "B": 64, "Hk": 8, "H": 16, "K": 128,
         "V": 128},
        # Prompts of many lengths packed end to end, from a kept state.
        {"name": "delta_prompts_packed", "kind": "delta_packed", "dtype": "bf16", "N": 13, "T": 6007, "Hk": 12,
         "H": 12, "K": 64, "V": 64},
        # One long document.
        {"name": "delta_prompt_long", "kind": "delta_fwd", "dtype": "fp16", "B": 1, "T": 16384, "Hk": 8, "H": 16,
         "K": 128, "V": 128},
        # A training batch: forward and every gradient.
        {"name": "delta_train_b8", "kind": "delta_train", "dtype": "bf16", "B": 8, "T": 2048, "Hk": 8, "H": 16,
         "K": 128, "V": 128},
        # A small training batch that no tile divides, at full precision.
        {"name": "delta_train_ragged", "kind": "delta_train", "dtype": "fp32", "B": 3, "T": 333, "Hk": 5, "H": 5,
         "K": 40, "V": 72},
        # Training through a norm at the 100M model's width.
        {"name": "norm_train_b16", "kind": "norm_train", "dtype": "bf16", "rows": 32768, "D": 1024},
        # The same on an odd number of narrow rows at full precision.
        {"name": "norm_train_ragged", "kind": "norm_train", "dtype": "fp32", "rows": 2331, "D": 200},
        # A serving batch's norm at the inner width.
        {"name": "norm_rows_b64", "kind": "norm_fwd", "dtype": "fp16", "rows": 64, "D": 1536},
        # One user's token with the command line's default settings.
        {"name": "sample_b1", "kind": "sample", "dtype": "fp32", "B": 1, "V": 65536, "mix": "cli"},
        # A serving batch whose requests ask for different settings.
        {"name": "sample_b64", "kind": "sample", "dtype": "fp32", "B": 64, "V": 32000, "mix": "each"},
        # Many samples at once from 16-bit logits: nucleus and min-p.
        {"name": "sample_b512", "kind": "sample", "dtype": "bf16", "B": 512, "V": 12000, "mix": "nucleus"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta_step", "delta_packed", "delta_fwd", "delta_train", "delta_train", "norm_train",
                       "norm_fwd", "sample", "sample"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if kind.startswith("delta"):
        Hk = _log(rng, 1, 12)
        H = Hk * rng.choice([1, 1, 2, 3])
        K, V = rng.choice([(64, 64), (128, 128), (128, 64), (_log(rng, 8, 128), _log(rng, 8, 192))])
        c = {"kind": kind, "dtype": dtype, "Hk": Hk, "H": H, "K": K, "V": V}
        if kind == "delta_step":
            return dict(c, B=min(_log(rng, 1, 256), max(1, (64 * 16 * 128 * 128) // (H * K * V))))
        # at most the listed training batch's work (the long document's where only forward)
        most = (8 * 2048 if kind == "delta_train" else 16384) * 16 * 128 * 128 // (H * K * V)
        if kind == "delta_packed":
            return dict(c, N=rng.randint(1, 24), T=min(_log(rng, 32, 8192), most))
        B = _log(rng, 1, 8)
        return dict(c, B=B, T=max(1, min(_log(rng, 1, 2048 if kind == "delta_train" else 8192), most // B)))
    if kind.startswith("norm"):
        D = rng.choice([_log(rng, 24, 6000), 64 * _log(rng, 2, 96)])
        most = 32768 * 1024 // D
        return {"kind": kind, "dtype": dtype, "D": D, "rows": min(_log(rng, 1, 65536), most)}
    V = rng.choice([_log(rng, 100, 150000), 12000, 32000, 65536])
    return {"kind": kind, "dtype": dtype, "B": min(_log(rng, 1, 512), 512 * 12000 // V), "V": V,
            "mix": rng.choice(["cli", "each", "nucleus", "plain"])}


# ---- inputs ------------------------------------------------------------------
def _split(rng, total, n):
    """n lengths of at least one token that sum to total."""
    n = min(n, total)
    cuts = sorted(rng.choice(np.arange(1, total), n - 1, replace=False).tolist()) if n > 1 else []
    edges = [0] + cuts + [total]
    return [b - a for a, b in zip(edges, edges[1:])]


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    kind = case["kind"]
    st = {"case": case}
    if kind.startswith("delta"):
        Hk, H, K, V = (case[n] for n in ("Hk", "H", "K", "V"))
        B, T = (1, case["T"]) if kind == "delta_packed" else (case["B"], case.get("T", 1))
        N = B
        if kind == "delta_packed":
            st["lens"] = _split(np.random.default_rng(seed), T, case["N"])
            N = len(st["lens"])
            edges = np.concatenate([[0], np.cumsum(st["lens"])])
            st["cu"] = torch.tensor(edges, dtype=torch.int32, device=DEV)
        lead = (B,) if kind == "delta_step" else (B, T)
        # queries and keys of unit length, as such layers normalise them; decays from
        # nearly none to strong ones, writes from weak to full
        for n, h, d in (("q", Hk, K), ("k", Hk, K)):
            x = rn(*lead, h, d)
            st[n] = (x / x.square().sum(-1, keepdim=True).sqrt()).to(dt)
        st["v"] = rn(*lead, H, V).to(dt)
        st["g"] = -torch.exp(1.5 * rn(*lead, H) - 3.0)
        st["beta"] = torch.sigmoid(rn(*lead, H))
        st["s0"] = 0.2 * rn(N, H, K, V)
        if kind == "delta_train":
            st["dout"] = rn(B, T, H, V).to(dt)
            st["dsend"] = rn(N, H, K, V)
            for n in ("q", "k", "v", "g", "beta", "s0"):
                st[n].requires_grad_()
    elif kind.startswith("norm"):
        R, D = case["rows"], case["D"]
        st["x"] = (rn(R, D) * (0.5 + torch.rand(R, 1, generator=g, device=DEV)) + 0.3 * rn(R, 1)).to(dt)
        st["w"] = 1.0 + 0.1 * rn(D)
        st["b"] = 0.1 * rn(D)
        st["eps"] = 4.1e-4
        if kind == "norm_train":
            st["dy"] = rn(R, D).to(dt)
            for n in ("x", "w", "b"):
                st[n].requires_grad_()
    else:
        B, V = case["B"], case["V"]
        st["logits"] = (2.5 * rn(B, V)).to(dt)
        f64 = dict(generator=g, device=DEV, dtype=torch.float64)
        st["u"] = torch.rand(B, **f64)
        if case["mix"] == "each":        # requests of a scheduler: one row's settings each
            pick = torch.rand(4, B, **f64)
            st["temperature"] = torch.where(pick[0] < 0.2, 0.0, 0.5 + pick[0])
            st["top_k"] = torch.where(pick[1] < 0.5, 0, 1 + (200 * pick[1]).long()).int()
            st["top_p"] = torch.where(pick[2] < 0.3, 1.0, 0.7 + 0.3 * pick[2])
            st["min_p"] = torch.where(pick[3] < 0.6, 0.0, 0.1 * pick[3])
        else:
            st["temperature"], st["top_k"], st["top_p"], st["min_p"] = {
                "cli": (0.8, 40, 0.95, 0.0), "nucleus": (0.9, 0, 0.9, 0.02), "plain": (1.0, 0, 1.0, 0.0)}[case["mix"]]
    return st


# ---- the plain forms -----------------------------------------------------------
def _plain_delta(q, k, v, g, beta, s0):
    """q, k (B,T,Hk,K), v (B,T,H,V), g, beta (B,T,H), s0 (B,H,K,V) -> out, send.

    Chunks of 64 tokens: with c the running sum of g in a chunk, the writes u solve
    (I + A) u = beta (v - e^c K S), A_ij = beta_i e^(c_i - c_j) k_i.k_j for j < i. The
    inverse of a unit lower triangular matrix is a finite product of its powers."""
    B, T, Hk, K = q.shape
    H, V = v.shape[2:]
    dt, pad, scale = v.dtype, -T % CHUNK, K ** -0.5
    n = (T + pad) // CHUNK

    def chunks(x, rep):      # (B,T,h,...) -> (n,B,H,CHUNK,...)
        x = x.float().repeat_interleave(rep, dim=2)
        x = torch.cat([x, x.new_zeros(B, pad, *x.shape[2:])], 1)
        x = x.reshape(B, n, CHUNK, H, *x.shape[3:])
        return x.movedim(1, 0).movedim(3, 2).contiguous()

    q, k = chunks(q, H // Hk) * scale, chunks(k, H // Hk)
    v, g, beta = chunks(v, 1), chunks(g, 1), chunks(beta, 1)[..., None]
    c = g.double().cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    D = (c[..., :, None] - c[..., None, :]).masked_fill(~low, -math.inf).exp()
    kt = k.transpose(-1, -2).contiguous()
    P = (q @ kt) * D.float()
    A = -(beta * (k @ kt)).double() * D.tril(-1)
    eye = torch.eye(CHUNK, dtype=torch.float64, device=q.device)
    M = eye + A
    for _ in range(5):       # (I - X)^-1 = (I + X)(I + X^2)(I + X^4) ... for nilpotent X
        A = A @ A
        M = M @ (eye + A)
    M = M.float()
    ec, ee = c.exp().float()[..., None], (c[..., -1:] - c).exp().float()[..., None]
    qe, ke, kl = q * ec, k * ec, (k * ee).transpose(-1, -2).contiguous()
    last = ec[..., -1:, :]
    S, outs = s0.float(), []
    for i in range(n):
        u = M[i] @ (beta[i] * (v[i] - ke[i] @ S))
        outs.append(qe[i] @ S + P[i] @ u)
        S = last[i] * S + kl[i] @ u
    out = torch.stack(outs).movedim(2, 3).movedim(0, 1).reshape(B, n * CHUNK, H, V)[:, :T]
    return out.to(dt), S


def _plain_step(q, k, v, g, beta, s0):
    rep = v.shape[1] // q.shape[1]
    q, k = (x.float().repeat_interleave(rep, dim=1) for x in (q, k))
    S = s0 * g.exp()[..., None, None]
    u = beta[..., None] * (v.float() - (S * k[..., None]).sum(-2))
    S = S + k[..., None] * u[..., None, :]
    return (q.shape[-1] ** -0.5 * (S * q[..., None]).sum(-2)).to(v.dtype), S


def _plain_packed(st):
    """The packed prompts side by side, each padded with tokens that change nothing."""
    lens = torch.tensor(st["lens"], device=DEV)
    most, first = max(st["lens"]), lens.cumsum(0) - lens
    t = torch.arange(most, device=DEV)
    live = t < lens[:, None]
    at = torch.where(live, first[:, None] + t, 0)
    wide = [st[n][0][at] * live.reshape(*live.shape, *[1] * (st[n].dim() - 2)) for n in ("q", "k", "v", "g", "beta")]
    out, send = _plain_delta(*wide, st["s0"])
    return out[live][None], send


def _plain_norm(x, w, b, eps):
    f = x.float()
    d = f - f.mean(-1, keepdim=True)
    r = (d.square().mean(-1, keepdim=True) + eps).rsqrt()
    return (d * r * w + b).to(x.dtype)


def _plain_sample(logits, u, temperature, top_k, top_p, min_p):
    """In 64 bits: a token's share may be smaller than a 32-bit sum's rounding."""
    B, V = logits.shape
    x = logits.double()
    col = {n: torch.as_tensor(v, device=DEV).double().expand(B)[:, None] for n, v in
           (("t", temperature), ("k", top_k), ("p", top_p), ("m", min_p))}
    z = x / torch.where(col["t"] > 0, col["t"], 1.0)
    z = z - z.amax(1, keepdim=True)
    zs, order = torch.sort(z, dim=1, descending=True, stable=True)
    kth = zs.gather(1, (col["k"].long() - 1).clamp(0, V - 1))
    kth = torch.where((col["k"] > 0) & (col["k"] < V), kth, -math.inf)
    ws = torch.where(zs >= kth, zs.exp(), 0.0)
    before = ws.cumsum(1) - ws
    cut = (before > col["p"] * ws.sum(1, keepdim=True)) & (col["p"] > 0) & (col["p"] < 1)
    ws = torch.where(cut | (ws < col["m"]), 0.0, ws)
    w = torch.zeros_like(ws).scatter_(1, order, ws)
    cdf = w.cumsum(1)
    pick = (cdf <= u[:, None] * cdf[:, -1:]).sum(1).clamp(max=V - 1)
    return torch.where(col["t"][:, 0] > 0, pick, x.argmax(1)).int()


def run(st):
    case, kind = st["case"], st["case"]["kind"]
    if own:
        from sunnynet_amd import runtime
    if kind == "delta_step":
        if own:
            send = torch.empty_like(st["s0"])      # s0 stays for the next pass
            out = runtime.delta_step(st["q"], st["k"], st["v"], st["g"], st["beta"], st["s0"], send=send)
            return out, send
        return _plain_step(*(st[n] for n in ("q", "k", "v", "g", "beta", "s0")))
    if kind == "delta_packed":
        if own:
            return runtime.gated_delta(*(st[n] for n in ("q", "k", "v", "g", "beta", "s0")), cu_seqlens=st["cu"])
        return _plain_packed(st)
    if kind.startswith("delta"):
        names = ("q", "k", "v", "g", "beta", "s0")
        out, send = (runtime.gated_delta if own else _plain_delta)(*(st[n] for n in names))
        if kind == "delta_fwd":
            return out, send
        grads = torch.autograd.grad((out, send), [st[n] for n in names], (st["dout"], st["dsend"]))
        return out.detach(), send.detach(), *grads
    if kind.startswith("norm"):
        y = (runtime.layer_norm if own else _plain_norm)(st["x"], st["w"], st["b"], st["eps"])
        if kind == "norm_fwd":
            return y
        return y.detach(), *torch.autograd.grad(y, [st["x"], st["w"], st["b"]], st["dy"])
    return (runtime.sample_tokens if own else _plain_sample)(
        st["logits"], st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])


# ---- what each cannot do without -------------------------------------------------
def work(case):
    kind, e = case["kind"], 4 if case["dtype"] == "fp32" else 2
    if kind.startswith("delta"):
        Hk, H, K, V = (case[n] for n in ("Hk", "H", "K", "V"))
        N = case.get("N", case.get("B"))
        tokens = case["T"] if kind == "delta_packed" else case["B"] * case.get("T", 1)
        inputs = tokens * (2 * Hk * K * e + H * V * e + 8 * H)
        state = 8 * N * H * K * V
        # per token and head: decay, read at k, write, read at q
        flops = tokens * H * 7 * K * V
        if kind != "delta_train":
            return {"bytes": inputs + tokens * H * V * e + state, "flops": flops}
        # out and send written, dout and dsend read, gradients of every input written
        return {"bytes": 2 * inputs + 2 * tokens * H * V * e + 2 * state, "flops": 3 * flops}
    if kind.startswith("norm"):
        n, D = case["rows"] * case["D"], case["D"]
        if kind == "norm_fwd":
            return {"bytes": 2 * n * e + 8 * D, "flops": 8 * n}
        return {"bytes": 4 * n * e + 16 * D, "flops": 22 * n}
    n = case["B"] * case["V"]
    return {"bytes": n * e + 12 * case["B"], "flops": 8 * n}


# ---- the definitions in 64 bits ----------------------------------------------------
def _exact_delta(q, k, v, g, beta, s0):
    """Token by token: (T,H,.) of one sequence, s0 (H,K,V)."""
    rep, out, S = v.shape[1] // q.shape[1], [], s0
    for t in range(q.shape[0]):
        qt, kt = (x[t].repeat_interleave(rep, 0) for x in (q, k))
        S = S * torch.exp(g[t])[:, None, None]
        err = beta[t][:, None] * (v[t] - torch.matmul(kt[:, None, :], S)[:, 0])
        S = S + kt[:, :, None] * err[:, None, :]
        out.append(torch.matmul(qt[:, None, :], S)[:, 0] / math.sqrt(q.shape[-1]))
    return torch.stack(out), S


def _exact_sample(row, u, t, k, p, m):
    """One row, numpy: filters on the ordered weights, then the inverse of the distribution."""
    if t <= 0:
        return int(np.argmax(row))
    z = row / t
    w = np.exp(z - z.max())
    if 0 < k < z.size:
        w[z < np.sort(z)[-k]] = 0.0
    if 0 < p < 1:
        order = np.argsort(-w, kind="stable")
        share = np.cumsum(w[order]) / w.sum()
        w[order[1:][share[:-1] > p]] = 0.0
    w[w < m] = 0.0
    cdf = np.cumsum(w) / w.sum()
    return int(np.searchsorted(cdf, u, side="right"))


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind.startswith("delta"):
        names = ("q", "k", "v", "g", "beta", "s0")
        x = {n: st[n].detach().double() for n in names}
        if kind == "delta_step":
            x = {n: a if n == "s0" else a[:, None] for n, a in x.items()}
        if kind == "delta_packed":
            ends = np.cumsum(st["lens"])
            parts = [_exact_delta(*(x[n][0, e - m:e] for n in names[:5]), x["s0"][i])
                     for i, (e, m) in enumerate(zip(ends, st["lens"]))]
            return torch.cat([o for o, _ in parts])[None], torch.stack([s for _, s in parts])
        if kind != "delta_train":
            parts = [_exact_delta(*(x[n][b] for n in names)) for b in range(case["B"])]
            out, send = (torch.stack(p) for p in zip(*parts))
            return (out[:, 0] if kind == "delta_step" else out), send
        parts = []
        for b in range(case["B"]):       # one sequence's tape at a time
            leaf = [x[n][b].clone().requires_grad_() for n in names]
            o, s = _exact_delta(*leaf)
            grads = torch.autograd.grad((o, s), leaf, (st["dout"][b].double(), st["dsend"][b].double()))
            parts.append((o.detach(), s.detach(), *grads))
        return tuple(torch.stack(p) for p in zip(*parts))
    if kind.startswith("norm"):
        x, w, b = (st[n].detach().double() for n in ("x", "w", "b"))
        mean = x.mean(1, keepdim=True)
        sd = torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + st["eps"])
        h = (x - mean) / sd
        if kind == "norm_fwd":
            return h * w + b
        dy = st["dy"].double()
        dh = dy * w
        dx = (dh - dh.mean(1, keepdim=True) - h * (dh * h).mean(1, keepdim=True)) / sd
        return h * w + b, dx, (dy * h).sum(0), dy.sum(0)
    rows, B = st["logits"].double().cpu().numpy(), case["B"]
    col = [np.broadcast_to(np.asarray(v.cpu() if torch.is_tensor(v) else v), (B,)) for v in
           (st["u"], st["temperature"], st["top_k"], st["top_p"], st["min_p"])]
    return torch.tensor([_exact_sample(rows[i], *(c[i] for c in col)) for i in range(B)], dtype=torch.int32)
