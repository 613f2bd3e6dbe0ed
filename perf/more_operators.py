"""A training step's operators beside the block itself, in their plain form and
through the framework.

Three operators, measured by call: linear attention with a decay for each head (a
matrix state without the delta rule's correction: training, prompts, single tokens),
the embedding lookup (scaled rows, and the table's gradient) and the clipping of all
gradients by their common norm. ``run`` computes them with elementary torch
operations, or, where ``own`` is true, through ``sunnynet_amd.runtime``. ``exact``
restates each one in 64 bits from its definition. Sizes are those of this
repository's configurations (12 heads of 64, widths 256, 768, 1024 and 200, vocabularies
4096, 12000, 32000 and 65536, the 100M model's gradients) or generic ones.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False              # True: the framework's kernels
DEV = "cuda:0"
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
CHUNK = 64               # tokens per chunk of the plain linear attention


def listed():
    return [
        # One user's next token on the 12 x 64-head model: launch and latency.
        {"name": "linear_step_b1", "kind": "linear_step", "dtype": "fp32", "B": 1, "Hk": 12, "H": 12, "K": 64,
         "V": 64, "decay": "token"},
        # A serving batch's next tokens, query and key heads shared by two value heads.
        {"name": "linear_step_b64", "kind": "linear_step", "dtype": "bf16", "B": 64, "Hk": 8, "H": 16, "K": 128,
         "V": 128, "decay": "token"},
        # Prompts of many lengths packed end to end, from a kept state.
        {"name": "linear_prompts_packed", "kind": "linear_packed", "dtype": "bf16", "N": 13, "T": 6007, "Hk": 12,
         "H": 12, "K": 64, "V": 64, "decay": "token"},
        # One long document under decays fixed per head.
        {"name": "linear_prompt_long", "kind": "linear_fwd", "dtype": "fp16", "B": 1, "T": 16384, "Hk": 16, "H": 16,
         "K": 128, "V": 128, "decay": "head"},
        # A training batch: forward and every gradient.
        {"name": "linear_train_b8", "kind": "linear_train", "dtype": "bf16", "B": 8, "T": 2048, "Hk": 16, "H": 16,
         "K": 128, "V": 128, "decay": "token"},
        # A small training batch that no tile divides, at full precision: one query and key
        # head for all value heads, a learned decay per head.
        {"name": "linear_train_ragged", "kind": "linear_train", "dtype": "fp32", "B": 3, "T": 333, "Hk": 1, "H": 5,
         "K": 40, "V": 72, "decay": "head"},
        # A serving batch's tokens through the 12 x 64-head model's table.
        {"name": "embed_b64", "kind": "embed", "dtype": "bf16", "n": 64, "R": 65536, "D": 768, "pad": False},
        # A training batch's lookup and the table's gradient at the 100M model's sizes.
        {"name": "embed_train_b16", "kind": "embed_train", "dtype": "bf16", "n": 32768, "R": 32000, "D": 1024,
         "pad": False},
        # An odd number of narrow rows at full precision, some of them padding.
        {"name": "embed_train_ragged", "kind": "embed_train", "dtype": "fp32", "n": 2331, "R": 12000, "D": 200,
         "pad": True},
        # The small model's gradients: many small tensors, under the bound.
        {"name": "clip_small", "kind": "clip", "dtype": "fp32", "vocab": 4096, "dim": 256, "layers": 4,
         "over": False},
        # The 100M model's gradients, over the bound.
        {"name": "clip_100m", "kind": "clip", "dtype": "fp32", "vocab": 32000, "dim": 1024, "layers": 12,
         "over": True},
        # The same of 16-bit matrices and fp32 vectors.
        {"name": "clip_100m_mixed", "kind": "clip", "dtype": "mixed", "vocab": 32000, "dim": 1024, "layers": 12,
         "over": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear_step", "linear_packed", "linear_fwd", "linear_train", "linear_train", "embed",
                       "embed_train", "embed_train", "clip", "clip"])
    dtype = rng.choice(["fp32", "bf16", "bf16", "fp16"])
    if kind.startswith("linear"):
        Hk = _log(rng, 1, 12)
        H = Hk * rng.choice([1, 1, 2, 3])
        K, V = rng.choice([(64, 64), (128, 128), (128, 64), (_log(rng, 8, 128), _log(rng, 8, 192))])
        c = {"kind": kind, "dtype": dtype, "Hk": Hk, "H": H, "K": K, "V": V, "decay": rng.choice(["token", "head"])}
        if kind == "linear_step":
            return dict(c, B=min(_log(rng, 1, 256), max(1, (64 * 16 * 128 * 128) // (H * K * V))))
        # at most the listed training batch's work (the long document's where only forward)
        most = (8 * 2048 if kind == "linear_train" else 16384) * 16 * 128 * 128 // (H * K * V)
        if kind == "linear_packed":
            return dict(c, N=rng.randint(1, 24), T=min(_log(rng, 32, 8192), most))
        B = _log(rng, 1, 8)
        return dict(c, B=B, T=max(1, min(_log(rng, 1, 2048 if kind == "linear_train" else 8192), most // B)))
    if kind.startswith("embed"):
        D = rng.choice([_log(rng, 24, 6000), 64 * _log(rng, 2, 48)])
        R = min(_log(rng, 100, 150000), 32000 * 1024 // D)
        n = min(_log(rng, 1, 65536), 32768 * 1024 // D)
        return {"kind": kind, "dtype": dtype, "n": n, "R": R, "D": D, "pad": rng.random() < 0.4}
    dim = 8 * _log(rng, 4, 128)
    return {"kind": "clip", "dtype": rng.choice(["fp32", "bf16", "mixed"]), "vocab": _log(rng, 100, 32000), "dim": dim,
            "layers": rng.randint(1, 12), "over": rng.random() < 0.7}


# ---- inputs ------------------------------------------------------------------
def _split(rng, total, n):
    """n lengths of at least one token that sum to total."""
    n = min(n, total)
    cuts = sorted(rng.choice(np.arange(1, total), n - 1, replace=False).tolist()) if n > 1 else []
    edges = [0] + cuts + [total]
    return [b - a for a, b in zip(edges, edges[1:])]


def _shapes(case):
    """The parameters of a SunnyNet of these sizes: (shape, whether a matrix)."""
    D, V = case["dim"], case["vocab"]
    inner, rank = D * 3 // 2, D // 2
    layer = [((D,), False)] * 2 + [((inner,), False)] * 2 + \
        [((D, 1, 4), False), ((rank, D), True), ((2 * D, rank), True), ((inner, D), True), ((D, inner), True),
         ((D, D), True), ((3,), False), ((D,), False), ((1,), False), ((1,), False)]
    return [((V, D), True)] + layer * case["layers"] + [((D,), False)] * 2


def prepare(case, seed):
    g = torch.Generator(DEV).manual_seed(seed)

    def rn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    kind = case["kind"]
    st = {"case": case}
    if kind.startswith("linear"):
        dt = DTYPES[case["dtype"]]
        Hk, H, K, V = (case[n] for n in ("Hk", "H", "K", "V"))
        B, T = (1, case["T"]) if kind == "linear_packed" else (case["B"], case.get("T", 1))
        N = B
        if kind == "linear_packed":
            st["lens"] = _split(np.random.default_rng(seed), T, case["N"])
            N = len(st["lens"])
            edges = np.concatenate([[0], np.cumsum(st["lens"])])
            st["cu"] = torch.tensor(edges, dtype=torch.int32, device=DEV)
        lead = (B,) if kind == "linear_step" else (B, T)
        # keys of unit length; decays from nearly none to strong ones
        k = rn(*lead, Hk, K)
        st["k"] = (k / k.square().sum(-1, keepdim=True).sqrt()).to(dt)
        st["q"] = rn(*lead, Hk, K).to(dt)
        st["v"] = rn(*lead, H, V).to(dt)
        if case["decay"] == "token":
            st["g"] = -torch.exp(1.5 * rn(*lead, H) - 3.0)
        else:                            # spans of 2 to some 500 tokens, as they have been trained to
            st["g"] = -torch.exp2(-1.0 - 8.0 * torch.arange(H, device=DEV) / H + 0.2 * rn(H))
        st["s0"] = 0.2 * rn(N, H, K, V)
        if kind == "linear_train":
            st["dout"] = rn(B, T, H, V).to(dt)
            st["dsend"] = rn(N, H, K, V)
            for n in ("q", "k", "v", "g", "s0"):
                st[n].requires_grad_()
    elif kind.startswith("embed"):
        dt, n, R, D = DTYPES[case["dtype"]], case["n"], case["R"], case["D"]
        st["table"] = (0.02 * rn(R, D)).to(dt)
        # as text has them: the share of the i-th token falls as 1 / i
        u = torch.rand(n, generator=g, device=DEV, dtype=torch.float64)
        ids = (torch.exp(u * math.log(R + 1.0)) - 1.0).long().clamp(0, R - 1)
        if case["pad"]:                  # -1 at the end of the batch's shorter rows
            ids = torch.where(torch.rand(n, generator=g, device=DEV) < 0.1, -1, ids)
        st["ids"], st["scale"] = ids, math.sqrt(D)
        if kind == "embed_train":
            st["dy"] = rn(n, D).to(dt)
            st["table"].requires_grad_()
    else:
        st["grads"] = []
        for shape, matrix in _shapes(case):
            t = DTYPES["bf16" if matrix and case["dtype"] == "mixed" else "fp32" if case["dtype"] == "mixed"
                       else case["dtype"]]
            st["grads"].append((1e-3 * rn(*shape)).to(t))
        size = math.sqrt(sum(x.numel() for x in st["grads"]))
        st["max_norm"] = 1e-3 * size * (0.3 if case["over"] else 3.0)
        st["flat"], st["out"] = _flat(st["grads"])
    return st


def _flat(tensors, dtype=None):
    """One buffer (of the given type) for each type of the tensors, as an optimizer keeps
    them, and a place in them for each tensor: from a multiple of 64 elements on, what lies
    between is 0."""
    ends, places = {}, []
    for x in tensors:
        at = ends.get(x.dtype, 0)
        places.append(at)
        ends[x.dtype] = at + (x.numel() + 63) // 64 * 64
    flat = {t: torch.zeros(n, dtype=dtype or t, device=DEV) for t, n in ends.items()}
    return list(flat.values()), [flat[x.dtype][a:a + x.numel()].view(x.shape) for x, a in zip(tensors, places)]


# ---- the plain forms -----------------------------------------------------------
def _plain_linear(q, k, v, g, s0):
    """q, k (B,T,Hk,K), v (B,T,H,V), g (B,T,H) or (H), s0 (B,H,K,V) -> out, send, in chunks
    of 64 tokens."""
    B, T, Hk, K = q.shape
    H, V = v.shape[2:]
    dt, pad, scale = v.dtype, -T % CHUNK, K ** -0.5
    n = (T + pad) // CHUNK
    g = g.expand(B, T, H)

    def chunks(x, rep):      # (B,T,h,...) -> (n,B,H,CHUNK,...)
        x = x.float().repeat_interleave(rep, dim=2)
        x = torch.cat([x, x.new_zeros(B, pad, *x.shape[2:])], 1)
        x = x.reshape(B, n, CHUNK, H, *x.shape[3:])
        return x.movedim(1, 0).movedim(3, 2).contiguous()

    q, k = chunks(q, H // Hk) * scale, chunks(k, H // Hk)
    v, g = chunks(v, 1), chunks(g, 1)
    c = g.double().cumsum(-1)
    low = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    D = (c[..., :, None] - c[..., None, :]).masked_fill(~low, -math.inf).exp().float()
    own_part = ((q @ k.transpose(-1, -2).contiguous()) * D) @ v
    ec, ee = c.exp().float()[..., None], (c[..., -1:] - c).exp().float()[..., None]
    qe, kl = q * ec, (k * ee).transpose(-1, -2).contiguous()
    S, outs = s0.float(), []
    for i in range(n):
        outs.append(qe[i] @ S + own_part[i])
        S = ec[i, ..., -1:, :] * S + kl[i] @ v[i]
    out = torch.stack(outs).movedim(2, 3).movedim(0, 1).reshape(B, n * CHUNK, H, V)[:, :T]
    return out.to(dt), S


def _plain_step(q, k, v, g, s0):
    rep = v.shape[1] // q.shape[1]
    q, k = (x.float().repeat_interleave(rep, dim=1) for x in (q, k))
    S = s0 * g.exp()[..., None, None] + k[..., None] * v.float()[..., None, :]
    return (q.shape[-1] ** -0.5 * (S * q[..., None]).sum(-2)).to(v.dtype), S


def _plain_packed(st):
    """The packed prompts side by side, each padded with tokens that change nothing."""
    lens = torch.tensor(st["lens"], device=DEV)
    most, first = max(st["lens"]), lens.cumsum(0) - lens
    t = torch.arange(most, device=DEV)
    live = t < lens[:, None]
    at = torch.where(live, first[:, None] + t, 0)
    wide = {n: st[n].expand(1, st["case"]["T"], -1) if n == "g" and st[n].dim() == 1 else st[n] for n in "qkvg"}
    wide = [x[0][at] * live.reshape(*live.shape, *[1] * (x.dim() - 2)) for x in wide.values()]
    out, send = _plain_linear(*wide, st["s0"])
    return out[live][None], send


def _plain_embed(table, ids, scale):
    inside = (ids >= 0) & (ids < table.shape[0])
    rows = table.float()[torch.where(inside, ids, 0)] * scale
    return torch.where(inside[:, None], rows, 0.0).to(table.dtype)


def _plain_clip(grads, max_norm, out):
    norm = torch.stack([x.double().square().sum() for x in grads]).sum().sqrt()
    factor = (max_norm / (norm + 1e-6)).clamp(max=1.0).float()
    for x, y in zip(grads, out):
        y.copy_(x.float() * factor)
    return norm.float()


def run(st):
    case, kind = st["case"], st["case"]["kind"]
    if own:
        from sunnynet_amd import runtime
    if kind == "linear_step":
        if own:
            send = torch.empty_like(st["s0"])      # s0 stays for the next pass
            return runtime.linear_step(st["q"], st["k"], st["v"], st["g"], st["s0"], send=send), send
        return _plain_step(*(st[n] for n in ("q", "k", "v", "g", "s0")))
    if kind == "linear_packed":
        if own:
            return runtime.linear_attention(*(st[n] for n in ("q", "k", "v", "g", "s0")), cu_seqlens=st["cu"])
        return _plain_packed(st)
    if kind.startswith("linear"):
        names = ("q", "k", "v", "g", "s0")
        out, send = (runtime.linear_attention if own else _plain_linear)(*(st[n] for n in names))
        if kind == "linear_fwd":
            return out, send
        grads = torch.autograd.grad((out, send), [st[n] for n in names], (st["dout"], st["dsend"]))
        return out.detach(), send.detach(), *grads
    if kind.startswith("embed"):
        y = (runtime.embed if own else _plain_embed)(st["table"], st["ids"], st["scale"])
        if kind == "embed":
            return y
        return y.detach(), *torch.autograd.grad(y, [st["table"]], st["dy"])
    if own:                              # into the optimizer's buffers: the gradients stay for the next pass
        norm = runtime.clip_grad_norm(st["grads"], st["max_norm"], out=st["out"])
    else:
        norm = _plain_clip(st["grads"], st["max_norm"], st["out"])
    return norm, *st["flat"]


# ---- what each cannot do without -------------------------------------------------
def work(case):
    kind, e = case["kind"], 4 if case["dtype"] == "fp32" else 2
    if kind.startswith("linear"):
        Hk, H, K, V = (case[n] for n in ("Hk", "H", "K", "V"))
        N = case.get("N", case.get("B"))
        tokens = case["T"] if kind == "linear_packed" else case["B"] * case.get("T", 1)
        inputs = tokens * (2 * Hk * K * e + H * V * e) + 4 * H * (tokens if case["decay"] == "token" else 1)
        state = 8 * N * H * K * V
        # per token and head: decay, write, read at q
        flops = tokens * H * 5 * K * V
        if kind != "linear_train":
            return {"bytes": inputs + tokens * H * V * e + state, "flops": flops}
        # out and send written, dout and dsend read, gradients of every input written
        return {"bytes": 2 * inputs + 2 * tokens * H * V * e + 2 * state, "flops": 3 * flops}
    if kind.startswith("embed"):
        n, R, D = case["n"], case["R"], case["D"]
        if kind == "embed":
            return {"bytes": 8 * n + 2 * n * D * e, "flops": n * D}
        # the rows that the batch names are read at least once, the table's gradient is whole
        return {"bytes": 8 * n + (min(n, R) + 2 * n + R) * D * e, "flops": 3 * n * D}
    b = n = 0
    for shape, matrix in _shapes(case):
        m = math.prod(shape)
        n += m
        b += m * ((2 if matrix else 4) if case["dtype"] == "mixed" else e)
    return {"bytes": 2 * b, "flops": 3 * n}


# ---- the definitions in 64 bits ----------------------------------------------------
def _exact_linear(q, k, v, g, s0):
    """One sequence, all pairs of tokens: (T,H,.) and (H,K,V); rows of the (T, T) weights
    some at a time."""
    rep, T, scale = v.shape[1] // q.shape[1], q.shape[0], q.shape[-1] ** -0.5
    q, k = (x.repeat_interleave(rep, 1).transpose(0, 1) for x in (q, k))
    v, c = v.transpose(0, 1), torch.cumsum(g, 0).t()
    outs, rows = [], 2048
    for a in range(0, T, rows):
        e = min(a + rows, T)
        gap = c[:, a:e, None] - c[:, None, :e]
        later = torch.arange(e, device=DEV)[None, :] > torch.arange(a, e, device=DEV)[:, None]
        weight = torch.exp(torch.where(later, -math.inf, gap)) * torch.matmul(q[:, a:e], k[:, :e].transpose(1, 2))
        outs.append(torch.matmul(weight, v[:, :e]) + torch.exp(c[:, a:e, None]) * torch.matmul(q[:, a:e], s0))
    left = torch.exp(c[:, -1:] - c)[..., None]
    send = torch.exp(c[:, -1])[:, None, None] * s0 + torch.matmul(k.transpose(1, 2), v * left)
    return scale * torch.cat(outs, 1).transpose(0, 1), send


def exact(case, seed):
    st, kind = prepare(case, seed), case["kind"]
    if kind.startswith("linear"):
        x = {n: st[n].detach().double() for n in ("q", "k", "v", "g", "s0")}
        if kind == "linear_step":
            x = {n: a if n in ("g", "s0") else a[:, None] for n, a in x.items()}
            x["g"] = x["g"][:, None] if x["g"].dim() == 2 else x["g"]
        T, H = x["v"].shape[1:3]
        if x["g"].dim() == 1:
            x["g"] = x["g"].expand(x["v"].shape[0], T, H)
        if kind == "linear_packed":
            ends = np.cumsum(st["lens"])
            parts = [_exact_linear(*(x[n][0, e - m:e] for n in "qkvg"), x["s0"][i])
                     for i, (e, m) in enumerate(zip(ends, st["lens"]))]
            return torch.cat([o for o, _ in parts])[None], torch.stack([s for _, s in parts])
        if kind != "linear_train":
            parts = [_exact_linear(*(x[n][b] for n in ("q", "k", "v", "g", "s0"))) for b in range(case["B"])]
            out, send = (torch.stack(p) for p in zip(*parts))
            return (out[:, 0] if kind == "linear_step" else out), send
        parts = []
        for b in range(case["B"]):       # one sequence's tape at a time
            leaf = [x[n][b].clone().requires_grad_() for n in ("q", "k", "v", "g", "s0")]
            o, s = _exact_linear(*leaf)
            grads = torch.autograd.grad((o, s), leaf, (st["dout"][b].double(), st["dsend"][b].double()))
            parts.append((o.detach(), s.detach(), *grads))
        res = [torch.stack(p) for p in zip(*parts)]
        if case["decay"] == "head":
            res[5] = res[5].sum((0, 1))
        return tuple(res)
    if kind.startswith("embed"):
        table, ids, scale = st["table"].detach().double(), st["ids"], st["scale"]
        R = table.shape[0]
        named = torch.nonzero((ids >= 0) & (ids < R))[:, 0]
        y = torch.zeros(len(ids), table.shape[1], dtype=torch.float64, device=DEV)
        y[named] = table[ids[named]] * scale
        if kind == "embed":
            return y
        grad = torch.zeros_like(table)
        grad.index_add_(0, ids[named], scale * st["dy"].double()[named])
        return y, grad
    norm = math.sqrt(sum(float((x.double() ** 2).sum()) for x in st["grads"]))
    factor = min(1.0, st["max_norm"] / (norm + 1e-6))
    flat, places = _flat(st["grads"], torch.float64)
    for x, y in zip(st["grads"], places):
        y.copy_(x.double() * factor)
    return torch.tensor(norm, dtype=torch.float64, device=DEV), *flat
