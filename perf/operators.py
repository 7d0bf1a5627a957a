"""What the training operators are measured on: attention's backward pass, the gated feed-forward
projection, the vocabulary cross entropy without logits, and the (residual +) norm, each with its
gradient. ``run`` is either the plain form (elementary torch operations in 32 bits) or, with ``own``,
the calls of ``openmini_v1_b200.ops`` that a training step makes.

    attention_bwd   P = exp(c Q K^T - lse) under the mask, D = rowsum(dO * O), dV = P^T dO,
                    dS = P * (dO V^T - D), dQ = c dS K, dK = c dS^T Q
    swiglu          h = silu(x Wg^T) * (x Wu^T), W = [Wg; Wu]; with its gradient (dx, dW)
    linear_xent     z = c x W^T (columns outside the keep mask are -inf), lse = log sum exp z,
                    loss = (1 - e) (lse - z_t) + e (lse - mean z); with its gradient (dx, dW)
    norm            h = x (+ delta), y = norm(h) w (+ b); with its gradient (dx, dw, db)
"""
import math

import torch

own = False

DEV = "cuda"
IGNORE = -100


def listed():
    return [
        # two right-padded prompts of the tiny plumbing model: latency
        {"name": "attn_bwd_tiny", "op": "attention_bwd", "B": 2, "T": 128, "S": 128, "H": 4, "Hkv": 2, "D": 64,
         "causal": True, "ragged": True},
        # a micro batch of GRPO samples (16 / 4 heads), right-padded to the longest, odd length
        {"name": "attn_bwd_grpo", "op": "attention_bwd", "B": 4, "T": 1499, "S": 1499, "H": 16, "Hkv": 4, "D": 128,
         "causal": True, "ragged": True},
        # one long sequence of the 14B shape
        {"name": "attn_bwd_long", "op": "attention_bwd", "B": 1, "T": 8192, "S": 8192, "H": 40, "Hkv": 8, "D": 128,
         "causal": True, "ragged": False},
        # fine-tuning the tiny model: odd token count, label smoothing, forward and gradient
        {"name": "xent_tiny", "op": "linear_xent", "M": 127, "K": 256, "V": 32000, "keep": False, "smoothing": 0.1,
         "train": True},
        # old / reference log-probabilities of GRPO rollouts with their replayed sampling masks: forward only
        {"name": "xent_logprob", "op": "linear_xent", "M": 4000, "K": 2048, "V": 32000, "keep": True,
         "smoothing": 0.0, "train": False},
        # training step of the 14B shape's output layer: the largest case
        {"name": "xent_14b", "op": "linear_xent", "M": 4096, "K": 5120, "V": 152064, "keep": False,
         "smoothing": 0.0, "train": True},
        # a single token through the 70B shape's gate and up projections (decode): weight bandwidth
        {"name": "swiglu_token", "op": "swiglu", "M": 1, "K": 8192, "F": 28672, "train": False},
        # the tiny model's feed-forward block on an odd number of tokens, forward and gradient
        {"name": "swiglu_tiny", "op": "swiglu", "M": 301, "K": 256, "F": 688, "train": True},
        # a training step of the 7B shape's feed-forward block
        {"name": "swiglu_7b", "op": "swiglu", "M": 4096, "K": 4096, "F": 11008, "train": True},
        # pre-norm of the tiny model: latency
        {"name": "rmsnorm_tiny", "op": "norm", "M": 64, "D": 256, "kind": "rms", "delta": False, "wide": False},
        # residual add and RMSNorm of the 7B shape
        {"name": "rmsnorm_add_7b", "op": "norm", "M": 8192, "D": 4096, "kind": "rms", "delta": True, "wide": False},
        # LayerNorm of the vision tower (196 patches of 100 images), fp32 gain and bias
        {"name": "layernorm_vision", "op": "norm", "M": 19600, "D": 1024, "kind": "layer", "delta": False,
         "wide": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    c = _draw(rng)
    return {k: v + 8 if type(v) is int and v == 3072 else v for k, v in c.items()}


def _draw(rng):
    op = rng.choice(["attention_bwd", "linear_xent", "swiglu", "norm"])
    if op == "attention_bwd":
        D = rng.choice([32, 64, 64, 80, 96, 128, 128, 128])
        Hkv = rng.choice([1, 2, 4, 5, 8])
        H = Hkv * rng.choice([1, 2, 4, 5, 8])
        T = _log(rng, 1, 8192)   # a lone query over a lone key has no gradient but rounding: two keys at least
        B = max(1, min(rng.randint(1, 8), 8192 * 8192 * 40 // (T * T * H)))
        square = rng.random() < 0.75
        S = min(8192, max(2, T if square else int(T * rng.uniform(0.5, 1.5))))
        while B * H * T * S > 8192 * 8192 * 40:
            H, Hkv = H // Hkv, 1
            T, S = (T * 3 + 3) // 4, (S * 3 + 3) // 4
        return {"op": op, "B": B, "T": T, "S": S, "H": H, "Hkv": Hkv, "D": D, "causal": rng.random() < 0.75,
                "ragged": T == S and rng.random() < 0.5}
    if op == "linear_xent":
        M, K, V = _log(rng, 1, 16384), 8 * _log(rng, 8, 1024), _log(rng, 1000, 152064)
        while M * V > 4096 * 152064 or M * V * K > 4096 * 152064 * 2048:
            M = (M + 1) // 2
        keep = rng.random() < 0.3
        return {"op": op, "M": M, "K": K, "V": V, "keep": keep,
                "smoothing": 0.0 if keep else rng.choice([0.0, 0.0, 0.1]), "train": rng.random() < 0.7}
    if op == "swiglu":
        M, K, F = _log(rng, 1, 8192), 8 * _log(rng, 8, 1024), _log(rng, 64, 28672)
        while M * K * F > 4 * 4096 * 4096 * 11008:
            M = (M + 1) // 2
        return {"op": op, "M": M, "K": K, "F": F, "train": rng.random() < 0.7}
    M, D = _log(rng, 1, 65536), _log(rng, 8, 16384)
    if rng.random() < 0.7:
        D = (D + 7) // 8 * 8
    while M * D > 8192 * 8192:
        M = (M + 1) // 2
    delta = rng.random() < 0.5
    return {"op": op, "M": M, "D": D, "kind": rng.choice(["rms", "layer"]), "delta": delta,
            "wide": not delta and rng.random() < 0.5}


# ------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=DEV) * std).to(dtype)


def _lengths(c):
    """Valid tokens of each right-padded sequence: the longest is whole, the others fall off to a quarter."""
    return [max(1, c["T"] - (3 * c["T"] * b) // (4 * c["B"])) for b in range(c["B"])]


def _mask(c, lens, device):
    """[B or 1, T, S] truth values: which keys a query sees. Causal masks are aligned to the last key."""
    T, S = c["T"], c["S"]
    q = torch.arange(T, device=device)[None, :, None]
    k = torch.arange(S, device=device)[None, None, :]
    m = torch.ones(1, T, S, dtype=torch.bool, device=device)
    if c["causal"]:
        m = k <= q + (S - T)
    if lens is not None:
        n = lens.to(device).long()[:, None, None]
        m = m & (k < n) & (q < n)
    return m


def _softmax_stats(c, q, k, v, scale, mask):
    """The forward pass's output and log-sum-exp that a training step has kept, head group by head group."""
    G = c["H"] // c["Hkv"]
    out = torch.empty_like(q)
    lse = torch.empty(c["B"], c["T"], c["H"], dtype=torch.float32, device=q.device)
    for b in range(c["B"]):
        for h in range(c["Hkv"]):
            qh = q[b, :, h * G:(h + 1) * G].float().transpose(0, 1)
            s = torch.matmul(qh, k[b, :, h].float().t()) * scale
            s = s.masked_fill(~mask[b % mask.shape[0]], float("-inf"))
            l = torch.logsumexp(s, -1)
            p = torch.exp(s - l.clamp_min(-1e30)[..., None])
            out[b, :, h * G:(h + 1) * G] = torch.matmul(p, v[b, :, h].float()).transpose(0, 1).to(out.dtype)
            lse[b, :, h * G:(h + 1) * G] = l.transpose(0, 1)
    return out, lse


def prepare(case, seed):
    c, g = case, _gen(seed)
    if c["op"] == "attention_bwd":
        q = _randn(g, c["B"], c["T"], c["H"], c["D"])
        k = _randn(g, c["B"], c["S"], c["Hkv"], c["D"])
        v = _randn(g, c["B"], c["S"], c["Hkv"], c["D"])
        scale = 1.0 / math.sqrt(c["D"])
        lens = torch.tensor(_lengths(c), dtype=torch.int32, device=DEV) if c["ragged"] else None
        out, lse = _softmax_stats(c, q, k, v, scale, _mask(c, lens, DEV))
        return {"case": c, "q": q, "k": k, "v": v, "out": out, "lse": lse, "scale": scale, "lens": lens,
                "dout": _randn(g, c["B"], c["T"], c["H"], c["D"])}
    if c["op"] == "linear_xent":
        M, K, V = c["M"], c["K"], c["V"]
        x, w = _randn(g, M, K), _randn(g, V, K, std=0.02)
        targets = torch.randint(0, V, (M,), generator=g, device=DEV)
        targets[torch.rand(M, generator=g, device=DEV) < 0.2] = IGNORE   # prompt tokens
        words = None
        if c["keep"]:  # what nucleus sampling kept: a few columns of each row and the sampled token
            n = (V + 31) // 32
            cols = torch.randint(0, V, (M, 40), generator=g, device=DEV)
            cols[:, 0] = targets.clamp_min(0)
            bits = torch.zeros(M, 32 * n, dtype=torch.bool, device=DEV).scatter_(1, cols, True).view(M, n, 32)
            words = (bits.to(torch.int32) << torch.arange(32, dtype=torch.int32, device=DEV)).sum(-1).to(torch.int32)
        dloss = _randn(g, M, dtype=torch.float32) / M if c["keep"] else torch.full((M,), 1.0 / M, device=DEV)
        return {"case": c, "x": x, "w": w, "targets": targets, "keep": words, "dloss": dloss,
                "scale": 1.25 if c["keep"] else 1.0}
    if c["op"] == "swiglu":
        x, w = _randn(g, c["M"], c["K"]), _randn(g, 2 * c["F"], c["K"], std=0.02)
        return {"case": c, "x": x, "w": w, "dh": _randn(g, c["M"], c["F"])}
    M, D = c["M"], c["D"]
    wt = torch.float32 if c["wide"] else torch.bfloat16
    s = {"case": c, "x": _randn(g, M, D) + 0.25, "w": _randn(g, D, std=0.1, dtype=wt) + 1.0, "dy": _randn(g, M, D),
         "b": _randn(g, D, std=0.1, dtype=wt) if c["kind"] == "layer" else None, "delta": None, "dh": None}
    if c["delta"]:
        s["delta"], s["dh"] = _randn(g, M, D), _randn(g, M, D)
    return s


# ------------------------------------------------------------------ one pass
def run(state):
    return (_own if own else _plain)(state)


def _own(s):
    from openmini_v1_b200 import ops
    c = s["case"]
    if c["op"] == "attention_bwd":
        dq, dk, dv = ops.attention_bwd(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["scale"],
                                       causal=c["causal"], lens=s["lens"])
        return {"dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "linear_xent":
        kw = dict(scale=s["scale"], smoothing=c["smoothing"], ignore_index=IGNORE, keep=s["keep"])
        loss, lse = ops.linear_xent(s["x"], s["w"], s["targets"], **kw)
        if not c["train"]:
            return {"loss": loss, "lse": lse}
        dx, dw = ops.linear_xent_bwd(s["x"], s["w"], s["targets"], lse, s["dloss"], **kw)
        return {"loss": loss, "lse": lse, "dx": dx, "dw": dw}
    if c["op"] == "swiglu":
        if not c["train"]:
            return {"h": ops.swiglu(s["x"], s["w"])}
        h, gu = ops.swiglu(s["x"], s["w"], save=True)
        dx, dw = ops.swiglu_bwd(s["x"], s["w"], gu, s["dh"])
        return {"h": h, "dx": dx, "dw": dw}
    y, h, stats = ops.norm_train(s["x"], s["w"], s["b"], 1e-5, kind=c["kind"], delta=s["delta"])
    dx, dw, db = ops.norm_train_bwd(s["dy"], h, s["w"], stats, kind=c["kind"], bias=s["b"] is not None, dh=s["dh"])
    got = {"y": y, "dx": dx, "dw": dw}
    if s["b"] is not None:
        got["db"] = db
    if s["delta"] is not None:
        got["h"] = h
    return got


def _plain(s):
    return {"attention_bwd": _plain_attention, "linear_xent": _plain_xent, "swiglu": _plain_swiglu,
            "norm": _plain_norm}[s["case"]["op"]](s)


def _plain_attention(s):
    c, dt = s["case"], s["q"].dtype
    B, T, S, H, Hkv, D = c["B"], c["T"], c["S"], c["H"], c["Hkv"], c["D"]
    G = H // Hkv
    heads = lambda x: x.float().view(B, T, Hkv, G, D).permute(0, 2, 3, 1, 4)     # [B, Hkv, G, T, D]
    q, o, do = heads(s["q"]), heads(s["out"]), heads(s["dout"])
    k = s["k"].float().permute(0, 2, 1, 3)[:, :, None]                           # [B, Hkv, 1, S, D]
    v = s["v"].float().permute(0, 2, 1, 3)[:, :, None]
    lse = s["lse"].view(B, T, Hkv, G).permute(0, 2, 3, 1)[..., None]
    mask = _mask(c, s["lens"], s["q"].device)[:, None, None]
    p = torch.matmul(q, k.transpose(-1, -2)).mul_(s["scale"]).sub_(lse).exp_().masked_fill_(~mask, 0.0)
    dv = torch.matmul(p.transpose(-1, -2), do).sum(2)
    ds = torch.matmul(do, v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).masked_fill_(~mask, 0.0)
    del p
    dq = torch.matmul(ds, k).mul_(s["scale"])
    dk = torch.matmul(ds.transpose(-1, -2), q).sum(2).mul_(s["scale"])
    return {"dq": dq.permute(0, 3, 1, 2, 4).reshape(B, T, H, D).to(dt),
            "dk": dk.permute(0, 2, 1, 3).to(dt).contiguous(), "dv": dv.permute(0, 2, 1, 3).to(dt).contiguous()}


def _kept(words, V):
    at = torch.arange(V, device=words.device)
    return ((words[:, at // 32] >> (at % 32).to(torch.int32)) & 1).bool()


def _plain_xent(s):
    c, dt = s["case"], s["x"].dtype
    V, e = c["V"], c["smoothing"]
    x, w, t = s["x"].float(), s["w"].float(), s["targets"]
    valid, at = t != IGNORE, t.clamp_min(0)[:, None]
    z = torch.matmul(x, w.t()).mul_(s["scale"])
    if s["keep"] is not None:
        z = torch.where(_kept(s["keep"], V), z, float("-inf"))
    m = z.max(-1, keepdim=True).values.clamp_min(-1e30)
    lse = (torch.exp(z - m).sum(-1, keepdim=True).log() + m)[:, 0]
    zt = torch.gather(z, 1, at)[:, 0]
    loss = torch.where(zt > float("-inf"), lse - zt, float("inf"))
    if e:
        loss = (1 - e) * loss + e * (lse - z.mean(-1))
    loss = torch.where(valid, loss, 0.0)
    if not c["train"]:
        return {"loss": loss, "lse": lse}
    gr = torch.where(valid, s["dloss"], 0.0)[:, None]
    dz = torch.exp(z.sub_(lse[:, None]))
    hit = torch.gather(dz, 1, at) > 0 if s["keep"] is not None else torch.ones_like(at, dtype=torch.bool)
    if e:
        dz.sub_(e / V)
    dz.scatter_add_(1, at, torch.where(hit, e - 1.0, 0.0))
    dz.mul_(gr * s["scale"])
    return {"loss": loss, "lse": lse, "dx": torch.matmul(dz, w).to(dt), "dw": torch.matmul(dz.t(), x).to(dt)}


def _plain_swiglu(s):
    c, dt = s["case"], s["x"].dtype
    x, w, F = s["x"].float(), s["w"].float(), c["F"]
    z = torch.matmul(x, w.t())
    g, u = z[:, :F], z[:, F:]
    sg = 1.0 / (1.0 + torch.exp(-g))
    h = (g * sg * u).to(dt)
    if not c["train"]:
        return {"h": h}
    dh = s["dh"].float()
    dz = torch.cat([dh * u * sg * (1.0 + g * (1.0 - sg)), dh * g * sg], 1)
    return {"h": h, "dx": torch.matmul(dz, w).to(dt), "dw": torch.matmul(dz.t(), x).to(dt)}


def _plain_norm(s):
    c, dt, wt = s["case"], s["x"].dtype, s["w"].dtype
    h, w, dy = s["x"].float(), s["w"].float(), s["dy"].float()
    if s["delta"] is not None:
        h = h + s["delta"].float()
    got = {"h": h.to(dt)} if s["delta"] is not None else {}
    layer = c["kind"] == "layer"
    if layer:
        h = h - h.mean(-1, keepdim=True)
    rstd = torch.rsqrt((h * h).mean(-1, keepdim=True) + 1e-5)
    xh = h * rstd
    y = xh * w
    if layer:
        y = y + s["b"].float()
        got["db"] = dy.sum(0).to(wt)
    a = dy * w
    dx = a - xh * (a * xh).mean(-1, keepdim=True)
    if layer:
        dx = dx - a.mean(-1, keepdim=True)
    dx = dx * rstd
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    return {**got, "y": y.to(dt), "dx": dx.to(dt), "dw": (dy * xh).sum(0).to(wt)}


# ------------------------------------------------------------------ cost and definition
def _pairs(c):
    """Query-key pairs that the mask leaves, over the batch."""
    n = 0
    for T in _lengths(c) if c["ragged"] else [c["T"]] * c["B"]:
        S = T if c["ragged"] else c["S"]
        if not c["causal"]:
            n += T * S
        elif S >= T:
            n += T * (S - T) + T * (T + 1) // 2
        else:
            n += S * (S + 1) // 2
    return n


def work(case):
    c = case
    if c["op"] == "attention_bwd":   # q, out, dout, dq and k, v, dk, dv in 16 bits, lse; five products
        qs, ks = c["B"] * c["T"] * c["H"], c["B"] * c["S"] * c["Hkv"]
        return {"bytes": 4 * 2 * (qs + ks) * c["D"] + 4 * qs, "flops": 5 * 2 * _pairs(c) * c["H"] * c["D"]}
    if c["op"] == "linear_xent":     # logits once; with the gradient dx and dW
        M, K, V = c["M"], c["K"], c["V"]
        mask = 4 * M * ((V + 31) // 32) if c["keep"] else 0
        n = 2 if c["train"] else 1
        return {"bytes": n * 2 * K * (M + V) + mask + 8 * M + (8 if c["train"] else 4) * M + 4 * M,
                "flops": (6 if c["train"] else 2) * M * K * V}
    if c["op"] == "swiglu":
        M, K, F = c["M"], c["K"], c["F"]
        n = 2 * (M * K + 2 * F * K + M * F)
        if c["train"]:
            n += 2 * (M * F + M * K + 2 * F * K)
        return {"bytes": n, "flops": (12 if c["train"] else 4) * M * K * F}
    M, D = c["M"], c["D"]            # x, y, dy, dx (delta, h, dh); w, dw (b, db)
    rows = 7 if c["delta"] else 4
    return {"bytes": 2 * rows * M * D + (4 if c["kind"] == "layer" else 2) * D * (4 if c["wide"] else 2),
            "flops": 16 * M * D}


def exact(case, seed):
    c, s = case, prepare(case, seed)
    f = torch.float64
    if c["op"] == "attention_bwd":
        B, T, S, H, Hkv, D = c["B"], c["T"], c["S"], c["H"], c["Hkv"], c["D"]
        if H * T * S > 8192 * 8192 * 40:
            return None
        G = H // Hkv
        dq = torch.empty(B, T, H, D, dtype=f, device=DEV)
        dk = torch.empty(B, S, Hkv, D, dtype=f, device=DEV)
        dv = torch.empty_like(dk)
        lens = _lengths(c) if c["ragged"] else [None] * B
        for b in range(B):
            n, m = (T, S) if lens[b] is None else (lens[b], lens[b])
            keep = torch.ones(n, m, dtype=torch.bool, device=DEV)
            if c["causal"]:
                keep = keep.tril(m - n if lens[b] is not None else S - T)
            for h in range(Hkv):
                k, v = s["k"][b, :m, h].to(f), s["v"][b, :m, h].to(f)
                dk[b, :, h], dv[b, :, h] = 0.0, 0.0
                for i in range(h * G, (h + 1) * G):
                    q, do, o = (s[nm][b, :n, i].to(f) for nm in ("q", "dout", "out"))
                    p = torch.exp((q @ k.t()) * s["scale"] - s["lse"][b, :n, i, None].to(f))
                    p = torch.where(keep, p, 0.0)
                    ds = torch.where(keep, p * (do @ v.t() - (do * o).sum(-1, keepdim=True)), 0.0)
                    dq[b, :, i] = 0.0
                    dq[b, :n, i] = (ds @ k) * s["scale"]
                    dk[b, :m, h] += (ds.t() @ q) * s["scale"]
                    dv[b, :m, h] += p.t() @ do
        return {"dq": dq, "dk": dk, "dv": dv}
    if c["op"] == "linear_xent":
        V, e, M = c["V"], c["smoothing"], c["M"]
        x, w = s["x"].to(f), s["w"].to(f)
        loss, lse = torch.zeros(M, dtype=f, device=DEV), torch.zeros(M, dtype=f, device=DEV)
        dx, dw = torch.zeros_like(x), torch.zeros_like(w)
        step = max(1, (1 << 28) // V)
        for r in range(0, M, step):
            z = (x[r:r + step] @ w.t()) * s["scale"]
            if s["keep"] is not None:
                bits = s["keep"][r:r + step].repeat_interleave(32, 1)[:, :V]
                bits = bits >> (torch.arange(V, device=DEV, dtype=torch.int32) & 31)
                z[(bits & 1) == 0] = float("-inf")
            lse[r:r + step] = torch.logsumexp(z, -1)
            y = torch.zeros_like(z)
            row = (s["targets"][r:r + step] != IGNORE).nonzero()[:, 0]
            col = s["targets"][r:r + step][row]
            y[row, col] = 1.0
            own_z = z[row, col]
            l = lse[r:r + step][row] - own_z
            l[own_z == float("-inf")] = float("inf")
            if e:
                l = (1 - e) * l + e * (lse[r:r + step][row] - z[row].mean(-1))
            loss[r + row] = l
            if c["train"]:
                y[z == float("-inf")] = 0.0
                live = torch.zeros(z.shape[0], 1, dtype=f, device=DEV)
                live[row, 0] = s["dloss"][r:r + step][row].to(f) * s["scale"]
                dz = (torch.softmax(z, -1) - (1 - e) * y - e / V) * live
                dx[r:r + step] = dz @ w
                dw += dz.t() @ x[r:r + step]
        return {"loss": loss, "lse": lse, "dx": dx, "dw": dw} if c["train"] else {"loss": loss, "lse": lse}
    if c["op"] == "swiglu":
        F = c["F"]
        x, wg, wu = s["x"].to(f), s["w"][:F].to(f), s["w"][F:].to(f)
        g, u = x @ wg.t(), x @ wu.t()
        a = g * torch.sigmoid(g)
        if not c["train"]:
            return {"h": a * u}
        dh = s["dh"].to(f)
        dg = dh * u * (torch.sigmoid(g) + a * (1.0 - torch.sigmoid(g)))
        du = dh * a
        return {"h": a * u, "dx": dg @ wg + du @ wu, "dw": torch.cat([dg.t() @ x, du.t() @ x])}
    x = s["x"].to(f)
    if s["delta"] is not None:
        x = x + s["delta"].to(f)
    w, dy = s["w"].to(f), s["dy"].to(f)
    mu = x.mean(-1, keepdim=True) if c["kind"] == "layer" else torch.zeros_like(x[:, :1])
    sd = torch.sqrt(((x - mu) ** 2).mean(-1, keepdim=True) + 1e-5)
    n = (x - mu) / sd
    gy = dy * w
    dx = gy - n * (gy * n).mean(-1, keepdim=True)
    if c["kind"] == "layer":
        dx = dx - gy.mean(-1, keepdim=True)
    dx = dx / sd
    got = {"dw": (dy * n).sum(0)}
    if s["dh"] is not None:
        dx, got["h"] = dx + s["dh"].to(f), x
    y = n * w
    if s["b"] is not None:
        y, got["db"] = y + s["b"].to(f), dy.sum(0)
    return {**got, "y": y, "dx": dx}
