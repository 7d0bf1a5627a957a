"""Differentiable wrappers of the native kernels for training.

``linear(x, w)`` computes x @ w^T with the tcgen05 GEMM on CUDA in forward
and backward (dX = dY @ W, dW = dY^T @ X, each expressed as the kernel's
x @ w^T form on transposed copies); on the CPU it is the fp32 torch statement.
"""
from __future__ import annotations

import torch
from torch.autograd.forward_ad import unpack_dual

from .. import ops


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        ctx.save_for_backward(x, w)
        return ops.linear(x, w)

    @staticmethod
    def backward(ctx, gy):
        x, w = ctx.saved_tensors
        gy = gy.contiguous().to(x.dtype)
        gx = gw = None
        if ctx.needs_input_grad[0]:
            padn = (-gy.shape[1]) % 8  # the output dim becomes the reduction dim (e.g. a 4-expert router)
            g2 = torch.nn.functional.pad(gy, (0, padn)) if padn else gy
            wt = torch.nn.functional.pad(w.t(), (0, padn)) if padn else w.t()
            gx = ops.linear(g2, wt.contiguous())                          # [M, K] = dY @ W
        if ctx.needs_input_grad[1]:
            pad = (-x.shape[0]) % 8  # the token dim becomes the reduction dim: keep rows 16-byte aligned
            xp = torch.nn.functional.pad(x, (0, 0, 0, pad)) if pad else x
            gp = torch.nn.functional.pad(gy, (0, 0, 0, pad)) if pad else gy
            gw = ops.linear(gp.t().contiguous(), xp.t().contiguous())     # [N, K] = dY^T @ X
        return gx, gw


def linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    if not x.is_cuda:
        return x @ w.t()
    shp = x.shape
    y = _Linear.apply(x.reshape(-1, shp[-1]).contiguous(), w)
    return y.reshape(*shp[:-1], w.shape[0])


class _FirstOnly(torch.autograd.Function):
    """A gradient as it is, tied to what it was computed from: differentiating it raises."""

    @staticmethod
    def forward(ctx, op, grad, *of):
        ctx.op = op
        return grad.view_as(grad)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError(f"{ctx.op} has first derivatives only: a gradient taken with create_graph=True cannot be "
                           "differentiated through it")


def _first_only(op):
    """Marks the backward of a Function whose gradients have no graph. (Without a mark their second
    derivatives would be left out of a sum in silence.)"""
    def mark(fn):
        def backward(ctx, *grads):
            with torch.no_grad():
                out = fn(ctx, *grads)
            if not torch.is_grad_enabled():
                return out
            of = [t for t in (*ctx.saved_tensors, *grads) if t is not None]
            return tuple(None if g is None else _FirstOnly.apply(op, g, *of) for g in out)
        return backward
    return mark


class _Norm(torch.autograd.Function):
    """y = norm(x (+ delta)) w (+ b) on the native kernels (``ops.norm_train``); with delta the sum
    h comes back too, and its gradient joins dx in the same pass."""

    @staticmethod
    def forward(ctx, x, delta, w, b, eps, kind):
        y, h, stats = ops.norm_train(x, w, b, eps, kind=kind, delta=delta)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(h, w, stats)
        ctx.kind, ctx.bias, ctx.summed, ctx.eps = kind, b is not None, delta is not None, eps
        return (y, h) if delta is not None else y

    @staticmethod
    def backward(ctx, gy, gh=None):
        h, w, stats = ctx.saved_tensors
        if gy is None:
            gy = torch.zeros_like(h)
        if torch.is_grad_enabled():
            dx, dw, db = _norm_grad(gy, h, w, ctx.eps, ctx.kind, gh)
        else:
            dx, dw, db = ops.norm_train_bwd(gy, h, w, stats, kind=ctx.kind, bias=ctx.bias, dh=gh)
        return dx, dx if ctx.summed else None, dw, db if ctx.bias else None, None, None


def _norm_grad(gy, h, w, eps, kind, gh):
    """(dx, dw, db) of a norm in plain operations on h, w and gy, for create_graph=True: a function
    of all three that differentiates on."""
    hf, g = h.float(), gy.float()
    d = hf - hf.mean(-1, keepdim=True) if kind == "layer" else hf
    r = torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + eps)
    n, a = d * r, g * w.float()
    dx = a - n * (a * n).mean(-1, keepdim=True)
    if kind == "layer":
        dx = dx - a.mean(-1, keepdim=True)
    dx = dx * r if gh is None else dx * r + gh.float()
    over_rows = lambda t: t.reshape(-1, t.shape[-1]).sum(0).to(w.dtype)  # noqa: E731
    return dx.to(h.dtype), over_rows(g * n), over_rows(g)


def _norm_native(x, w, delta=None, b=None):
    """Whether the kernels take this norm. The plain statement takes the rest: other types, gains and
    deltas that broadcast, and what torch.func or a forward-mode dual has to see through."""
    return (x.is_cuda and x.dim() > 0 and x.dtype in (torch.bfloat16, torch.float32)
            and w.dtype in (x.dtype, torch.float32) and w.shape == x.shape[-1:] and 0 < x.shape[-1] <= 16384
            and (delta is None or (delta.shape == x.shape and delta.dtype == x.dtype))
            and (b is None or (b.shape == w.shape and b.dtype == w.dtype))
            and not torch._C._are_functorch_transforms_active()
            and all(t is None or unpack_dual(t).tangent is None for t in (x, w, delta, b)))


def rmsnorm(x, w, eps):
    if _norm_native(x, w):
        return _Norm.apply(x, None, w, None, eps, "rms")
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps) * w.float()).to(x.dtype)


def add_rmsnorm(x, delta, w, eps):
    """(rmsnorm(h), h) with h = x + delta: the residual add and the norm that follows it."""
    if _norm_native(x, w, delta):
        return _Norm.apply(x, delta, w, None, eps, "rms")
    h = x + delta
    return rmsnorm(h, w, eps), h


def layernorm(x, w, b, eps):
    """LayerNorm with gain and (optional) bias over the last dimension."""
    if _norm_native(x, w, b=b):
        return _Norm.apply(x, None, w, b, eps, "layer")
    xf = x.float()
    mu = xf.mean(-1, keepdim=True)
    y = (xf - mu) * torch.rsqrt((xf - mu).pow(2).mean(-1, keepdim=True) + eps) * w.float()
    return (y if b is None else y + b.float()).to(x.dtype)


class _SwiGLU(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w):
        h, gu = ops.swiglu(x, w, save=True)
        ctx.save_for_backward(x, w, gu)
        return h

    @staticmethod
    @_first_only("swiglu")
    def backward(ctx, gh):
        x, w, gu = ctx.saved_tensors
        return ops.swiglu_bwd(x, w, gu, gh, ctx.needs_input_grad[0], ctx.needs_input_grad[1])


def swiglu(x, w):
    """silu(x Wg^T) * (x Wu^T) of x [..., K], w [2F, K] (gate rows first): one GEMM forward, the
    gradient from its fp32 projections."""
    if not x.is_cuda:
        z = x @ w.t()
        F = w.shape[0] // 2
        return torch.nn.functional.silu(z[..., :F]) * z[..., F:]
    if not (torch.is_grad_enabled() and (x.requires_grad or w.requires_grad)):
        return ops.swiglu(x, w)
    return _SwiGLU.apply(x, w)


class _LinearXent(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, targets, scale, smoothing, ignore_index, keep):
        loss, lse = ops.linear_xent(x, w, targets, scale, smoothing, ignore_index, keep)
        ctx.save_for_backward(x, w, targets, lse, keep)
        ctx.args = (scale, smoothing, ignore_index)
        return loss

    @staticmethod
    @_first_only("linear_xent")
    def backward(ctx, gl):
        x, w, targets, lse, keep = ctx.saved_tensors
        dx, dw = ops.linear_xent_bwd(x, w, targets, lse, gl, *ctx.args, keep=keep, need_dx=ctx.needs_input_grad[0],
                                     need_dw=ctx.needs_input_grad[1])
        return dx, dw, None, None, None, None, None


def linear_xent(x, w, targets, scale=1.0, smoothing=0.0, ignore_index=-100, keep=None):
    """Cross entropy [...] (fp32, row by row) of the logits scale * x w^T against ``targets`` [...],
    without the logits; ``keep`` restricts the vocabulary (see ``ops.linear_xent``)."""
    if x.is_cuda:
        return _LinearXent.apply(x, w, targets, scale, smoothing, ignore_index, keep)
    z = (x @ w.t()).float().reshape(-1, w.shape[0]) * scale
    if keep is not None:
        if smoothing:
            raise ValueError("linear_xent: label smoothing over a keep mask is not defined")
        bits = (keep[:, :, None] >> torch.arange(32, dtype=torch.int32, device=keep.device)) & 1
        z = z.masked_fill(bits.reshape(keep.shape[0], -1)[:, :w.shape[0]] == 0, float("-inf"))
    loss = torch.nn.functional.cross_entropy(z, targets.reshape(-1).long(), ignore_index=ignore_index,
                                             label_smoothing=smoothing, reduction="none")
    return loss.view(targets.shape)


def _attend_batch(q, k, v, scale):
    """Causal attention of a whole batch in one launch of the tcgen05 prefill kernel: K and V laid
    out as a paged cache (16-token blocks), heads narrower than 128 filled up with zeros.
    (out [B, T, H, D], lse fp32 [B, T, H])."""
    B, T, H, D = q.shape
    S, Hkv, dev = k.shape[1], k.shape[2], q.device
    nb, off = (S + 15) // 16, S - T
    fill = lambda x, t: torch.nn.functional.pad(x, (0, 128 - D, 0, 0, 0, t)) if t or D < 128 else x  # noqa: E731

    def paged(x):
        return fill(x, nb * 16 - S).reshape(B * nb, 16, Hkv, 128).transpose(1, 2).contiguous()

    tiles = [(b * T + t, min(128, T - t), b, off + min(T, t + 128)) for t in range((T - 1) // 128 * 128, -1, -128)
             for b in range(B)]   # longest first
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)  # noqa: E731
    out = torch.empty(B * T, H * 128, dtype=q.dtype, device=dev)
    lse = torch.empty(B * T, H, dtype=torch.float32, device=dev)
    ops.flash_prefill(fill(q, 0).reshape(B * T, H * 128), paged(k), paged(v),
                      torch.arange(B * nb, dtype=torch.int32, device=dev).view(B, nb),
                      torch.arange(B, dtype=torch.int32, device=dev).repeat_interleave(T),
                      torch.arange(off + 1, S + 1, dtype=torch.int32, device=dev).repeat(B), ints(tiles), H, scale,
                      out=out, lse=lse)
    return out.view(B, T, H, 128)[..., :D], lse.view(B, T, H)


class _Attention(torch.autograd.Function):
    """Causal attention of q [B, T, H, D] over k, v [B, S, Hkv, D].

    Forward: the repo's attention (on CUDA one launch of the tcgen05 FlashAttention kernel, on the
    CPU the fp32 statement per sequence), which also returns the natural-log sum of exponentials L
    of every row. Backward: ``ops.attention_bwd``, which recomputes the probabilities from L."""

    @staticmethod
    def forward(ctx, q, k, v, scale, lens):
        if q.is_cuda and q.numel():
            out, lse = _attend_batch(q, k, v, scale)
        else:
            from ..parallel.ring_attention import attend
            got = [attend(q[b], k[b], v[b], scale, causal=True) for b in range(q.shape[0])]
            out, lse = (torch.stack(t) for t in zip(*got)) if got else (q.float(), q[..., 0].float())
        ctx.save_for_backward(q, k, v, out, lse, lens)
        ctx.scale = scale
        return out.to(q.dtype)

    @staticmethod
    @_first_only("attention")
    def backward(ctx, go):
        q, k, v, out, lse, lens = ctx.saved_tensors
        dq, dk, dv = ops.attention_bwd(q, k, v, out, lse, go, ctx.scale, causal=True, lens=lens)
        return dq, dk, dv, None, None


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, lens=None) -> torch.Tensor:
    """Differentiable causal attention, q [B, T, H, D], k / v [B, S, Hkv, D] -> [B, T, H, D]: the
    queries are the last T of S >= T tokens.

    ``lens`` int32 [B]: valid tokens of right-padded sequences (T == S). Their rows do not depend on it
    (a causal row sees no padding); the gradient leaves the padding out, in work and in value."""
    if lens is not None and k.shape[1] != q.shape[1]:
        raise ValueError("attention: lens needs as many queries as keys")
    if q.is_cuda and (k.shape[1] < q.shape[1] or v.shape != k.shape):
        raise ValueError("attention: k and v [B, S, Hkv, D] need at least as many keys as q has queries")
    return _Attention.apply(q, k, v, scale, lens)
