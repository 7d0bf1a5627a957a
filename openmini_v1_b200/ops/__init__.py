"""Operator layer.

CUDA tensors run the hand-written sm_100a kernels of ``openmini_v1_b200._C``
(no library GEMM, no Triton, no fallback: a missing extension raises).
CPU tensors run the fp32 statements in :mod:`.reference`, which double as the
numerics oracle.
"""
from __future__ import annotations

import threading

import torch
import torch.distributed as dist

from .. import _native
from . import reference as ref

__all__ = [
    "DeviceContext", "ctx", "linear", "rmsnorm", "layernorm", "silu_mul", "gelu", "softmax",
    "embedding", "rope_kv", "kv_write", "paged_attention", "sample", "repetition_penalty",
    "check_status", "attention_bwd", "swiglu", "swiglu_bwd", "linear_xent", "linear_xent_bwd", "norm_train",
    "norm_train_bwd",
]


class DeviceContext:
    """Per-device scratch owned by the op layer: a status word that kernels set
    on a bounded-wait timeout (after which other waits stop early, so later
    results may be incomplete) or a bounds violation (which touches no other
    call), and growable fp32 workspaces for split-K GEMM partials and split-KV
    attention partials."""

    def __init__(self, device: torch.device):
        self.device = device
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self._ws = {}
        self.frozen = False  # set while capturing a CUDA graph: no reallocation allowed

    def semaphores(self) -> torch.Tensor:
        """Zeroed int32 tile counters of the in-kernel split-K reduction (every kernel that
        uses them leaves them zeroed again)."""
        s = self._ws.get("__sem")
        if s is None:
            if self.frozen:
                raise RuntimeError("semaphores first requested during graph capture")
            s = torch.zeros(1 << 16, dtype=torch.int32, device=self.device)
            self._ws["__sem"] = s
        return s

    def workspace(self, name: str, numel: int) -> torch.Tensor:
        buf = self._ws.get(name)
        if buf is None or buf.numel() < numel:
            if self.frozen:
                raise RuntimeError(f"workspace {name!r} too small during graph capture ({numel})")
            buf = torch.empty(max(numel, 1 << 16), dtype=torch.float32, device=self.device)
            self._ws[name] = buf
        return buf


_ctx_lock = threading.Lock()
_ctxs: dict = {}


def ctx(device) -> DeviceContext:
    device = torch.device(device)
    if device.type == "cuda" and device.index is None:
        device = torch.device("cuda", torch.cuda.current_device())
    key = str(device)
    c = _ctxs.get(key)
    if c is None:
        with _ctx_lock:
            c = _ctxs.get(key)
            if c is None:
                c = DeviceContext(device)
                _ctxs[key] = c
    return c


def status_text(v: int) -> str:
    """What a device status word says."""
    waits = {1: "a wait for a filled stage", 2: "a wait for a free stage", 3: "a wait for an accumulator",
             4: "a wait for a peer"}
    said = [f"{waits[v & 255]} gave up"] if v & 255 in waits else []
    if 5 in (v & 255, v >> 8):
        said.append("an index in the data was out of range")
    return "; ".join(said)


def check_status(device=None, across=False, group=None):
    """Raise if any kernel on ``device`` recorded an error (timeout / bounds). With ``across`` the
    ranks of ``group`` (None: all) call this together, and all of them raise if one has an error."""
    if device is None:
        device = torch.device("cuda", torch.cuda.current_device())
    c = ctx(device)
    if across:
        worst = c.status.clone()
        dist.all_reduce(worst, op=dist.ReduceOp.MAX, group=group)
        worst = int(worst.item())
    v = int(c.status.item())
    if v != 0:
        c.status.zero_()
        raise RuntimeError(f"device kernel reported error status {v} ({status_text(v)}) on {device}")
    if across and worst != 0:
        raise RuntimeError(f"device kernel of another rank reported error status {worst} ({status_text(worst)})")


# Split-K scratch: sized for the largest decode GEMM partial (splits x M x N fp32).
GEMM_WS_FLOATS = 64 << 20


def linear(x: torch.Tensor, w, out: torch.Tensor | None = None, resid: torch.Tensor | None = None,
           peer: list | None = None):
    """y = x @ w^T (+ resid). ``w`` is a bf16 [N, K] tensor or a quantised weight object.

    ``peer`` (CUDA only) = [partials byte offset, rows per rank, this rank, base pointer of
    every rank]: output row m is stored into rank m // rows_per_rank's symmetric buffer
    (slot of this rank) over NVLink and the kernel publishes the epoch when done; ``out``
    then only supplies the row stride."""
    if not isinstance(w, torch.Tensor):
        if peer is not None:
            return w.linear(x, out=out, resid=resid, peer=peer)
        return w.linear(x, out=out, resid=resid)
    if not x.is_cuda:
        y = ref.linear(x, w, resid)
        if out is not None:
            out.copy_(y.reshape(out.shape))
            return out
        return y
    x2 = x.reshape(-1, x.shape[-1])
    if x2.stride(-1) != 1:
        x2 = x2.contiguous()
    M, N = x2.shape[0], w.shape[0]
    if out is None:
        out = torch.empty(*x.shape[:-1], N, dtype=x.dtype, device=x.device)
    o2 = out.view(-1, N)
    if M == 0:
        return out
    c = ctx(x.device)
    ws = c.workspace("gemm", GEMM_WS_FLOATS)
    r2 = resid.reshape(-1, N) if resid is not None else None
    if peer is not None:
        _native.C().gemm(x2, w, o2, r2, ws, c.status, peer=peer)
    else:
        _native.C().gemm(x2, w, o2, r2, ws, c.status)
    return out


def rmsnorm(x, w, eps, out=None, delta=None):
    """rmsnorm(x [+= delta]) * w. With ``delta`` the residual x is updated in place."""
    if not x.is_cuda:
        y = ref.rmsnorm(x, w, eps, delta)
        if out is not None:
            out.copy_(y)
            return out
        return y
    if out is None:
        out = torch.empty_like(x)
    _native.C().rmsnorm(x, delta, w, out, float(eps))
    return out


def layernorm(x, w, b, eps, out=None):
    if not x.is_cuda:
        return ref.layernorm(x, w, b, eps)
    out = torch.empty_like(x) if out is None else out
    _native.C().layernorm(x.contiguous(), w, b, out, float(eps))
    return out


def silu_mul(gu, out=None):
    if not gu.is_cuda:
        return ref.silu_mul(gu)
    F = gu.shape[-1] // 2
    out = torch.empty(*gu.shape[:-1], F, dtype=gu.dtype, device=gu.device) if out is None else out
    _native.C().silu_mul(gu.contiguous(), out)
    return out


def gelu(x):
    if not x.is_cuda:
        return ref.gelu(x)
    y = torch.empty_like(x)
    _native.C().gelu(x.contiguous(), y)
    return y


def softmax(x, scale=1.0):
    if not x.is_cuda:
        return ref.softmax(x, scale)
    y = torch.empty(x.shape, dtype=torch.float32, device=x.device)
    _native.C().softmax(x.contiguous(), y, float(scale))
    return y


def embedding(ids, table, out=None):
    if not ids.is_cuda:
        return ref.embedding(ids, table)
    out = torch.empty(ids.numel(), table.shape[1], dtype=table.dtype, device=table.device) if out is None else out
    _native.C().embedding(ids.to(torch.int32), table, out, ctx(ids.device).status)
    return out


def rope_kv(qkv, positions, slots, k_cache, v_cache, inv_freq, Hq, Hkv, D, mode=0):
    if not qkv.is_cuda:
        return ref.rope_kv(qkv, positions, slots, k_cache, v_cache, inv_freq, Hq, Hkv, D, mode)
    _native.C().rope_kv(qkv, positions, slots, k_cache, v_cache, inv_freq, Hq, Hkv, D, mode,
                        ctx(qkv.device).status)


def kv_write(k, v, slots, k_cache, v_cache):
    if not k.is_cuda:
        return ref.kv_write(k, v, slots, k_cache, v_cache)
    _native.C().kv_write(k, v, slots, k_cache, v_cache)


def mla_decode(q, cache, block_tables, row_seq, row_ctx, max_ctx, scale, out=None):
    """Latent attention (absorbed MLA) of q [rows, H, 576] over the paged latent cache
    [blocks, 16, 576] -> [rows, H, 512] (see ``csrc/attn/mla.cu``)."""
    if not q.is_cuda:
        o = ref.mla_decode(q, cache, block_tables, row_seq, row_ctx, scale)
        if out is not None:
            out.copy_(o)
            return out
        return o
    rows, H = q.shape[0], q.shape[1]
    if out is None:
        out = torch.empty(rows, H, 512, dtype=q.dtype, device=q.device)
    c = ctx(q.device)
    ws = c.workspace("mla", _native.C().mla_workspace(rows, H, int(max_ctx)))
    _native.C().mla_decode(q.contiguous(), cache, block_tables, row_seq, row_ctx, out, ws, int(max_ctx),
                           float(scale), c.status)
    return out


def paged_attention(q, k_cache, v_cache, block_tables, row_seq, row_ctx, Hq, scale, max_ctx, out=None, impl=None):
    """Attention of query rows over the paged cache. ``max_ctx`` bounds the split count.

    On the GPU, head_dim 128 with <= 16 query heads per KV head runs the
    tensor-core kernel ("tc"); other shapes run the CUDA-core kernel ("simt")."""
    rows = row_seq.shape[0]
    D = k_cache.shape[3]
    if not q.is_cuda:
        o = ref.paged_attention(q, k_cache, v_cache, block_tables, row_seq, row_ctx, Hq, scale)
        if out is not None:
            out.copy_(o.reshape(out.shape))
            return out
        return o.reshape(rows, Hq * D)
    if out is None:
        out = torch.empty(rows, Hq * D, dtype=q.dtype, device=q.device)
    c = ctx(q.device)
    need = _native.C().paged_attention_workspace(rows, Hq, D, max_ctx)
    ws = c.workspace("attn", need)
    if impl is None:
        impl = "tc" if D == 128 and Hq // k_cache.shape[1] <= 16 else "simt"
    fn = _native.C().paged_attention_tc if impl == "tc" else _native.C().paged_attention
    fn(q.reshape(rows, -1), k_cache, v_cache, block_tables, row_seq, row_ctx, out.view(rows, -1), ws, Hq,
       int(max_ctx), float(scale), c.status)
    return out


def flash_prefill(q, k_cache, v_cache, block_tables, row_seq, row_ctx, tiles, Hq, scale, out=None, lse=None):
    """Causal prefill attention of query tiles (consecutive rows of one sequence) over the
    paged cache; on the GPU the tcgen05 FlashAttention kernel (head_dim 128). With ``lse``
    (fp32 [T, Hq]) the natural-log sum-exp of every row's scaled scores is written too."""
    T = row_seq.shape[0]
    D = k_cache.shape[3]
    if not q.is_cuda:
        o = ref.paged_attention(q, k_cache, v_cache, block_tables, row_seq, row_ctx, Hq, scale)
        if out is not None:
            out.copy_(o.reshape(out.shape))
            return out
        return o.reshape(T, Hq * D)
    if out is None:
        out = torch.empty(T, Hq * D, dtype=q.dtype, device=q.device)
    c = ctx(q.device)
    _native.C().flash_prefill(q.reshape(T, -1), k_cache, v_cache, block_tables, row_ctx, tiles, out.view(T, -1),
                              Hq, float(scale), c.status, lse=lse)
    return out


def sample(logits, temperature, top_p, top_k, rng, want_mask=False):
    """Returns (tokens int32, logprob fp32, packed keep mask int32 [B, ceil(V/32)] or None).

    Each row's random draw depends only on its request's (seed, offset): the same
    request samples the same token whatever the batch or the tensor-parallel split."""
    B, V = logits.shape
    if not logits.is_cuda:
        t, lp, m = ref.sample(logits, temperature, top_p, top_k, rng)
        return t, lp, (ref.pack_mask(m) if want_mask else None)
    tok = torch.empty(B, dtype=torch.int32, device=logits.device)
    lp = torch.empty(B, dtype=torch.float32, device=logits.device)
    mask = torch.empty(B, (V + 31) // 32, dtype=torch.int32, device=logits.device) if want_mask else None
    _native.C().sample(logits, temperature, top_p, top_k, rng, tok, lp, mask)
    return tok, lp, mask


def repetition_penalty(logits, prev, penalty):
    if not logits.is_cuda:
        return ref.repetition_penalty(logits, prev, penalty)
    _native.C().repetition_penalty(logits, prev.to(torch.int32).contiguous(), penalty)
    return logits


# ------------------------------------------------------------------ training operators
# The native entries take tensors as they are (a layout that a TMA copy cannot read is copied) and
# allocate results and scratch on the current stream, so calls on different streams never share any.

def _same_device(op, *tensors):
    d = tensors[0].device
    for t in tensors:
        if t is not None and t.device != d:
            raise ValueError(f"{op}: all tensors must be on {d}")


def attention_bwd(q, k, v, out, lse, dout, scale, causal=True, lens=None):
    """Gradient (dq, dk, dv) of attention from what its forward kept: q, out, dout [B, T, H, D],
    k, v [B, S, Hkv, D], ``lse`` fp32 [B, T, H] (natural log of the sum of exp of the scaled scores;
    -inf for a row without a visible key, whose gradient is 0).

    ``causal`` masks are aligned to the last key (query i sees keys <= i + S - T). ``lens`` int32 [B]
    (T == S) is the number of valid tokens of right-padded sequences: padding takes no gradient,
    whatever it holds. head_dim: a multiple of 8 up to 128."""
    _same_device("attention_bwd", q, k, v, out, lse, dout, lens)
    if not q.is_cuda:
        return ref.attention_bwd(q, k, v, out, lse, dout, scale, causal, lens)
    if v.shape != k.shape or out.shape != q.shape or dout.shape != q.shape:
        raise ValueError("attention_bwd: q, out, dout [B, T, H, D] and k, v [B, S, Hkv, D]")
    return _native.C().attention_bwd(q, k, v, out, lse, dout, lens, scale, causal, ctx(q.device).status)


def swiglu(x, w, save=False):
    """silu(x Wg^T) * (x Wu^T) of x [..., K] and w [2F, K] (gate rows first) -> [..., F]. With
    ``save`` also the fp32 projections that :func:`swiglu_bwd` reads (on the GPU their rows and h's
    are a multiple of 8 elements apart, so h of an odd F is a strided view)."""
    _same_device("swiglu", x, w)
    if w.dim() != 2 or w.shape[0] % 2 or w.shape[1] != x.shape[-1]:
        raise ValueError("swiglu: w must be [2F, K]")
    if not x.is_cuda:
        return ref.swiglu(x, w, save)
    h, gu = _native.C().swiglu(x, w, save, ctx(x.device).status)
    return (h, gu) if save else h


def swiglu_bwd(x, w, gu, dh, need_dx=True, need_dw=True):
    """Gradient (dx, dw) of :func:`swiglu` from its saved projections and dh [..., F]."""
    _same_device("swiglu_bwd", x, w, gu, dh)
    if not x.is_cuda:
        return ref.swiglu_bwd(x, w, gu, dh, need_dx, need_dw)
    return _native.C().swiglu_bwd(x, w, gu, dh, need_dx, need_dw, ctx(x.device).status)


def _xent_args(op, x, w, targets, smoothing, keep):
    _same_device(op, x, w, targets, keep)
    if w.dim() != 2 or w.shape[1] != x.shape[-1] or targets.shape != x.shape[:-1]:
        raise ValueError(f"{op}: x [..., K], w [V, K], targets [...]")
    if targets.is_floating_point() or targets.dtype == torch.bool:
        raise ValueError(f"{op}: targets must be integers")
    if not 0.0 <= smoothing < 1.0:
        raise ValueError(f"{op}: label smoothing must be in [0, 1)")
    if keep is not None and smoothing:
        raise ValueError(f"{op}: label smoothing over a keep mask is not defined")


def linear_xent(x, w, targets, scale=1.0, smoothing=0.0, ignore_index=-100, keep=None):
    """Cross entropy of the logits scale * x w^T, which are never stored: (loss, lse) fp32 [...] of
    x [..., K], w [V, K] and targets [...].

    Rows whose target is ``ignore_index`` have loss 0. ``keep``: packed mask int32 [rows, ceil(V / 32)]
    as :func:`sample` returns it; columns outside it have probability 0 (a target outside it has an
    infinite loss, an empty row lse = -inf). Other targets outside [0, V) count as ignored and set
    the device status."""
    _xent_args("linear_xent", x, w, targets, smoothing, keep)
    if not x.is_cuda:
        return ref.linear_xent(x, w, targets, scale, smoothing, ignore_index, keep)
    return _native.C().linear_xent(x, w, targets, keep, scale, smoothing, ignore_index, ctx(x.device).status)


def linear_xent_bwd(x, w, targets, lse, dloss, scale=1.0, smoothing=0.0, ignore_index=-100, keep=None, need_dx=True,
                    need_dw=True):
    """Gradient (dx, dw) of :func:`linear_xent`; ``dloss`` [...] is the loss's gradient row by row."""
    _xent_args("linear_xent_bwd", x, w, targets, smoothing, keep)
    _same_device("linear_xent_bwd", x, lse, dloss)
    if not x.is_cuda:
        return ref.linear_xent_bwd(x, w, targets, lse, dloss, scale, smoothing, ignore_index, keep, need_dx, need_dw)
    return _native.C().linear_xent_bwd(x, w, targets, keep, scale, smoothing, ignore_index, lse, dloss, need_dx,
                                       need_dw, ctx(x.device).status)


def _norm_kind(kind, bias):
    if kind not in ("rms", "layer"):
        raise ValueError(f"norm kind {kind!r}: 'rms' or 'layer'")
    if kind == "rms" and bias:
        raise ValueError("RMSNorm takes no bias")
    return kind == "layer"


def norm_train(x, w, b=None, eps=1e-5, kind="rms", delta=None):
    """(y, h, stats): y = norm(h) * w (+ b) with h = x (+ delta, rounded to x's type), and the rows'
    fp32 (mean, 1 / std) that :func:`norm_train_bwd` reads. x bf16 (w, b bf16 or fp32) or fp32."""
    layer = _norm_kind(kind, b is not None)
    _same_device("norm_train", x, w, b, delta)
    if delta is not None and (delta.shape != x.shape or delta.dtype != x.dtype):
        raise ValueError("norm_train: delta must be like x")
    if not x.is_cuda:
        return ref.norm_train(x, w, b, eps, kind, delta)
    return _native.C().norm_train(x, w, b, eps, layer, delta, ctx(x.device).status)


def norm_train_bwd(dy, h, w, stats, kind="rms", bias=False, dh=None):
    """(dx, dw, db) of :func:`norm_train`: ``dh`` is the gradient that h itself receives (the residual
    stream's), added to dx; dw, db have w's type; db is None without ``bias``."""
    layer = _norm_kind(kind, bias)
    _same_device("norm_train_bwd", dy, h, w, stats, dh)
    if not h.is_cuda:
        return ref.norm_train_bwd(dy, h, w, stats, kind, bias, dh)
    return _native.C().norm_train_bwd(dy, h, w, stats, layer, bias, dh, ctx(h.device).status)
