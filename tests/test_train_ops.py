"""The training operators (attention backward, gated feed-forward projection, vocabulary cross
entropy, norms) against 64-bit forward definitions differentiated by autograd, on the CPU
(reference statements) and on the GPU (kernels).

Tolerances are bounds, entry by entry. U = 2^-9 is the rounding of a 16-bit value. A result that
is stored in 16 bits and was summed from terms t_i of which each went through 16 bits once is off
by at most U |result| + U sum |t_i|; both are doubled for the exponential's and the fp32 sums'
own errors. E = 2^-20 stands for fp32 sums of up to a few thousand terms (K 2^-24 at the worst)."""
import math

import pytest
import torch

from openmini_v1_b200 import ops

U, E = 2.0 ** -9, 2.0 ** -20
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]
on_devices = pytest.mark.parametrize("dev", DEVICES)


def gen(dev, seed):
    return torch.Generator(device=dev).manual_seed(seed)


def randn(g, *shape, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(*shape, generator=g, device=g.device) * std).to(dtype)


def close(got, want, tol, what):
    got = got.double()
    assert got.shape == want.shape, what
    assert torch.isfinite(got).all(), f"{what}: not finite"
    d = (got - want).abs()
    bad = d > tol
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((d / tol).max()):.2f} x tol"


# ----------------------------------------------------------------------------- attention
def visible(B, T, S, causal, lens, dev):
    m = torch.ones(B, 1, T, S, dtype=torch.bool, device=dev)
    if causal:
        m = m.tril(S - T)
    if lens is not None:
        n = torch.tensor(lens, device=dev).view(B, 1, 1, 1)
        m = m & (torch.arange(T, device=dev).view(1, 1, T, 1) < n) & (torch.arange(S, device=dev).view(1, 1, 1, S) < n)
    return m


def attention64(q, k, v, scale, mask):
    """(out [B, T, H, D], lse [B, T, H]) in 64 bits; rows that see no key: 0 and -inf."""
    G = q.shape[2] // k.shape[2]
    kk, vv = k.repeat_interleave(G, 2), v.repeat_interleave(G, 2)
    s = (torch.einsum("bqhd,bkhd->bhqk", q, kk) * scale).masked_fill(~mask, -1e300)
    p = torch.softmax(s, -1) * mask
    lse = torch.logsumexp(s, -1).masked_fill(~mask.any(-1), float("-inf"))
    return torch.einsum("bhqk,bkhd->bqhd", p, vv), lse.transpose(1, 2)


def attention_case(dev, B, T, S, H, Hkv, D, causal, lens, seed=0, std=1.0):
    g = gen(dev, seed)
    q, k, v, do = (randn(g, *s, std=std) for s in ((B, T, H, D), (B, S, Hkv, D), (B, S, Hkv, D), (B, T, H, D)))
    scale = 1 / math.sqrt(D)
    mask = visible(B, T, S, causal, lens, dev)
    q6, k6, v6 = (t.double().requires_grad_(True) for t in (q, k, v))
    o6, lse6 = attention64(q6, k6, v6, scale, mask)
    rows = mask.any(-1).transpose(1, 2)[..., None]
    d6 = do.double() * rows
    (o6 * d6).sum().backward()
    G = H // Hkv
    with torch.no_grad():   # magnitudes of the summed terms
        kk, vv = k6.repeat_interleave(G, 2), v6.repeat_interleave(G, 2)
        s = torch.einsum("bqhd,bkhd->bhqk", q6, kk) * scale
        p = torch.exp(s - lse6.transpose(1, 2)[..., None].clamp_min(-1e30)) * mask
        dp = torch.einsum("bqhd,bkhd->bhqk", d6, vv)
        delta = (d6 * o6).sum(-1).transpose(1, 2)[..., None]
        ds = (p * (dp - delta)).abs()
        big = torch.einsum("bqhd,bkhd->bhqk", d6.abs(), vv.abs())
        dlt = (d6 * o6).abs().sum(-1).transpose(1, 2)[..., None]
        # dS: its own rounding, the rounding of out in delta, fp32 sums (also in the exponent)
        e_ds = 2 * U * ds + U * p * dlt + E * p * (big + dlt) + 16 * E * ds
        tq = torch.einsum("bhqk,bkhd->bqhd", e_ds, kk.abs()) * scale + 2 * U * q6.grad.abs()
        tk = torch.einsum("bhqk,bqhd->bkhd", e_ds, q6.abs()) * scale
        tv = torch.einsum("bhqk,bqhd->bkhd", 2 * U * p, d6.abs())
        tk = tk.view(B, S, Hkv, G, D).sum(3) + 2 * U * k6.grad.abs()
        tv = tv.view(B, S, Hkv, G, D).sum(3) + 2 * U * v6.grad.abs()
    return dict(q=q, k=k, v=v, do=do, out=o6.detach().to(q.dtype), lse=lse6.detach().float().contiguous(),
                scale=scale, lens=None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev),
                want=(q6.grad, k6.grad, v6.grad), tol=tuple(t + 1e-9 for t in (tq, tk, tv)))


def check_attention(c, causal, **over):
    a = {**c, **over}
    got = ops.attention_bwd(a["q"], a["k"], a["v"], a["out"], a["lse"], a["do"], a["scale"], causal=causal,
                            lens=a["lens"])
    for name, g, w, t in zip(("dq", "dk", "dv"), got, c["want"], c["tol"]):
        close(g, w, t, name)
    return got


ATTENTION = [
    # B, T, S, H, Hkv, D, causal, lens
    (1, 1, 1, 1, 1, 64, True, None),
    (2, 1, 77, 4, 2, 128, True, None),         # one query over a prefix
    (1, 2, 2, 2, 1, 8, True, None),
    (2, 63, 63, 4, 2, 64, True, [63, 1]),
    (1, 65, 65, 5, 1, 128, True, None),
    (3, 128, 128, 8, 2, 128, True, [0, 100, 128]),
    (1, 129, 257, 2, 2, 128, True, None),
    (1, 200, 77, 3, 1, 64, True, None),        # rows 0 .. 122 see nothing
    (2, 191, 191, 6, 3, 80, False, None),
    (2, 130, 130, 10, 2, 96, True, [130, 67]),
    (2, 130, 130, 2, 2, 32, False, [64, 128]),
    (1, 70, 300, 2, 1, 128, False, None),
    (1, 520, 520, 8, 1, 128, True, None),
]


@on_devices
@pytest.mark.parametrize("shape", ATTENTION, ids=str)
def test_attention_bwd(dev, shape):
    B, T, S, H, Hkv, D, causal, lens = shape
    check_attention(attention_case(dev, B, T, S, H, Hkv, D, causal, lens), causal)


@on_devices
def test_attention_bwd_large_scores(dev):
    """Scores of a few hundred: a row's probability sits on one key."""
    check_attention(attention_case(dev, 1, 96, 96, 2, 2, 64, True, None, std=6.0), True)


@on_devices
def test_attention_bwd_ignores_padding_contents(dev):
    c = attention_case(dev, 2, 100, 100, 4, 2, 64, True, [100, 37])
    dirty = {}
    for n in ("q", "k", "v", "do", "out", "lse"):
        t = c[n].clone()
        t[1, 37:] = float("nan") if n != "k" else float("inf")
        dirty[n] = t
    check_attention(c, True, **dirty)
    clean = check_attention(c, True)
    assert all(float(g[1, 37:].abs().max()) == 0.0 for g in clean)


@on_devices
def test_attention_bwd_strided_inputs(dev):
    """q, k, v as views of one projection, dout expanded over the batch."""
    B, T, H, Hkv, D = 2, 90, 4, 2, 64
    c = attention_case(dev, B, T, T, H, Hkv, D, True, None)
    x = torch.cat([c["q"].flatten(2), c["k"].flatten(2), c["v"].flatten(2)], 2)
    q, k, v = x.split([H * D, Hkv * D, Hkv * D], 2)
    q, k, v = q.view(B, T, H, D), k.view(B, T, Hkv, D), v.view(B, T, Hkv, D)
    a = check_attention(c, True)
    b = check_attention(c, True, q=q, k=k, v=v, out=c["out"].transpose(1, 2).contiguous().transpose(1, 2))
    assert all(torch.equal(s, t) for s, t in zip(a, b))
    one = c["do"][:1].expand(B, T, H, D)
    wide = ops.attention_bwd(c["q"], c["k"], c["v"], c["out"], c["lse"], one, c["scale"])
    flat = ops.attention_bwd(c["q"], c["k"], c["v"], c["out"], c["lse"], one.contiguous(), c["scale"])
    assert all(torch.equal(s, t) for s, t in zip(wide, flat))


@on_devices
def test_attention_bwd_refusals(dev):
    c = attention_case(dev, 1, 8, 8, 2, 2, 64, True, None)
    args = [c[n] for n in ("q", "k", "v", "out", "lse", "do")]
    lens = torch.tensor([4], dtype=torch.int32, device=dev)
    with pytest.raises((ValueError, RuntimeError)):
        ops.attention_bwd(args[0], args[1][:, :4], args[2][:, :4], *args[3:], c["scale"], lens=lens)
    if dev == "cpu":
        return
    with pytest.raises(RuntimeError, match="head_dim"):
        ops.attention_bwd(*[t[..., :60].contiguous() if t.dim() == 4 else t for t in args], c["scale"])
    with pytest.raises(RuntimeError, match="bf16"):
        ops.attention_bwd(*[t.half() if t.dim() == 4 else t for t in args], c["scale"])
    with pytest.raises(RuntimeError, match="multiple of KV heads"):
        ops.attention_bwd(args[0], args[1].repeat(1, 1, 2, 1)[:, :, :3], args[2].repeat(1, 1, 2, 1)[:, :, :3],
                          *args[3:], c["scale"])
    with pytest.raises(ValueError):
        ops.attention_bwd(args[0], args[1], args[2][:, :4], *args[3:], c["scale"])
    with pytest.raises(ValueError, match="must be on"):
        ops.attention_bwd(args[0], args[1].cpu(), *args[2:], c["scale"])


# ----------------------------------------------------------------------------- gated projection
def swiglu_case(dev, M, K, F, seed=0):
    g = gen(dev, seed)
    x, w, dh = randn(g, M, K), randn(g, 2 * F, K, std=1 / math.sqrt(K)), randn(g, M, F)
    x6, w6 = x.double().requires_grad_(True), w.double().requires_grad_(True)
    z = x6 @ w6.t()
    gg, uu = z[:, :F], z[:, F:]
    h = torch.nn.functional.silu(gg) * uu
    (h * dh.double()).sum().backward()
    with torch.no_grad():
        d, s = dh.double().abs(), torch.sigmoid(gg)
        zsum = x6.abs() @ w6.abs().t()
        th = 2 * U * h.abs() + E * (1.1 * zsum[:, :F] * uu.abs() + gg.abs() * zsum[:, F:]) + 1e-9
        dg, du = d * (uu * s * (1 + gg * (1 - s))).abs(), d * (gg * s).abs()
        # rounded g and u (|d2 silu| <= 0.5, |d silu| <= 1.1), the rounding of dg and du themselves
        e = torch.cat([3 * U * dg + U * d * uu.abs() * gg.abs() * 0.5, 3 * U * du + U * d * 1.1 * gg.abs()], 1)
        tx = e @ w6.abs() + 2 * U * x6.grad.abs() + 1e-9
        tw = e.t() @ x6.abs() + 2 * U * w6.grad.abs() + 1e-9
    return x, w, dh, (h.detach(), x6.grad, w6.grad), (th, tx, tw)


SWIGLU = [(1, 8, 1), (1, 256, 700), (3, 64, 33), (127, 200, 688), (130, 72, 129), (301, 256, 1376), (1000, 64, 40),
          (2000, 136, 1001)]


@on_devices
@pytest.mark.parametrize("M,K,F", SWIGLU)
def test_swiglu(dev, M, K, F):
    x, w, dh, want, tol = swiglu_case(dev, M, K, F)
    h, gu = ops.swiglu(x, w, save=True)
    assert torch.equal(h, ops.swiglu(x, w))
    dx, dw = ops.swiglu_bwd(x, w, gu, dh)
    for name, g, a, t in zip(("h", "dx", "dw"), (h, dx, dw), want, tol):
        close(g, a, t, name)
    assert ops.swiglu_bwd(x, w, gu, dh, need_dx=False)[0] is None
    assert torch.equal(ops.swiglu_bwd(x, w, gu, dh, need_dw=False)[0], dx)


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,F", [(2600, 72, 1100), (2700, 200, 1104), (4100, 64, 4001)])
def test_swiglu_many_tiles(M, K, F):
    """Enough tiles for the CTA-pair GEMM, whole and ragged ones, rows on and off 16-byte boundaries."""
    x, w, dh, want, tol = swiglu_case("cuda", M, K, F)
    h, gu = ops.swiglu(x, w, save=True)
    dx, dw = ops.swiglu_bwd(x, w, gu, dh)
    for name, g, a, t in zip(("h", "dx", "dw"), (h, dx, dw), want, tol):
        close(g, a, t, name)
    assert torch.equal(ops.swiglu(x, w), h)
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("c", [dict(M=2049, K=136, V=4100, smoothing=0.1), dict(M=1500, K=4096, V=6500, scale=1.2),
                               dict(M=700, K=72, V=9000, keep=0.1)], ids=str)
def test_linear_xent_many_tiles(c):
    check_xent(xent_case("cuda", **c))
    ops.check_status()


@on_devices
def test_swiglu_extreme_gates(dev):
    """Gates of +-1000: the activation saturates to the product or to 0 without NaN."""
    x = torch.ones(2, 8, dtype=torch.bfloat16, device=dev)
    w = torch.zeros(4, 8, dtype=torch.bfloat16, device=dev)
    w[0, 0], w[1, 0], w[2:, 0] = 1000.0, -1000.0, 3.0
    h, gu = ops.swiglu(x, w, save=True)
    assert torch.equal(h.cpu(), torch.tensor([[3000.0, 0.0]] * 2).to(torch.bfloat16).cpu())
    dx, dw = ops.swiglu_bwd(x, w, gu, torch.ones_like(h))
    assert torch.isfinite(dx).all() and torch.isfinite(dw).all()
    assert abs(float(dw[0, 0]) - 6.0) < 6 * 2 * U and float(dw[1].abs().max()) == 0.0


@on_devices
def test_swiglu_empty_strided_and_refusals(dev):
    x, w, dh, want, tol = swiglu_case(dev, 6, 64, 24)
    assert ops.swiglu(x[:0], w).shape == (0, 24)
    h0, gu0 = ops.swiglu(x[:0], w, save=True)
    dx, dw = ops.swiglu_bwd(x[:0], w, gu0, dh[:0])
    assert dx.shape == (0, 64) and float(dw.abs().max()) == 0.0
    wide = torch.zeros(6, 100, dtype=x.dtype, device=dev)
    wide[:, 3:67] = x
    close(ops.swiglu(wide[:, 3:67], w), want[0], tol[0], "h of an unaligned view")
    close(ops.swiglu(x.view(2, 3, 64), w).view(6, 24), want[0], tol[0], "h of a batch")
    with pytest.raises((ValueError, RuntimeError)):
        ops.swiglu(x, w[:, :32])
    if dev == "cuda":
        with pytest.raises(RuntimeError, match="multiple of 8"):
            ops.swiglu(x[:, :60], w[:, :60])
        with pytest.raises(RuntimeError, match="bf16"):
            ops.swiglu(x.float(), w.float())
        with pytest.raises(ValueError):
            ops.swiglu(x, w[:47])


# ----------------------------------------------------------------------------- cross entropy
def words_of(mask):
    M, V = mask.shape
    n = (V + 31) // 32
    full = torch.zeros(M, n * 32, dtype=torch.int64, device=mask.device)
    full[:, :V] = mask
    w = (full.view(M, n, 32) << torch.arange(32, device=mask.device)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def xent_case(dev, M, K, V, keep=None, smoothing=0.0, scale=1.0, ignored=0.2, seed=0, std=None):
    g = gen(dev, seed)
    x, w = randn(g, M, K), randn(g, V, K, std=std or 1 / math.sqrt(K))
    t = torch.randint(0, V, (M,), generator=g, device=dev)
    t[torch.rand(M, generator=g, device=dev) < ignored] = -100
    dl = randn(g, M, dtype=torch.float32)
    mask = None
    if keep is not None:
        mask = torch.rand(M, V, generator=g, device=dev) < keep
        mask[torch.arange(M, device=dev), t.clamp_min(0)] = True
        mask[::5] = torch.rand(mask[::5].shape, generator=g, device=dev) < keep   # targets may be outside
        mask[0] = False                                                            # nothing left
    x6, w6 = x.double().requires_grad_(True), w.double().requires_grad_(True)
    z = (x6 @ w6.t()) * scale
    zm = z if mask is None else z.masked_fill(~mask, -1e300)
    lse = torch.logsumexp(zm, -1)
    empty = torch.zeros(M, dtype=torch.bool, device=dev) if mask is None else ~mask.any(-1)
    valid = t != -100
    out_of = torch.zeros_like(valid) if mask is None else ~mask[torch.arange(M, device=dev), t.clamp_min(0)]
    zt = z.gather(1, t.clamp_min(0)[:, None])[:, 0]
    # a masked target: its logit is a constant, the gradient is that of lse
    loss = (1 - smoothing) * (lse - torch.where(out_of, zt.detach(), zt)) + smoothing * (lse - z.mean(-1))
    (torch.where(valid & ~empty, loss, 0.0 * loss) * dl.double()).sum().backward()
    with torch.no_grad():
        inf = float("inf")
        wl = torch.where(valid, torch.where(out_of, torch.full_like(loss, inf), loss), torch.zeros_like(loss))
        wlse = torch.where(empty, torch.full_like(lse, -inf), lse)
        zsum = float((x6.abs() @ w6.abs().t()).max()) * scale
        tl = E * zsum + E * (1 + wl.abs().nan_to_num(posinf=0.0) + lse.abs().clamp_max(1e6))
        gr = (valid & ~empty) * dl.double().abs() * scale
        hot = torch.nn.functional.one_hot(t.clamp_min(0), V) if M * V < 1 << 26 else None
        p = torch.exp(zm - lse[:, None])
        dz = p - smoothing / V
        if hot is not None:
            dz = dz - (1 - smoothing) * hot * ~out_of[:, None]
        else:
            dz[torch.arange(M, device=dev), t.clamp_min(0)] -= (1 - smoothing)
        if mask is not None:
            dz = dz * mask
        e = (2 * U * dz.abs() + 32 * E * (1 + zsum) * p) * gr[:, None]
        tx = e @ w6.abs() + 2 * U * x6.grad.abs() + 1e-9
        tw = e.t() @ x6.abs() + 2 * U * w6.grad.abs() + 1e-9
    kw = dict(scale=scale, smoothing=smoothing, keep=None if mask is None else words_of(mask))
    return x, w, t, dl, kw, (wl, wlse, x6.grad, w6.grad), (tl, tx, tw)


def check_xent(case):
    x, w, t, dl, kw, (wl, wlse, wx, ww), (tl, tx, tw) = case
    loss, lse = ops.linear_xent(x, w, t, **kw)
    for name, g, a in (("loss", loss, wl), ("lse", lse, wlse)):
        assert g.dtype == torch.float32
        inf = torch.isinf(a)
        assert torch.equal(g[inf].double(), a[inf]), name
        close(torch.where(inf, torch.zeros_like(g), g), torch.where(inf, torch.zeros_like(a), a), tl, name)
    dx, dw = ops.linear_xent_bwd(x, w, t, lse, dl, **kw)
    close(dx, wx, tx, "dx")
    close(dw, ww, tw, "dw")
    return loss, lse, dx, dw


XENT = [
    dict(M=1, K=8, V=1, ignored=0.0), dict(M=1, K=64, V=31, ignored=0.0), dict(M=3, K=200, V=33),
    dict(M=127, K=256, V=1000, smoothing=0.1), dict(M=128, K=64, V=256), dict(M=130, K=72, V=257, scale=0.7),
    dict(M=300, K=64, V=3001, smoothing=0.2, scale=1.5), dict(M=40, K=64, V=100, ignored=1.0),
    dict(M=65, K=64, V=999, keep=0.05, scale=1.25), dict(M=131, K=128, V=2048, keep=0.5),
    dict(M=20, K=32, V=40, keep=0.0), dict(M=64, K=64, V=9001), dict(M=50, K=64, V=500, std=3.0),
]


@on_devices
@pytest.mark.parametrize("c", XENT, ids=str)
def test_linear_xent(dev, c):
    check_xent(xent_case(dev, **c))


@pytest.mark.gpu
def test_linear_xent_in_pieces():
    """More columns than one piece of the gradient's workspace holds, the last one short."""
    check_xent(xent_case("cuda", M=20000, K=64, V=7001, smoothing=0.1))


@on_devices
def test_linear_xent_views_and_refusals(dev):
    x, w, t, dl, kw, want, tol = xent_case(dev, M=12, K=64, V=100, ignored=0.0)
    loss, lse = ops.linear_xent(x, w, t, **kw)
    l2, _ = ops.linear_xent(x.view(3, 4, 64), w, t.to(torch.int32).view(3, 4), **kw)
    assert torch.equal(l2.view(-1), loss)
    dx, dw = ops.linear_xent_bwd(x, w, t, lse, dl, **kw)
    d2, none = ops.linear_xent_bwd(x.view(3, 4, 64), w, t.view(3, 4), lse.view(3, 4), dl.view(3, 4), need_dw=False,
                                   **kw)
    assert none is None and torch.equal(d2.view(12, 64), dx)
    e, _ = ops.linear_xent(x[:0], w, t[:0])
    assert e.shape == (0,)
    assert float(ops.linear_xent_bwd(x[:0], w, t[:0], lse[:0], dl[:0])[1].abs().max()) == 0.0
    with pytest.raises(ValueError):
        ops.linear_xent(x, w[:, :32], t)
    with pytest.raises(ValueError):
        ops.linear_xent(x, w, t[:5])
    with pytest.raises(ValueError):
        ops.linear_xent(x, w, t.float())
    with pytest.raises(ValueError):
        ops.linear_xent(x, w, t, smoothing=1.5)
    with pytest.raises(ValueError):
        ops.linear_xent(x, w, t, smoothing=0.1, keep=torch.zeros(12, 4, dtype=torch.int32, device=dev))
    if dev == "cuda":
        with pytest.raises(RuntimeError, match="keep"):
            ops.linear_xent(x, w, t, keep=torch.zeros(12, 3, dtype=torch.int32, device=dev))
        with pytest.raises(RuntimeError, match="multiple of 8"):
            ops.linear_xent(x[:, :60], w[:, :60], t)
        ops.check_status()
        bad = t.clone()
        bad[3] = 100    # one past the vocabulary: no access, loss 0, the status says so
        got, _ = ops.linear_xent(x, w, bad)
        assert float(got[3]) == 0.0
        with pytest.raises(RuntimeError, match="status"):
            ops.check_status()
        ops.check_status()


# ----------------------------------------------------------------------------- norms
def norm_case(dev, M, D, kind, delta, xt, wt, bias=True, seed=0):
    g = gen(dev, seed)
    x, dy = randn(g, M, D, dtype=xt) + 0.5, randn(g, M, D, dtype=xt)
    w = randn(g, D, std=0.2, dtype=wt) + 1.0
    b = randn(g, D, std=0.2, dtype=wt) if kind == "layer" and bias else None
    d = randn(g, M, D, dtype=xt) if delta else None
    dh = randn(g, M, D, dtype=xt) if delta else None
    h = x if d is None else (x.float() + d.float()).to(xt)
    h6, w6 = h.double().requires_grad_(True), w.double().requires_grad_(True)
    b6 = torch.zeros_like(w6) if b is None else b.double().requires_grad_(True)
    mu = h6.mean(-1, keepdim=True) if kind == "layer" else 0.0
    r = ((h6 - mu).pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt()
    y = (h6 - mu) * r * w6 + b6
    L = (y * dy.double()).sum()
    if dh is not None:
        L = L + (h6 * dh.double()).sum()
    L.backward()
    with torch.no_grad():
        ux = 2 * U if xt == torch.bfloat16 else 0.0
        uw = 2 * U if wt == torch.bfloat16 else 0.0
        n = ((h6 - mu) * r).abs()
        gy = dy.double().abs()
        cond = 1 + h6.abs().amax(-1, keepdim=True) * r        # cancellation in h - mu
        a = gy * w6.abs()
        ty = ux * y.abs() + E * (cond * w6.abs() * (1 + n) + b6.abs()) + 1e-9
        tx = ux * h6.grad.abs() + 4 * E * cond * r * (a + (1 + n) * ((a * n).mean(-1, keepdim=True)
                                                                    + a.mean(-1, keepdim=True))) + 1e-9
        if dh is not None:
            tx = tx + E * dh.double().abs()
        tw = uw * w6.grad.abs() + E * (gy * (cond + n)).sum(0) + 1e-9
        tb = uw * (0 if b is None else b6.grad.abs()) + E * gy.sum(0) + 1e-9
    return x, w, b, d, dy, dh, h, (y.detach(), h6.grad, w6.grad, None if b is None else b6.grad), (ty, tx, tw, tb)


B16, F32 = torch.bfloat16, torch.float32
NORM = [
    (1, 8, "rms", False, B16, B16), (3, 7, "layer", False, B16, F32), (64, 256, "rms", True, B16, B16),
    (5, 1, "rms", False, F32, F32), (33, 100, "layer", True, B16, B16), (700, 512, "layer", False, B16, F32),
    (129, 1000, "rms", True, B16, F32), (257, 1024, "layer", True, B16, B16), (31, 1031, "layer", False, F32, F32),
    (65, 2048, "rms", False, F32, F32), (300, 4096, "rms", True, B16, B16), (9, 4097, "rms", False, B16, B16),
    (40, 8192, "layer", True, B16, F32), (7, 16384, "layer", False, B16, B16), (4, 16383, "layer", False, B16, B16),
    (2500, 16, "layer", False, B16, B16),
]


@on_devices
@pytest.mark.parametrize("c", NORM, ids=str)
def test_norm_train(dev, c):
    M, D, kind, delta, xt, wt = c
    x, w, b, d, dy, dh, h, want, tol = norm_case(dev, M, D, kind, delta, xt, wt)
    y, hh, stats = ops.norm_train(x, w, b, 1e-5, kind=kind, delta=d)
    assert torch.equal(hh, h)
    dx, dw, db = ops.norm_train_bwd(dy, hh, w, stats, kind=kind, bias=b is not None, dh=dh)
    assert dx.dtype == xt and dw.dtype == wt
    for name, g, a, t in zip(("y", "dx", "dw", "db"), (y, dx, dw, db), want, tol):
        if a is None:
            assert g is None
        else:
            close(g, a, t, name)


@on_devices
def test_norm_train_views_and_refusals(dev):
    x, w, b, d, dy, dh, h, want, tol = norm_case(dev, 12, 64, "layer", True, B16, F32)
    y, hh, stats = ops.norm_train(x, w, b, 1e-5, kind="layer", delta=d)
    wide = torch.zeros(12, 131, dtype=B16, device=dev)
    wide[:, 5:69] = x                      # rows that start off a 16-byte boundary
    y2, h2, s2 = ops.norm_train(wide[:, 5:69], w, b, 1e-5, kind="layer", delta=d)
    close(y2, want[0], tol[0], "y of a view")
    assert torch.equal(h2, hh)
    dx, dw, db = ops.norm_train_bwd(dy.view(3, 4, 64), hh.view(3, 4, 64), w, stats, kind="layer", bias=True,
                                    dh=dh.view(3, 4, 64))
    close(dx.view(12, 64), want[1], tol[1], "dx of a batch")
    y0, _, s0 = ops.norm_train(x[:0], w, b, 1e-5, kind="layer")
    assert y0.shape == (0, 64)
    assert float(ops.norm_train_bwd(dy[:0], x[:0], w, s0, kind="layer", bias=True)[1].abs().max()) == 0.0
    with pytest.raises(ValueError):
        ops.norm_train(x, w, b, 1e-5, kind="rms")
    with pytest.raises(ValueError):
        ops.norm_train(x, w, kind="batch")
    if dev == "cuda":
        with pytest.raises(ValueError):
            ops.norm_train(x, w, delta=d[:3])
        with pytest.raises(RuntimeError, match=r"\[D\]"):
            ops.norm_train(x, w[:32])
        with pytest.raises(RuntimeError, match="16384"):
            ops.norm_train(torch.zeros(2, 16392, dtype=B16, device=dev), torch.ones(16392, dtype=B16, device=dev))
        with pytest.raises(RuntimeError, match="bf16 or fp32"):
            ops.norm_train(x.half(), w)


# ----------------------------------------------------------------------------- differences, streams, repeats
@on_devices
def test_gradients_against_differences(dev):
    """Central differences of the 64-bit losses along a random direction against <gradient, direction>."""
    eps = 1e-5
    x, w, t, dl, kw, want, tol = xent_case(dev, M=24, K=64, V=300, smoothing=0.1, scale=0.8)
    g = gen(dev, 9)
    d = torch.randn(x.shape, generator=g, device=dev, dtype=torch.float64)

    def loss(xx):
        z = (xx @ w.double().t()) * 0.8
        l = torch.logsumexp(z, -1)
        v = 0.9 * (l - z.gather(1, t.clamp_min(0)[:, None])[:, 0]) + 0.1 * (l - z.mean(-1))
        return (torch.where(t >= 0, v, 0.0) * dl.double()).sum()

    num = (loss(x.double() + eps * d) - loss(x.double() - eps * d)) / (2 * eps)
    _, lse = ops.linear_xent(x, w, t, **kw)
    dx, _ = ops.linear_xent_bwd(x, w, t, lse, dl, **kw)
    assert abs(float((dx.double() * d).sum() - num)) <= float((tol[1] * d.abs()).sum()) + 1e-6

    c = attention_case(dev, 1, 40, 40, 2, 1, 64, True, None)
    mask = visible(1, 40, 40, True, None, dev)
    d = torch.randn(c["k"].shape, generator=g, device=dev, dtype=torch.float64)
    f = lambda kk: (attention64(c["q"].double(), kk, c["v"].double(), c["scale"], mask)[0] * c["do"].double()).sum()  # noqa: E731
    num = (f(c["k"].double() + eps * d) - f(c["k"].double() - eps * d)) / (2 * eps)
    dk = check_attention(c, True)[1]
    assert abs(float((dk.double() * d).sum() - num)) <= float((c["tol"][1] * d.abs()).sum()) + 1e-6

    x, w, dh, want, tol = swiglu_case(dev, 20, 64, 48)
    d = torch.randn(w.shape, generator=g, device=dev, dtype=torch.float64)

    def f(ww):
        z = x.double() @ ww.t()
        return (torch.nn.functional.silu(z[:, :48]) * z[:, 48:] * dh.double()).sum()

    num = (f(w.double() + eps * d) - f(w.double() - eps * d)) / (2 * eps)
    dw = ops.swiglu_bwd(x, w, ops.swiglu(x, w, save=True)[1], dh)[1]
    assert abs(float((dw.double() * d).sum() - num)) <= float((tol[2] * d.abs()).sum()) + 1e-6

    x, w, b, _, dy, _, h, want, tol = norm_case(dev, 9, 72, "layer", False, F32, F32)
    d = torch.randn(x.shape, generator=g, device=dev, dtype=torch.float64)

    def f(xx):
        mu = xx.mean(-1, keepdim=True)
        return ((xx - mu) * ((xx - mu).pow(2).mean(-1, keepdim=True) + 1e-5).rsqrt() * w.double() * dy.double()).sum()

    num = (f(x.double() + eps * d) - f(x.double() - eps * d)) / (2 * eps)
    dx = ops.norm_train_bwd(dy, x, w, ops.norm_train(x, w, b, 1e-5, kind="layer")[2], kind="layer")[0]
    assert abs(float((dx.double() * d).sum() - num)) <= float((tol[1] * d.abs()).sum()) + 1e-6


@pytest.mark.gpu
def test_same_result_on_every_run_and_stream():
    dev = "cuda"
    c = attention_case(dev, 2, 300, 300, 8, 2, 128, True, [300, 111])
    xc = xent_case(dev, M=256, K=128, V=5000)
    sc = swiglu_case(dev, 200, 128, 300)
    nc = norm_case(dev, 3000, 512, "layer", True, B16, F32)

    def all_of():
        out = list(ops.attention_bwd(c["q"], c["k"], c["v"], c["out"], c["lse"], c["do"], c["scale"], lens=c["lens"]))
        loss, lse = ops.linear_xent(xc[0], xc[1], xc[2])
        out += [loss, lse, *ops.linear_xent_bwd(xc[0], xc[1], xc[2], lse, xc[3])]
        h, gu = ops.swiglu(sc[0], sc[1], save=True)
        out += [h, *ops.swiglu_bwd(sc[0], sc[1], gu, sc[2])]
        y, hh, st = ops.norm_train(nc[0], nc[1], nc[2], kind="layer", delta=nc[3])
        return out + [y, *ops.norm_train_bwd(nc[4], hh, nc[1], st, kind="layer", bias=True, dh=nc[5])]

    first = all_of()
    again = all_of()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(s1):
        a = all_of()
    with torch.cuda.stream(s2):
        b = all_of()
    torch.cuda.synchronize()
    ops.check_status()
    for p, q, r, s in zip(first, again, a, b):
        assert torch.equal(p, q) and torch.equal(p, r) and torch.equal(p, s)


def test_native_refusals_name_their_numbers():
    """An error raised by the native entry (sizes in its text) reaches Python as an exception."""
    from openmini_v1_b200 import _native
    if not _native.have_C():
        pytest.skip("native extension not built")
    t = torch.zeros(1, 2, 2, 60, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="got 60"):
        _native.C().attention_bwd(t, t, t, t, t, t, None, 1.0, True, t)


# ----------------------------------------------------------------------------- through autograd and the policy
def test_autograd_forms_on_cpu():
    """The CPU forms of ops.autograd differentiate to the reference statements of the kernels."""
    from openmini_v1_b200.ops import autograd as ag
    g = gen("cpu", 3)
    x, w = randn(g, 2, 5, 16, dtype=F32).requires_grad_(True), randn(g, 24, 16, dtype=F32).requires_grad_(True)
    t = torch.randint(0, 24, (2, 5), generator=g)
    t[0, 1] = -100
    words = words_of(torch.rand(10, 24, generator=g) < 0.7)
    for kw in (dict(smoothing=0.1), dict(scale=0.5), dict(keep=words)):
        loss = ag.linear_xent(x, w, t, **kw)
        want, lse = ops.linear_xent(x.detach(), w.detach(), t, **kw)
        torch.testing.assert_close(loss.detach(), want)
        gl = torch.where(torch.isfinite(want), torch.ones_like(want), torch.zeros_like(want))
        dx, dw = torch.autograd.grad(loss.masked_fill(~torch.isfinite(want), 0.0), (x, w), gl)
        rx, rw = ops.linear_xent_bwd(x.detach(), w.detach(), t, lse, gl, **kw)
        torch.testing.assert_close(dx, rx, atol=1e-5, rtol=1e-5)
        torch.testing.assert_close(dw, rw, atol=1e-5, rtol=1e-5)
    h = ag.swiglu(x, w)
    dx, dw = torch.autograd.grad(h, (x, w), torch.ones_like(h))
    rh, gu = ops.swiglu(x.detach(), w.detach(), save=True)
    rx, rw = ops.swiglu_bwd(x.detach(), w.detach(), gu, torch.ones_like(h))
    for a, b in ((h.detach(), rh), (dx, rx), (dw, rw)):
        torch.testing.assert_close(a, b, atol=1e-5, rtol=1e-5)


def small_policy(dev, moe=False, head_dim=64):
    from openmini_v1_b200.models.config import ModelConfig, MoEConfig
    from openmini_v1_b200.models.policy import Policy
    cfg = ModelConfig(name="p", vocab_size=520, hidden_size=192, num_layers=2, num_heads=4, num_kv_heads=2,
                      head_dim=head_dim, intermediate_size=344, max_position=512, dtype="float32",
                      moe=MoEConfig(num_experts=4, top_k=2, expert_ffn=72, layer_rule="all") if moe else MoEConfig())
    return Policy(cfg, device=dev, seed=5)


def test_policy_loss_is_the_logits_loss():
    from openmini_v1_b200.train.loss import causal_lm_loss
    p = small_policy("cpu")
    ids = torch.randint(0, 520, (3, 20), generator=gen("cpu", 1))
    labels = ids.clone()
    labels[:, :6] = -100
    for s in (0.0, 0.1):
        torch.testing.assert_close(p.loss(ids, labels, s), causal_lm_loss(p(ids), labels, s))
    assert float(p.loss(ids, torch.full_like(ids, -100))) == 0.0
    from openmini_v1_b200.models.policy import token_logprobs
    h, lg = p.hidden(ids)[0], p(ids)[0]
    mask = torch.rand(20, 520, generator=gen("cpu", 2)) < 0.5
    mask[torch.arange(20), ids[1]] = True
    torch.testing.assert_close(p.logprobs(h, ids[1], 0.7, words_of(mask)), token_logprobs(lg, ids[1], 0.7, mask),
                               atol=1e-5, rtol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("moe,head_dim", [(False, 64), (False, 128), (True, 48)])
def test_policy_loss_and_gradients_on_gpu(moe, head_dim):
    """A training step on the kernels against the same weights in fp32 on the CPU (bf16 activations
    through two layers: compared in norm)."""
    import copy
    cpu = small_policy("cpu", moe, head_dim)
    gpu = copy.deepcopy(cpu).to("cuda")
    gpu.device, gpu.cdt, gpu.inv_freq = torch.device("cuda"), torch.bfloat16, gpu.inv_freq.to("cuda")
    ids = torch.randint(0, 520, (3, 150), generator=gen("cpu", 1))
    labels = ids.clone()
    labels[:, :20] = -100
    labels[2, 90:] = -100
    a, b = cpu.loss(ids, labels, 0.05), gpu.loss(ids.cuda(), labels.cuda(), 0.05)
    assert abs(float(a) - float(b)) < 2e-3 * float(a)
    a.backward()
    b.backward()
    ops.check_status()
    for (n, pc), (_, pg) in zip(cpu.named_parameters(), gpu.named_parameters()):
        if pc.grad is None:
            continue
        rel = float((pg.grad.cpu() - pc.grad).norm() / (pc.grad.norm() + 1e-12))
        assert rel < 0.1, (n, rel)


@pytest.mark.gpu
def test_trainer_step_on_gpu_uses_no_logits():
    from openmini_v1_b200.train.trainer import Trainer, TrainingConfig
    p = small_policy("cuda")

    def no_logits(*a, **k):
        raise AssertionError("the logits were computed")

    p.forward = no_logits
    ids = torch.randint(0, 520, (4, 64), generator=gen("cpu", 4))

    class Loader(list):
        def set_epoch(self, e):
            pass

    import tempfile
    with tempfile.TemporaryDirectory() as d:
        cfg = TrainingConfig(num_train_epochs=1, learning_rate=1e-3, output_dir=d, save_steps=0, logging_steps=1)
        tr = Trainer(p, cfg, Loader([{"input_ids": ids, "labels": ids}] * 8))
        st = tr.train()
    losses = [r["loss"] for r in st.history if "loss" in r]
    assert losses[-1] < losses[0] and all(math.isfinite(v) for v in losses)
    ops.check_status()


@pytest.mark.gpu
def test_trainer_stops_at_a_label_outside_the_vocabulary():
    import tempfile

    from openmini_v1_b200.train.trainer import Trainer, TrainingConfig
    p = small_policy("cuda")
    before = p.lm_head.detach().clone()
    ids = torch.randint(0, 520, (2, 32), generator=gen("cpu", 4))
    labels = ids.clone()
    labels[1, 7] = 520

    class Loader(list):
        def set_epoch(self, e):
            pass

    with tempfile.TemporaryDirectory() as d:
        tr = Trainer(p, TrainingConfig(num_train_epochs=1, output_dir=d, save_steps=0),
                     Loader([{"input_ids": ids, "labels": labels}]))
        with pytest.raises(RuntimeError, match="status"):
            tr.train()
    assert torch.equal(before, p.lm_head.detach())
    ops.check_status()


# ----------------------------------------------------------------------------- errors in the data
def test_status_text():
    """A status word's low byte is the first wait that gave up or 5, its second byte 5 beside a wait."""
    assert ops.status_text(5) == "an index in the data was out of range"
    assert ops.status_text(1) == "a wait for a filled stage gave up"
    assert ops.status_text(3 | 5 << 8) == "a wait for an accumulator gave up; an index in the data was out of range"


@pytest.mark.gpu
def test_targets_outside_the_vocabulary_leave_other_results_alone():
    """They count as ignored, the status says so, and neither the gradient of the same call nor later calls
    (products of several waves of tiles, with long waits) stop early."""
    ops.check_status()
    g = gen("cuda", 0)
    x, w, dl = randn(g, 2049, 1024), randn(g, 4100, 1024, std=1 / 32), randn(g, 2049, dtype=F32)
    wf, dh = randn(g, 4400, 1024, std=1 / 32), randn(g, 2049, 2200)
    t = torch.randint(0, 4100, (2049,), generator=g, device="cuda")
    t[::97] = -100
    bad = t.clone()
    bad[::97] = 4100
    bad[97] = -7

    def all_of(t):
        loss, lse = ops.linear_xent(x, w, t)
        h, gu = ops.swiglu(x, wf, save=True)
        return [loss, lse, *ops.linear_xent_bwd(x, w, t, lse, dl), h, *ops.swiglu_bwd(x, wf, gu, dh)]

    want, got = all_of(t), all_of(bad)
    with pytest.raises(RuntimeError, match="out of range"):
        ops.check_status()
    for a, b in zip(want, got):
        assert torch.equal(a, b)
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [2 ** 31 - 256, 2 ** 31 - 1])
def test_swiglu_refuses_rows_whose_tiles_pass_32_bits(rows):
    """The last row tile's index must not wrap; refused before anything of that size is allocated."""
    x = torch.zeros(1, 8, dtype=B16, device="cuda").expand(rows, 8)
    w = torch.zeros(16, 8, dtype=B16, device="cuda")
    before = torch.cuda.memory_allocated()
    for call in (lambda: ops.swiglu(x, w), lambda: ops.swiglu_bwd(x, w, x, x)):
        with pytest.raises(RuntimeError, match="too large"):
            call()
    assert torch.cuda.memory_allocated() == before


@on_devices
@pytest.mark.parametrize("B,T,S,H,Hkv", [(0, 3, 3, 2, 1), (2, 0, 5, 2, 1), (2, 5, 0, 2, 2), (1, 4, 4, 0, 1)])
def test_attention_bwd_of_nothing(dev, B, T, S, H, Hkv):
    """No sequence, query, key or query head: empty results, and zeros for the keys nobody reads."""
    q, k = (torch.ones(B, n, h, 64, dtype=B16, device=dev) for n, h in ((T, H), (S, Hkv)))
    lse = torch.zeros(B, T, H, device=dev)
    got = ops.attention_bwd(q, k, k, q, lse, q, 1.0, causal=False)
    for g, like in zip(got, (q, k, k)):
        assert g.shape == like.shape and not g.any()


@on_devices
def test_linear_xent_of_nan_rows(dev):
    """A row of NaN logits has a NaN lse; -inf is the lse of a row without a column alone."""
    g = gen(dev, 1)
    x, w = randn(g, 5, 64), randn(g, 300, 64)
    x[1] = float("nan")
    t = torch.tensor([0, 1, 2, -100, 4], device=dev)
    loss, lse = ops.linear_xent(x, w, t)
    dx, dw = ops.linear_xent_bwd(x, w, t, lse, torch.ones(5, device=dev))
    ok = torch.tensor([True, False, True, True, True])
    for v in (loss, lse, dx.float().sum(-1)):
        assert torch.equal(torch.isfinite(v).cpu(), ok) and bool(torch.isnan(v[1]))


def _norm_forms():
    from openmini_v1_b200.ops import autograd as ag
    rms = lambda x, w: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w  # noqa: E731

    def layer(x, w, b):
        d = x - x.mean(-1, keepdim=True)
        return d * torch.rsqrt(d.pow(2).mean(-1, keepdim=True) + 1e-5) * w + b

    return {"rms": (lambda x, y, w: ag.rmsnorm(x, w, 1e-5), lambda x, y, w: rms(x, w)),
            "add": (lambda x, y, w: sum(ag.add_rmsnorm(x, y, w, 1e-5)), lambda x, y, w: rms(x + y, w) + x + y),
            "layer": (lambda x, y, w: ag.layernorm(x, w, y[0], 1e-5), lambda x, y, w: layer(x, w, y[0]))}


@on_devices
@pytest.mark.parametrize("form,shape", [("rms", (6, 48)), ("add", (6, 48)), ("layer", (6, 48)), ("rms", (48,))])
def test_norms_differentiate_twice(dev, form, shape):
    """A gradient taken with create_graph=True differentiates on: f(x) = sum norm(x)^3, then |grad f|^2."""
    got, want = _norm_forms()[form]
    g = gen(dev, 2)
    inputs = [randn(g, *shape, dtype=F32), randn(g, *shape, dtype=F32), randn(g, 48, dtype=F32)]
    out = []
    for f, dt in ((got, F32), (want, torch.float64)):
        a = [t.to(dt).requires_grad_(True) for t in inputs]
        used = [t for t, name in zip(a, "xyw") if not (form == "rms" and name == "y")]
        first = torch.autograd.grad((f(*a) ** 3).sum(), used, create_graph=True)
        out.append([*first, *torch.autograd.grad(sum((v ** 2).sum() for v in first), used)])
    for a, b in zip(*out):
        torch.testing.assert_close(a.double(), b, rtol=2e-4, atol=2e-4 * float(b.abs().max()))


@on_devices
def test_second_derivatives_of_the_fused_products_are_refused(dev):
    """swiglu, linear_xent and attention have first derivatives only, and say so, also beside a path
    that has more (on the CPU the first two are plain operations)."""
    from openmini_v1_b200.ops import autograd as ag
    g = gen(dev, 2)
    x, w = randn(g, 8, 64).requires_grad_(True), randn(g, 48, 64).requires_grad_(True)
    q = randn(g, 1, 16, 2, 64).requires_grad_(True)
    t = torch.randint(0, 48, (8,), generator=g, device=dev)
    forms = [(lambda: ag.attention(q, q, q, 0.1), q)]
    if dev == "cuda":
        forms += [(lambda: ag.swiglu(x, w), x), (lambda: ag.linear_xent(x, w, t), x)]
    for f, v in forms:
        want, = torch.autograd.grad(f().float().sum(), v)
        first, = torch.autograd.grad(f().float().sum() + v.float().pow(3).sum(), v, create_graph=True)
        torch.testing.assert_close(first.float(), want.float() + 3 * v.detach().float().pow(2), atol=0.1, rtol=2e-2)
        with pytest.raises(RuntimeError, match="first derivatives only"):
            torch.autograd.grad(first.float().pow(2).sum(), v)


@on_devices
def test_rmsnorm_under_transforms_and_with_other_gains(dev):
    """vmap, jvp and forward-mode duals go through ag.rmsnorm, and a gain need not be a vector of the row's length."""
    import torch.autograd.forward_ad as fw

    from openmini_v1_b200.ops import autograd as ag
    g = gen(dev, 4)
    x, v, w = randn(g, 3, 5, 48, dtype=F32), randn(g, 3, 5, 48, dtype=F32), randn(g, 48, dtype=F32)
    plain = lambda x, w: x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-5) * w  # noqa: E731
    f = lambda x: ag.rmsnorm(x, w, 1e-5)  # noqa: E731
    torch.testing.assert_close(torch.func.vmap(f)(x), plain(x, w))
    y, dy = torch.func.jvp(f, (x,), (v,))
    wy, wdy = torch.func.jvp(lambda x: plain(x, w), (x,), (v,))
    torch.testing.assert_close(y, wy)
    torch.testing.assert_close(dy, wdy)
    with fw.dual_level():
        torch.testing.assert_close(fw.unpack_dual(f(fw.make_dual(x, v))).tangent, wdy)
    torch.testing.assert_close(torch.func.grad(lambda x: f(x).pow(3).sum())(x),
                               torch.func.grad(lambda x: plain(x, w).pow(3).sum())(x), rtol=1e-4, atol=1e-4)
    for gain in (w[None], w[:1], torch.tensor(0.5, device=dev), randn(g, 5, 48, dtype=F32)):
        torch.testing.assert_close(ag.rmsnorm(x, gain, 1e-5), plain(x, gain))
    torch.testing.assert_close(ag.layernorm(x, w[None], None, 1e-5),
                               torch.nn.functional.layer_norm(x, (48,)) * w, rtol=1e-4, atol=1e-4)
    torch.testing.assert_close(ag.add_rmsnorm(x, v[:1], w, 1e-5)[0], plain(x + v[:1], w))


@pytest.mark.gpu
def test_a_label_outside_the_vocabulary_has_no_loss():
    """Neither Policy.loss nor an evaluation returns a number for it."""
    import tempfile

    from openmini_v1_b200.train.trainer import Trainer, TrainingConfig
    p = small_policy("cuda")
    ids = torch.randint(0, 520, (2, 32), generator=gen("cpu", 4))
    labels = ids.clone()
    labels[1, 7] = 520
    with pytest.raises(RuntimeError, match="out of range"):
        p.loss(ids.cuda(), labels.cuda())
    ops.check_status()
    good = {"input_ids": ids, "labels": ids}
    with tempfile.TemporaryDirectory() as d:
        tr = Trainer(p, TrainingConfig(num_train_epochs=1, output_dir=d, save_steps=0), [good],
                     eval_loader=[good, {"input_ids": ids, "labels": labels}, good])
        with pytest.raises(RuntimeError, match="out of range"):
            tr.evaluate()
        tr.eval_loader = [good]
        assert math.isfinite(tr.evaluate())


@pytest.mark.gpu
def test_trainer_runs_the_models_own_forward():
    """A subclass's forward and forward hooks decide the loss on the GPU as they do on the CPU."""
    import tempfile

    from openmini_v1_b200.models.policy import Policy
    from openmini_v1_b200.train.loss import causal_lm_loss
    from openmini_v1_b200.train.trainer import Trainer, TrainingConfig

    class Sharp(Policy):
        def forward(self, *a, **k):
            return super().forward(*a, **k) * 3.0

    base = small_policy("cuda")
    ids = torch.randint(0, 520, (2, 32), generator=gen("cpu", 4))
    batch = {"input_ids": ids, "labels": ids}
    want = float(causal_lm_loss(base(ids.cuda()) * 3.0, ids.cuda()))
    sharp = Sharp(base.cfg, device="cuda", seed=5)
    hooked = small_policy("cuda")
    hooked.register_forward_hook(lambda m, a, out: out * 3.0)
    for m in (sharp, hooked):
        with tempfile.TemporaryDirectory() as d:
            tr = Trainer(m, TrainingConfig(num_train_epochs=1, output_dir=d, save_steps=0), [batch])
            assert abs(float(tr._loss(batch)) - want) < 1e-3 * want
    plain = float(causal_lm_loss(base(ids.cuda()), ids.cuda()))
    assert abs(plain - want) > 1e-3 * want


def grpo_case(cls=None):
    """A trainer without its engine, samples of unequal lengths, kept sets for some of them."""
    from openmini_v1_b200.models.policy import Policy
    from openmini_v1_b200.rl.replay import EnforceMode, KeepRouting, KeepSamplingMask
    from openmini_v1_b200.rl.trainer import GRPOTrainer
    pol = small_policy("cuda", moe=True) if cls is None else cls(small_policy("cpu").cfg, device="cuda", seed=5)
    tr = GRPOTrainer.__new__(GRPOTrainer)
    tr.policy, tr.temperature, tr.train_batch = pol, 0.8, 3
    tr.keep_routing, tr.keep_mask = KeepRouting(100, EnforceMode.NONE), KeepSamplingMask(100)
    g = gen("cpu", 6)
    samples = []
    for i, (n, c) in enumerate([(4, 9), (17, 1), (3, 30), (40, 12), (5, 5)]):
        toks = torch.randint(0, 520, (n + c,), generator=g).tolist()
        samples.append({"key": f"s{i}", "prompt": toks[:n], "completion": toks[n:]})
        if i % 2 == 0:
            mask = torch.rand(c, 520, generator=g) < 0.3
            mask[torch.arange(c), torch.tensor(toks[n:])] = True
            tr.keep_mask.save(f"s{i}", words_of(mask))
    return tr, pol, samples


def grpo_case(cls=None):
    """A trainer without its engine, samples of unequal lengths, kept sets for some of them."""
    from openmini_v1_b200.models.policy import Policy
    from openmini_v1_b200.rl.replay import EnforceMode, KeepRouting, KeepSamplingMask
    from openmini_v1_b200.rl.trainer import GRPOTrainer
    pol = small_policy("cuda", moe=True) if cls is None else cls(small_policy("cpu").cfg, device="cuda", seed=5)
    tr = GRPOTrainer.__new__(GRPOTrainer)
    tr.policy, tr.temperature, tr.train_batch = pol, 0.8, 3
    tr.keep_routing, tr.keep_mask = KeepRouting(100, EnforceMode.NONE), KeepSamplingMask(100)
    g = gen("cpu", 6)
    samples = []
    for i, (n, c) in enumerate([(4, 9), (17, 1), (3, 30), (40, 12), (5, 5)]):
        toks = torch.randint(0, 520, (n + c,), generator=g).tolist()
        samples.append({"key": f"s{i}", "prompt": toks[:n], "completion": toks[n:]})
        if i % 2 == 0:
            mask = torch.rand(c, 520, generator=g) < 0.3
            mask[torch.arange(c), torch.tensor(toks[n:])] = True
            tr.keep_mask.save(f"s{i}", words_of(mask))
    return tr, pol, samples


@pytest.mark.gpu
def test_grpo_runs_the_models_own_forward():
    from openmini_v1_b200.models.policy import Policy

    class Sharp(Policy):
        def forward(self, *a, **k):
            return super().forward(*a, **k) * 3.0

    tr, pol, samples = grpo_case(Sharp)
    tr.keep_mask.clear()
    got = tr._batch_logp(pol, samples[:1])[0]
    ids = torch.tensor(samples[0]["prompt"] + samples[0]["completion"], device="cuda")
    want = torch.log_softmax(pol(ids[None, :-1])[0, 3:] / 0.8, -1).gather(-1, ids[4:, None])[:, 0]
    torch.testing.assert_close(got, want, atol=2e-2, rtol=2e-2)


@pytest.mark.gpu
def test_grpo_batch_of_empty_completions():
    tr, pol, samples = grpo_case()
    for s in samples:
        s["completion"] = []
    rows = tr._batch_logp(pol, samples)
    assert [tuple(r.shape) for r in rows] == [(0,)] * 5


@on_devices
@pytest.mark.parametrize("T,S,D", [(1, 5, 64), (5, 21, 128), (40, 173, 48), (129, 300, 128)])
def test_attention_over_a_prefix(dev, T, S, D):
    """Queries that are the last T of S tokens: keys up to their own."""
    from openmini_v1_b200.ops import autograd as ag
    c = attention_case(dev, 2, T, S, 4, 2, D, True, None)
    q, k, v = (c[n].clone().requires_grad_(True) for n in "qkv")
    out = ag.attention(q, k, v, c["scale"])
    o6 = attention64(c["q"].double(), c["k"].double(), c["v"].double(), c["scale"], visible(2, T, S, True, None, dev))[0]
    assert float((out.double() - o6).abs().max()) < 4 * U * float(c["v"].abs().max())
    out.backward(c["do"])
    for got, want, tol in zip((q.grad, k.grad, v.grad), c["want"], c["tol"]):
        # the forward's own 16-bit out enters through rowsum(dO O)
        assert float((got.double() - want).norm()) < 4 * U * float(want.norm()) + float(tol.norm())


@on_devices
def test_attention_refuses_what_it_cannot_mean(dev):
    from openmini_v1_b200.ops import autograd as ag
    q, k = randn(gen(dev, 1), 1, 5, 2, 64), randn(gen(dev, 2), 1, 3, 2, 64)
    if dev == "cuda":
        with pytest.raises(ValueError, match="keys"):
            ag.attention(q, k, k, 0.1)
    with pytest.raises(ValueError, match="lens"):
        ag.attention(k, q, q, 0.1, torch.tensor([3], dtype=torch.int32, device=dev))


@pytest.mark.gpu
def test_grpo_log_probabilities_are_those_of_the_logits():
    """Hidden rows and kept words (samples without any: all ones) against masked logits, with gradients."""
    tr, pol, samples = grpo_case()

    class Logits:  # no logprobs: the logits' path
        def __call__(self, ids, forced_routing=None):
            return pol(ids, forced_routing=forced_routing)

    out = []
    for model in (pol, Logits()):
        pol.zero_grad()
        rows = tr._batch_logp(model, samples)
        assert [len(r) for r in rows] == [9, 1, 30, 12, 5]
        w = torch.linspace(-1, 1, 57, device="cuda")
        (torch.cat(rows) * w).sum().backward()
        out.append((torch.cat(rows).detach(), {n: p.grad.clone() for n, p in pol.named_parameters() if p.grad is not None}))
    ops.check_status()
    (a, ga), (b, gb) = out
    # the logits' path rounds logits of size up to 4 / 0.8 to 16 bits, in log p twice
    assert float((a - b).abs().max()) < 2 * 2.0 ** -9 * 5 + 1e-3
    for n in gb:
        assert float((ga[n] - gb[n]).norm()) < 0.05 * float(gb[n].norm()) + 1e-6, n


# ----------------------------------------------------------------------------- paths that need large grids
@pytest.mark.gpu
@pytest.mark.parametrize("shape", [
    (6, 300, 300, 16, 4, 128, True, [300, 0, 129, 1, 64, 257]), (3, 700, 700, 12, 2, 64, True, None),
    (2, 520, 777, 16, 16, 96, True, None), (4, 390, 390, 16, 8, 128, False, [390, 0, 65, 389]),
    (2, 900, 500, 8, 4, 64, True, None)], ids=str)
def test_attention_bwd_several_items_a_cta(shape):
    """More work items than SMs (up to three each), full, ragged and empty ones in turn: the resident rows, the
    accumulators and the tiles' places in tensor memory are handed from item to item."""
    check_attention(attention_case("cuda", *shape), shape[6])
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("M,K,F", [(2300, 2056, 1100), (2305, 776, 1101)])
def test_swiglu_on_cta_pairs(M, K, F):
    """Contractions long enough for the CTA-pair GEMM: in all three products / in the forward one, odd F."""
    x, w, dh, want, tol = swiglu_case("cuda", M, K, F)
    h, gu = ops.swiglu(x, w, save=True)
    assert torch.equal(ops.swiglu(x, w), h)
    for name, g, a, t in zip(("h", "dx", "dw"), (h, *ops.swiglu_bwd(x, w, gu, dh)), want, tol):
        close(g, a, t, name)
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("c", [dict(M=4100, K=1280, V=33001), dict(M=1000, K=1024, V=150001, scale=1.2),
                               dict(M=1000, K=1024, V=140000, keep=0.3)], ids=str)
def test_linear_xent_in_pieces_of_large_products(c):
    """Pieces of the vocabulary whose sums for dx run on CTA pairs / as split contractions."""
    check_xent(xent_case("cuda", **c))
    ops.check_status()


@pytest.mark.gpu
@pytest.mark.parametrize("c", [
    (70001, 256, "rms", True, B16, B16), (20011, 1000, "layer", False, B16, B16), (20011, 1024, "layer", True, B16, F32),
    (9001, 2048, "rms", False, B16, B16), (5003, 4096, "rms", True, B16, B16), (3001, 8192, "layer", False, F32, F32),
    (30011, 301, "layer", True, B16, F32), (30011, 301, "rms", False, F32, F32), (8009, 1031, "layer", False, B16, B16),
    (2503, 4097, "rms", True, B16, B16)], ids=str)
def test_norm_rows_refill_their_ring(c):
    """More rows than all groups' rings hold at once: every stage is filled again and its phase turns."""
    M, D, kind, delta, xt, wt = c
    x, w, b, d, dy, dh, h, want, tol = norm_case("cuda", M, D, kind, delta, xt, wt)
    y, hh, stats = ops.norm_train(x, w, b, 1e-5, kind=kind, delta=d)
    assert torch.equal(hh, h)
    for name, g, a, t in zip(("y", "dx", "dw", "db"),
                             (y, *ops.norm_train_bwd(dy, hh, w, stats, kind=kind, bias=b is not None, dh=dh)), want, tol):
        if a is not None:
            close(g, a, t, name)
    ops.check_status()
