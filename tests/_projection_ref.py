"""The operators around a projection in 64 bits (CPU), with how far fp32 arithmetic
may be from them: each bound counts roundings of half a step (2^-24 of a value in
fp32, HALF of one in the output's type) along the longest chain of the sum."""
import torch

HALF = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}  # half a step, relative
SMALLEST = {torch.float32: 2.0**-150, torch.bfloat16: 2.0**-134, torch.float16: 2.0**-25}  # half the smallest step
U = 2.0**-24
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def f64(t):
    return t.detach().cpu().double()


def assert_close(got, want, bound, what=""):
    """|got - want| <= bound + half a step of got's type, with the same infinities and NaN."""
    g, w = f64(got), want
    assert g.shape == w.shape, (what, g.shape, w.shape)
    assert torch.equal(torch.isnan(g), torch.isnan(w)), what
    fine = torch.isfinite(w)
    assert torch.equal(torch.isfinite(g), fine) and torch.equal(g[~fine & ~torch.isnan(w)], w[~fine & ~torch.isnan(w)]), what
    limit = (bound * (1 + 2 * HALF[got.dtype]) + HALF[got.dtype] * w.abs() + SMALLEST[got.dtype]).expand_as(w)
    off = (g - w).abs() - limit
    assert not (off[fine] > 0).any(), f"{what}: over the bound by {float(off[fine].max()):.3g}, limit {float(limit[fine].max()):.3g}"


# ------------------------------------------------------------------- norm
def norm_chain(H):
    """Roundings of a row's sum: a thread's own elements, its wave's and its block's; then r's own few."""
    return 32 + H / 256


def norm(x, w, eps, res=None):
    h = f64(x) + (f64(res) if res is not None else 0.0)
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    y = h * r * f64(w)
    # h, two products, and half of the sum's relative error in r with its quotient, root and reciprocal
    return h, r, y, y.abs() * U * (norm_chain(x.shape[1]) / 2 + 8)


def norm_grad(dy, h, w, eps, dres=None):
    dy, h, w = f64(dy), f64(h), f64(w)
    T, H = h.shape
    r = 1 / torch.sqrt((h * h).mean(-1, keepdim=True) + eps)
    g = dy * w
    dx = r * (g - h * r * r * (g * h).mean(-1, keepdim=True))
    size = r * (g.abs() + h.abs() * r * r * (g * h).abs().mean(-1, keepdim=True))
    bound = size * U * (2 * norm_chain(H) + 24)
    if dres is not None:
        dx = dx + f64(dres)
        bound = bound + 2 * U * f64(dres).abs()
    each = dy * h * r
    # a block adds every 512th row, a wave a sixteenth of the blocks' parts
    dw_bound = each.abs().sum(0) * U * (norm_chain(H) / 2 + 10 + T / 512 + 48)
    return dx, bound, each.sum(0), dw_bound


# --------------------------------------------------------------- adapters
def lora(x, A, B, ids, y, scaling=None, parts_bits=None):
    """(v, its bound, out, its bound); v is 0 where a token has no adapter."""
    x, A, B = f64(x), f64(A), f64(B)
    L, R, K = A.shape
    T, N = x.shape[0], B.shape[1]
    v, vb = torch.zeros(T, R, dtype=torch.float64), torch.zeros(T, R, dtype=torch.float64)
    out, ob = f64(y).clone(), torch.zeros(T, N, dtype=torch.float64)
    # the parts of v: two of 8 bits each to 2^-17 (fp16: 2^-22) for 16-bit outputs, exact for fp32 ones
    lost = 0.0 if y.dtype == torch.float32 else 2.0**-16
    for i in range(L):
        t = torch.nonzero(ids.cpu() == i)[:, 0]
        if not len(t):
            continue
        s = float(scaling[i]) if scaling is not None else 1.0
        v[t] = x[t] @ A[i].t()
        # (a product's sum inside the matrix unit may drop a bit more than a rounding: two steps each)
        vb[t] = x[t].abs() @ A[i].abs().t() * 4 * U * (K / 8 + 40)
        d = s * (v[t] @ B[i].t())
        size = abs(s) * (v[t].abs() @ B[i].abs().t())
        out[t] += d
        ob[t] = abs(s) * (vb[t] @ B[i].abs().t()) + size * (lost + 4 * U * (3 * R + 16)) + f64(y)[t].abs() * 4 * U * (3 * R + 16)
    return v, vb, out, ob


def lora_grad(dy, x, A, B, ids, v, scaling=None, dx=None):
    """((dx, bound) or None, dA, bound, dB, bound)"""
    dy, x, A, B, v = f64(dy), f64(x), f64(A), f64(B), f64(v)
    L, R, K = A.shape
    N, T = B.shape[1], x.shape[0]
    gx = f64(dx).clone() if dx is not None else None
    gb = torch.zeros(T, K, dtype=torch.float64)
    dA, dB = torch.zeros_like(A), torch.zeros_like(B)
    bA, bB = torch.zeros_like(A), torch.zeros_like(B)
    for i in range(L):
        t = torch.nonzero(ids.cpu() == i)[:, 0]
        if not len(t):
            continue
        s = float(scaling[i]) if scaling is not None else 1.0
        dv = dy[t] @ B[i]
        dvb = dy[t].abs() @ B[i].abs() * 4 * U * (N / 8 + 40)
        chain = 4 * U * (5 * len(t) + 64)
        dA[i], dB[i] = s * (dv.t() @ x[t]), s * (dy[t].t() @ v[t])
        bA[i] = abs(s) * (dvb.t() @ x[t].abs() + (dv.abs().t() @ x[t].abs()) * chain)
        bB[i] = abs(s) * (dy[t].abs().t() @ v[t].abs()) * chain
        if gx is not None:
            gx[t] += s * (dv @ A[i])
            size = abs(s) * (dv.abs() @ A[i].abs())
            gb[t] = abs(s) * (dvb @ A[i].abs()) + size * (2.0**-16 + 4 * U * (3 * R + 16)) + f64(dx)[t].abs() * 4 * U * (3 * R + 16)
    return (gx, gb) if gx is not None else None, dA, bA, dB, bB


# -------------------------------------------------------- log probabilities
def logprobs(logits, tokens, top=0):
    """(logp, entropy, lse, top ids, top logp) and the bounds of (logp, entropy, lse)."""
    l, tok = f64(logits), tokens.cpu().long()
    T, V = l.shape
    bad = torch.isnan(l).any(1) | (l == float("inf")).any(1)
    none = (l == float("-inf")).all(1)
    m = l.amax(-1, keepdim=True)
    d = torch.where(l == float("-inf"), float("-inf"), l - torch.where(torch.isfinite(m), m, 0.0))
    e = torch.exp(d)
    s = e.sum(-1)
    d0 = torch.where(e > 0, d, 0.0)
    lse = torch.where(none, float("-inf"), m[:, 0] + torch.log(s))
    mean = (e * d0).sum(-1) / s
    entropy = torch.where(none, 0.0, torch.log(s) - mean)
    lse, entropy = torch.where(bad, float("nan"), lse), torch.where(bad, float("nan"), entropy)
    asked = (tok >= 0) & (tok < V)
    lt = l.gather(1, tok.clamp(0, V - 1)[:, None])[:, 0]
    logp = torch.where(asked, torch.where(none, float("-inf"), lt - lse), 0.0)
    # every exp has an argument off by U |d| and an own error of two steps; a lane adds V / 256 values or fewer, and
    # is rescaled (two roundings, and the argument's) at most as often
    mean1, mean2 = (e * d0.abs()).sum(-1) / s, (e * d0 * d0).sum(-1) / s
    rel = 2 * U * (V / 64 + 80 + 3 * mean1)
    b_lse = rel + 2 * U * torch.where(torch.isfinite(lse), lse, 0.0).abs()
    b_ent = rel * (2 + mean1) + 6 * U * mean2 + 4 * U * (torch.log(s).abs() + mean1)
    b_lp = torch.where(asked, b_lse + 2 * U * torch.where(torch.isfinite(lt), lt, 0.0).abs(), 0.0)
    b_lp, b_ent, b_lse = (torch.where(bad | none, 0.0, b) for b in (b_lp, b_ent, b_lse))
    ids = tops = None
    if top:
        order = torch.sort(-torch.where(torch.isnan(l), float("-inf"), l), dim=1, stable=True).indices[:, :top]
        ids = torch.where(bad[:, None], -1, order).to(torch.int32)
        tops = torch.where(none[:, None], float("-inf"), l.gather(1, order) - lse[:, None])
    return (logp, entropy, lse, ids, tops), (b_lp, b_ent, b_lse)


def logprobs_grad(logits, tokens, lse, entropy, dlogp, dentropy):
    """(dlogits, bound), from lse and entropy as given."""
    l, tok, lse, h = f64(logits), tokens.cpu().long(), f64(lse), f64(entropy)
    T, V = l.shape
    asked = (tok >= 0) & (tok < V)
    g = torch.where(asked, f64(dlogp), 0.0) if dlogp is not None else torch.zeros(T, dtype=torch.float64)
    gh = f64(dentropy) if dentropy is not None else torch.zeros(T, dtype=torch.float64)
    lp = l - lse[:, None]
    p = torch.exp(lp)
    lp0 = torch.where(p > 0, lp, 0.0)
    inner = torch.where(p > 0, g[:, None] + gh[:, None] * (lp0 + h[:, None]), 0.0)
    d = -p * inner
    d.scatter_add_(1, tok.clamp(0, V - 1)[:, None], torch.where(asked, g, 0.0)[:, None])
    none = torch.isneginf(lse)
    d = torch.where(none[:, None], 0.0, d)
    size = p * (g.abs()[:, None] + gh.abs()[:, None] * (lp0.abs() + h.abs()[:, None]))
    bound = size * U * (16 + 4 * lp0.abs()) + 2 * U * d.abs()
    return d, torch.where(none[:, None], 0.0, bound)
