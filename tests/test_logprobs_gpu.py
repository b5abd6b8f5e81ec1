"""qw_logprobs and qw_logprobs_backward against 64 bits."""
import pytest
import torch

import qwq4
import _projection_ref as ref
from _projection_ref import TYPES, assert_close, f64

pytestmark = pytest.mark.gpu
INF = float("inf")


def make(seed, T, V, t, gpu, pad=0, off=0, kind="peaks"):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn(T, V + pad, generator=g) * 2 - 3
    if kind == "peaks":
        l[torch.arange(T), torch.randint(0, V, (T,), generator=g)] += 14
    elif kind == "masked":
        l[torch.rand(T, V + pad, generator=g) < 0.9] = -INF
        l[::3, V // 2:] = -INF
    elif kind == "ties":
        l = torch.randint(-2, 3, (T, V + pad), generator=g).float()
        l[l == 0] = -0.0
        l[:, ::5] += 0.0
    elif kind == "same":
        l[:] = 0.25
    elif kind == "lowest":
        l[:] = torch.finfo(TYPES[t]).min
        l[1::2, V // 3] = 1.0
    elif kind == "rising":
        l = torch.arange(T * (V + pad)).view(T, V + pad).float() / (T * V) * 20
    elif kind == "wide":
        l *= 30
    tokens = torch.randint(0, V, (T,), generator=g).to(torch.int32)
    tokens[3::7] = -1
    tokens[5::7] = V
    flat = torch.empty(T * (V + pad) + off, dtype=TYPES[t], device=gpu)
    flat[off:] = l.to(TYPES[t]).flatten().to(gpu)
    return flat[off:].view(T, V + pad)[:, :V], tokens.to(gpu), g


def check(logits, tokens, top, got):
    (logp, ent, lse, ids, tops), (blp, bent, blse) = ref.logprobs(logits, tokens, top)
    assert_close(got[0], logp, blp, "logp")
    assert_close(got[1], ent, bent, "entropy")
    assert_close(got[2], lse, blse, "lse")
    if top:
        assert torch.equal(got[3].cpu(), ids)
        assert_close(got[4], tops, (blse[:, None] + 2 * ref.U * torch.where(torch.isfinite(tops), tops, 0.0).abs()), "top")
    else:
        assert got[3] is None and got[4] is None


CASES = [(1, 1, 1), (1, 2, 2), (3, 7, 5), (2, 64, 64), (5, 513, 0), (1, 151936, 20), (1, 151669, 5), (4, 50257, 64),
         (33, 32000, 8), (64, 4099, 1), (65, 8192, 3), (300, 2051, 20), (2100, 777, 4), (700, 9001, 0)]


@pytest.mark.parametrize("T,V,top", CASES)
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_logprobs(gpu, T, V, top, t):
    print(f"logprobs T={T} V={V} top={top} {t}", flush=True)
    logits, tokens, _ = make(T + V, T, V, t, gpu)
    check(logits, tokens, top, qwq4.logprobs(logits, tokens, top=top))


@pytest.mark.parametrize("kind", ["masked", "ties", "same", "lowest", "rising", "wide"])
@pytest.mark.parametrize("T,V", [(1, 40000), (2, 12), (70, 5000), (2100, 300)])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_kinds_of_rows(gpu, kind, T, V, t):
    """Masked vocabularies, ties (also of both zeros), constant rows, the type's lowest value, every value the best so
    far: alternatives in order with ties by the lowest index."""
    print(f"logprobs {kind} T={T} V={V} {t}", flush=True)
    logits, tokens, _ = make(V, T, V, t, gpu, kind=kind)
    for top in (1, 7, min(64, V)):
        check(logits, tokens, min(top, V), qwq4.logprobs(logits, tokens, top=min(top, V)))


@pytest.mark.parametrize("pad,off", [(0, 1), (1, 0), (3, 5), (8, 0), (8, 3)])
@pytest.mark.parametrize("t", ["f32", "bf16"])
def test_strides_and_alignment(gpu, pad, off, t):
    for T, V in ((3, 9001), (70, 1030), (2050, 77)):
        logits, tokens, g = make(off, T, V, t, gpu, pad, off)
        got = qwq4.logprobs(logits, tokens, top=6)
        check(logits, tokens, 6, got)
        dlogp, dent = torch.randn(T, generator=g).to(gpu), torch.randn(T, generator=g).to(gpu)
        want, bound = ref.logprobs_grad(logits, tokens, got[2], got[1], dlogp, dent)
        for other in (0, 2):  # (the gradient's rows aligned as the logits', and otherwise)
            buf = torch.full((T, V + pad + other), 7.0, dtype=logits.dtype, device=gpu)
            d = qwq4.logprobs_backward(logits, tokens, got[2], got[1], dlogp, dent, dlogits=buf[:, :V])
            assert_close(d, want, bound, f"pad {pad + other}")
            assert (buf[:, V:] == 7).all()


@pytest.mark.parametrize("T,V", [(6, 30000), (2100, 200)])
def test_rows_without_an_answer(gpu, T, V):
    """Everything masked; a NaN; an infinity: each in its own row."""
    logits, tokens, g = make(1, T, V, "f32", gpu)
    logits, tokens = logits.contiguous(), tokens.clamp(0, V - 1)
    logits[1] = -INF
    logits[2, V - 1] = float("nan")
    logits[3, 0] = INF
    logits[4] = float("nan")
    logits[5, 1:] = -INF
    got = qwq4.logprobs(logits, tokens, top=5)
    check(logits, tokens, 5, got)
    assert got[1][1] == 0 and got[0][1] == -INF and (got[4][1] == -INF).all() and got[3][1].tolist() == [0, 1, 2, 3, 4]
    assert got[1][5] == 0 and got[3][5].tolist() == [0, 1, 2, 3, 4] and (got[4][5, 1:] == -INF).all()
    dlogp = torch.ones(T, device=gpu)
    d = qwq4.logprobs_backward(logits, tokens, got[2], got[1], dlogp, dlogp)
    assert (d[1] == 0).all() and torch.isnan(d[2]).all() and torch.isnan(d[3]).all() and torch.isfinite(d[5]).all()
    assert torch.isfinite(d[0]).all()


def test_bad_tokens_of_bad_rows(gpu):
    """A token outside the vocabulary has logp 0 in any row."""
    logits = torch.full((3, 100), -INF, device=gpu)
    logits[1] = 1.0
    tokens = torch.tensor([-5, 100, 2**31 - 1], dtype=torch.int32, device=gpu)
    assert (qwq4.logprobs(logits, tokens)[0] == 0).all()


@pytest.mark.parametrize("T,V", [(1, 1), (1, 151936), (7, 30), (33, 5001), (601, 2048), (2, 70001)])
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("kind", ["peaks", "masked"])
def test_backward(gpu, T, V, t, kind):
    print(f"logprobs_backward T={T} V={V} {t} {kind}", flush=True)
    logits, tokens, g = make(T + V, T, V, t, gpu, kind=kind)
    _, ent, lse, _, _ = qwq4.logprobs(logits, tokens)
    dlogp, dent = torch.randn(T, generator=g).to(gpu), torch.randn(T, generator=g).to(gpu)
    for a, b in ((dlogp, dent), (dlogp, None), (None, dent)):
        d = qwq4.logprobs_backward(logits, tokens, lse, ent if b is not None else None, a, b)
        want, bound = ref.logprobs_grad(logits, tokens, lse, ent, a, b)
        assert_close(d, want, bound, f"{a is not None} {b is not None}")
    same = logits.clone()
    assert qwq4.logprobs_backward(same, tokens, lse, ent, dlogp, dent, dlogits=same) is same
    assert torch.equal(same, qwq4.logprobs_backward(logits, tokens, lse, ent, dlogp, dent))


def test_backward_is_the_derivative(gpu):
    """Along random directions, against central differences in 64 bits."""
    T, V, step = 5, 300, 1e-5
    logits, tokens, g = make(3, T, V, "f32", gpu)
    _, ent, lse, _, _ = qwq4.logprobs(logits, tokens)
    dlogp, dent = torch.randn(T, generator=g).to(gpu), torch.randn(T, generator=g).to(gpu)
    d = qwq4.logprobs_backward(logits, tokens, lse, ent, dlogp, dent)
    (_, _, _, _, _), (_, bent, blse) = ref.logprobs(logits, tokens)
    _, bound = ref.logprobs_grad(logits, tokens, lse, ent, dlogp, dent)
    p = torch.exp(f64(logits) - f64(lse)[:, None])
    size = f64(dlogp).abs()[:, None] + f64(dent).abs()[:, None] * (2 + (f64(logits) - f64(lse)[:, None]).abs() + f64(ent)[:, None])
    # (lse and entropy are rounded: p moves by lse's error, the entropy's part by its own)
    bound = bound + p * (size * (blse + 2.0**-20)[:, None] + f64(dent).abs()[:, None] * (bent + 2.0**-20)[:, None])
    for seed in range(5):
        e = torch.randn(T, V, generator=g).double()

        def f(s):
            (logp, h, *_), _ = ref.logprobs(f64(logits) + s * e, tokens)
            return float((logp * f64(dlogp)).sum() + (h * f64(dent)).sum())

        slope = (f(step) - f(-step)) / (2 * step)
        got = float((f64(d) * e).sum())
        limit = float(((bound + ref.U * f64(d).abs()) * e.abs()).sum()) + 1e-7 * float(size.sum())
        assert abs(got - slope) <= limit, (got, slope, limit)


def test_fp16_gradient_overflows(gpu):
    logits, tokens = torch.zeros(2, 64, dtype=torch.float16, device=gpu), torch.zeros(2, dtype=torch.int32, device=gpu)
    _, ent, lse, _, _ = qwq4.logprobs(logits, tokens)
    d = qwq4.logprobs_backward(logits, tokens, lse, ent, torch.tensor([1e6, 1.0], device=gpu))
    assert torch.isposinf(d[0, 0]) and torch.isfinite(d[1]).all()


def test_offsets_past_32_bits(gpu):
    """The last rows of more than 2^32 bytes."""
    T, V = 20000, 60007
    logits = torch.zeros(T, V, device=gpu)
    few, tokens, g = make(5, 3, V, "f32", gpu)
    logits[-3:] = few
    tok = torch.zeros(T, dtype=torch.int32, device=gpu)
    tok[-3:] = torch.tensor([5, V - 1, -1], dtype=torch.int32)
    got = qwq4.logprobs(logits, tok, top=3)
    check(logits[-3:], tok[-3:], 3, tuple(x[-3:] for x in got))
    dlogp = torch.ones(T, device=gpu)
    d = qwq4.logprobs_backward(logits, tok, got[2], got[1], dlogp, dlogp, dlogits=logits.clone())
    want, bound = ref.logprobs_grad(logits[-3:], tok[-3:], got[2][-3:], got[1][-3:], dlogp[-3:], dlogp[-3:])
    assert_close(d[-3:], want, bound)


@pytest.mark.parametrize("top", [31, 32, 33, 63, 64])
@pytest.mark.parametrize("T,V", [(1, 151936), (9, 20011), (70, 9001), (600, 2500)])
@pytest.mark.parametrize("kind", ["peaks", "wide"])
def test_many_alternatives(gpu, T, V, top, kind):
    """Where the groups that bound the alternatives change."""
    print(f"logprobs T={T} V={V} top={top} {kind}", flush=True)
    logits, tokens, _ = make(T + top, T, V, "bf16", gpu, kind=kind)
    check(logits, tokens, top, qwq4.logprobs(logits, tokens, top=top))


@pytest.mark.parametrize("kind,top", [("peaks", 20), ("peaks", 64), ("ties", 3)])
def test_very_long_rows(gpu, kind, top):
    """Several steps to each largest value that is kept."""
    logits, tokens, _ = make(top, 1, 17_500_001, "f32", gpu, kind=kind)
    check(logits, tokens, top, qwq4.logprobs(logits, tokens, top=top))


# ------------------------------------------- logits far from zero
def apart(logits, tokens, top):
    """(logp, entropy, top logp) in 64 bits with bounds that know the logits' differences only: every sum's relative error
    (as in the other cases' bounds), and roundings of l - m, of log S and of their difference. No bound grows with lse."""
    l, tok = f64(logits), tokens.cpu().long()
    V = l.shape[1]
    d = l - l.amax(-1, keepdim=True)
    e = torch.exp(d)
    s = e.sum(-1)
    d0 = torch.where(e > 0, d, 0.0)
    mean1 = (e * d0.abs()).sum(-1) / s
    log_s = torch.log(s)
    off = 2 * ref.U * (V / 64 + 80 + 3 * mean1) + 4 * ref.U * log_s.abs()

    def at(i):
        dv = d.gather(1, i)
        return dv - log_s[:, None], off[:, None] + 2 * ref.U * dv.abs() + 2 * ref.U * (dv - log_s[:, None]).abs()

    asked = (tok >= 0) & (tok < V)
    lp, b = at(tok.clamp(0, V - 1)[:, None])
    logp = torch.where(asked, lp[:, 0], 0.0), torch.where(asked, b[:, 0], 0.0)
    order = torch.sort(-l, dim=1, stable=True).indices[:, :top]
    return logp, at(order), order


SHIFTS = [(1e3, "f32"), (1e5, "f32"), (-3e6, "f32"), (-1e3, "bf16"), (3e4, "f16"), (4096.0, "same"), (-1e9, "same"),
          (torch.finfo(torch.float32).min, "same")]


def shifted(seed, T, V, shift, t, gpu, pad=0, off=0):
    logits, tokens, g = make(seed, T, V, "f32" if t == "same" else t, gpu, pad, off)
    if t == "same":
        logits[:] = shift
    else:
        logits.copy_(logits.float() + shift)
    return logits, tokens, g


@pytest.mark.parametrize("shift,t", SHIFTS)
@pytest.mark.parametrize("T,V", [(1, 1000), (3, 151936), (2100, 300)])
def test_shifted_rows(gpu, T, V, shift, t):
    """Rows far from zero, constant finite ones among them (logp is -log V there): as exact as rows next to it."""
    print(f"logprobs shifted by {shift} T={T} V={V} {t}", flush=True)
    logits, tokens, _ = shifted(T, T, V, shift, t, gpu)
    got = qwq4.logprobs(logits, tokens, top=7)
    (logp, blp), (tops, btop), order = apart(logits, tokens, 7)
    assert torch.equal(got[3].cpu().long(), order)
    assert_close(got[0], logp, blp, "logp")
    assert_close(got[4], tops, btop, "top")


@pytest.mark.parametrize("shift,t", SHIFTS)
@pytest.mark.parametrize("T,V,pad,off", [(1, 1000, 0, 0), (3, 70001, 3, 1), (601, 2048, 0, 0), (2, 20000, 8, 0)])
def test_backward_of_shifted_rows(gpu, T, V, pad, off, shift, t):
    """The gradient by the definition, not by a rounded lse: in rows of their own, of another alignment, in place."""
    print(f"logprobs_backward shifted by {shift} T={T} V={V} {t}", flush=True)
    logits, tokens, g = shifted(T + V, T, V, shift, t, gpu, pad, off)
    _, ent, lse, _, _ = qwq4.logprobs(logits, tokens)
    dlogp, dent = torch.randn(T, generator=g).to(gpu), torch.randn(T, generator=g).to(gpu)
    l, tok = f64(logits), tokens.cpu().long()
    d = l - l.amax(-1, keepdim=True)
    lp = d - torch.log(torch.exp(d).sum(-1, keepdim=True))
    p, h = torch.exp(lp), -(torch.exp(lp) * lp).sum(-1, keepdim=True)
    asked = (tok >= 0) & (tok < V)
    gl, gh = torch.where(asked, f64(dlogp), 0.0)[:, None], f64(dent)[:, None]
    want = -p * (gl + gh * (lp + h))
    want.scatter_add_(1, tok.clamp(0, V - 1)[:, None], gl)
    # p: its argument's roundings, and the row's sum, whose relative error shows in it; where the sum is not made anew
    # (lse up to 64 for fp32 rows, 1024 for 16-bit ones), half a step of lse. The entropy is the forward's.
    mean1 = (p * (d - 0).abs()).sum(-1, keepdim=True)
    off_lp = 2 * ref.U * (V / 64 + 80 + 3 * mean1) + ref.U * (16 + 4 * lp.abs()) + (2.0**-19 if t in ("f32", "same") else 2.0**-15)
    off_h = (ref.logprobs(logits, tokens)[1][1])[:, None]
    size = gl.abs() + gh.abs() * (lp.abs() + h.abs())
    bound = p * (size * off_lp + gh.abs() * (off_lp + off_h)) + 2 * ref.U * want.abs()
    other = torch.empty(T, V + 1, dtype=logits.dtype, device=gpu)[:, :V]
    for out in (None, other):
        assert_close(qwq4.logprobs_backward(logits, tokens, lse, ent, dlogp, dent, dlogits=out), want, bound)
    assert_close(qwq4.logprobs_backward(logits, tokens, lse, ent, dlogp, dent, dlogits=logits), want, bound, "in place")


@pytest.mark.parametrize("shift", [0.0, 100.0, -3e4])
def test_backward_of_a_shard(gpu, shift):
    """A shard of the vocabulary with the lse and the entropy of the whole row: the probabilities are the whole row's."""
    T, V, own = 5, 4000, 1000
    logits, tokens, g = shifted(3, T, V, shift, "f32", gpu)
    _, ent, lse, _, _ = qwq4.logprobs(logits, tokens)
    dlogp, dent = torch.randn(T, generator=g).to(gpu), torch.randn(T, generator=g).to(gpu)
    for r in range(V // own):
        part, tok = logits[:, r * own:(r + 1) * own], tokens - r * own
        d = qwq4.logprobs_backward(part, tok, lse, ent, dlogp, dent)
        want, bound = ref.logprobs_grad(part, tok, lse, ent, dlogp, dent)
        # (a shard that holds nearly everything may have half a step of lse put right: its p moves by as much)
        p = torch.exp(f64(part) - f64(lse)[:, None])
        lp = (f64(part) - f64(lse)[:, None]).abs()
        size = p * (f64(dlogp).abs()[:, None] + f64(dent).abs()[:, None] * (1 + lp + f64(ent)[:, None]))
        assert_close(d, want, bound + 2 * size * 2 * ref.U * f64(lse).abs()[:, None], f"shard {r}")


def test_outputs_are_tensors_of_their_own(gpu):
    """What torch asks of a Function's outputs: in-place work on one, with the others' graphs still read; and no output
    keeps another's memory."""
    T, V = 6, 300
    logits, tokens, g = make(8, T, V, "f32", gpu)

    class LogProbs(torch.autograd.Function):
        @staticmethod
        def forward(ctx, l):
            logp, entropy, lse, _, _ = qwq4.logprobs(l, tokens)
            ctx.save_for_backward(l, lse, entropy)
            return logp, entropy

        @staticmethod
        def backward(ctx, dlogp, dentropy):
            l, lse, entropy = ctx.saved_tensors
            return qwq4.logprobs_backward(l, tokens, lse, entropy, dlogp.contiguous(), dentropy.contiguous())

    leaf = logits.clone().requires_grad_()
    logp, entropy = LogProbs.apply(leaf)
    mask = torch.tensor([1.0, 0, 1, 1, 0, 1], device=gpu)
    logp.mul_(mask)
    (logp.sum() + 0.5 * entropy.sum()).backward()
    _, ent, lse, _, _ = got = qwq4.logprobs(logits, tokens, top=3)
    assert torch.equal(leaf.grad, qwq4.logprobs_backward(logits, tokens, lse, ent, mask, torch.full((T,), 0.5, device=gpu)))
    assert len({t.untyped_storage().data_ptr() for t in got}) == 5
    assert all(t._base is None and t.untyped_storage().nbytes() == t.numel() * t.element_size() for t in got)


@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
def test_gradient_of_a_masked_token(gpu, t):
    """A masked logit has no gradient, but for a token that is itself masked: its logp is -inf, and its dlogp passes on to
    its logit as the formula has it (and torch's log_softmax)."""
    T, V = 5, 203
    logits, tokens, g = make(12, T, V, t, gpu)
    tokens = tokens.clamp(0, V - 1)
    at = torch.arange(T, device=gpu)
    logits[:, 50:90] = -INF
    tokens[:3] = 60
    logp, ent, lse, _, _ = qwq4.logprobs(logits, tokens)
    assert (logp[:3] == -INF).all() and torch.isfinite(logp[3:]).all()
    dlogp, dent = torch.randn(T, generator=g).to(gpu), torch.randn(T, generator=g).to(gpu)
    d = qwq4.logprobs_backward(logits, tokens, lse, ent, dlogp, dent)
    want, bound = ref.logprobs_grad(logits, tokens, lse, ent, dlogp, dent)
    assert_close(d, want, bound)
    assert torch.equal(d[at[:3], 60], dlogp[:3].to(d.dtype))
    masked = d[:, 50:90].clone()
    masked[:3, 10] = 0
    assert (masked == 0).all()
    l = logits.double().cpu().requires_grad_()
    torch.log_softmax(l, -1)[torch.arange(T), tokens.cpu().long()].backward(f64(dlogp))
    d = qwq4.logprobs_backward(logits, tokens, lse, ent, dlogp)
    assert_close(d, l.grad, ref.logprobs_grad(logits, tokens, lse, ent, dlogp, None)[1] + 2.0**-18 * torch.exp(f64(logits) - f64(lse)[:, None]) * f64(dlogp).abs()[:, None])
