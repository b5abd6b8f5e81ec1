"""The operators around a projection together, as a served token and a training step
use them: each stage against 64 bits of what the stage got, then on a stream of its
own, two runs at once, under autograd, and captured and replayed with new inputs
between eager calls."""
import pytest
import torch

import qwq4
import _projection_ref as ref
from _projection_ref import assert_close, f64

pytestmark = pytest.mark.gpu
EPS = 1e-5


# ----------------------------------------------------------------- serving
class Serve:
    """norm + residual (rows in 8 and 16 bits) -> W8A8 projection -> adapters -> norm -> log probabilities"""

    def __init__(self, seed, T, H, V, R, L, gpu, top):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
        self.top, self.L = top, L
        self.w1, self.w2 = (1 + 0.1 * rnd(H)).to(gpu), (1 + 0.1 * rnd(V)).bfloat16().to(gpu)
        self.W, self.sw = torch.randint(-127, 128, (V, H), generator=g).to(torch.int8).to(gpu), (rnd(V).abs() * 1e-3).to(gpu)
        self.A, self.B = (rnd(L, R, H) * H**-0.5).bfloat16().to(gpu), (rnd(L, V, R) * R**-0.5).bfloat16().to(gpu)
        self.scaling = (0.5 + torch.rand(L, generator=g)).to(gpu)
        self.x, self.res = torch.empty(T, H, dtype=torch.bfloat16, device=gpu), torch.empty(T, H, device=gpu)
        self.ids, self.tokens = (torch.empty(T, dtype=torch.int32, device=gpu) for _ in range(2))
        self.T, self.H, self.V = T, H, V
        self.fill(seed)

    def fill(self, seed):
        g = torch.Generator().manual_seed(seed + 1000)
        self.x.copy_(torch.randn(self.T, self.H, generator=g))
        self.res.copy_(torch.randn(self.T, self.H, generator=g))
        self.ids.copy_(torch.randint(-1, self.L, (self.T,), generator=g))
        self.tokens.copy_(torch.randint(0, self.V, (self.T,), generator=g))

    def run(self):
        q, scale, h = qwq4.rms_norm_i8(self.x, self.w1, EPS, residual=self.res)
        n, _ = qwq4.rms_norm(self.x, self.w1, EPS, residual=self.res)
        y0 = qwq4.gemm_w8a8(self.W, self.sw, q, scale, y_dtype=torch.bfloat16)
        y = qwq4.lora(n, self.A, self.B, self.ids, y0, scaling=self.scaling, out=torch.empty_like(y0))
        z = qwq4.rms_norm(y, self.w2, EPS, y_dtype=torch.float32)
        return (q, scale, h, n, y0, y, z) + qwq4.logprobs(z, self.tokens, top=self.top)


SERVE = [(1, 640, 1000, 16, 3, 5), (37, 512, 2056, 16, 8, 20), (130, 272, 4104, 40, 2, 1)]


@pytest.mark.parametrize("T,H,V,R,L,top", SERVE)
def test_served_tokens(gpu, T, H, V, R, L, top):
    s = Serve(T, T, H, V, R, L, gpu, top)
    q, scale, h, n, y0, y, z, *lp = s.run()
    wh, wr, wn, bn = ref.norm(s.x, s.w1, EPS, s.res)
    assert_close(h, wh, wh.abs() * ref.U)
    assert_close(n, wn, bn)
    # a row in 8 bits is off by half a step of its scale, and by what the scale is off
    assert ((f64(q) * f64(scale)[:, None] - wn).abs() <= f64(scale)[:, None] * 0.5001 + 2 * bn).all()
    exact = (f64(q) @ f64(s.W).t()) * f64(s.sw) * f64(scale)[:, None]
    assert_close(y0, exact, exact.abs() * 4 * ref.U)
    _, _, wy, by = ref.lora(n, s.A, s.B, s.ids, y0, s.scaling)
    assert_close(y, wy, by)
    _, _, wz, bz = ref.norm(y, s.w2, EPS)
    assert_close(z, wz, bz)
    (wlp, went, wlse, wids, wtop), (blp, bent, blse) = ref.logprobs(z, s.tokens, top)
    for got, want, bound in zip(lp, (wlp, went, wlse), (blp, bent, blse)):
        assert_close(got, want, bound)
    assert torch.equal(lp[3].cpu(), wids)
    assert_close(lp[4], wtop, (blse[:, None] + 2 * ref.U * wtop.abs()).expand_as(wtop))


@pytest.mark.parametrize("T,H,V,R,L,top", SERVE)
def test_served_tokens_streams_and_graph(gpu, T, H, V, R, L, top):
    a, b = Serve(1, T, H, V, R, L, gpu, top), Serve(2, T, H, V, R, L, gpu, top)
    want = [a.run(), b.run()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):  # two runs at once
        got = []
        for s, stream in zip((a, b), streams):
            with torch.cuda.stream(stream):
                got.append(s.run())
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = a.run()
    with torch.cuda.graph(other):
        captured_b = b.run()
    for seed in (3, 4, 5, 6):
        a.fill(seed)
        b.fill(seed + 50)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured + captured_b]
        eager = a.run() + b.run()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, eager))


# ---------------------------------------------------------------- training
class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, res):
        y, h = qwq4.rms_norm(x, w, EPS, residual=res)
        ctx.save_for_backward(h, w)
        return y, h

    @staticmethod
    def backward(ctx, dy, dh):
        dx, dw = qwq4.rms_norm_backward(dy, *ctx.saved_tensors, EPS, dres=dh)
        return dx, dw, dx


class Adapters(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, A, B, ids, y, scaling):
        v = torch.empty(x.shape[0], A.shape[1], device=x.device)
        ctx.save_for_backward(x, A, B, ids, v, scaling)
        return qwq4.lora(x, A, B, ids, y, scaling=scaling, out=torch.empty_like(y), v=v)

    @staticmethod
    def backward(ctx, dy):
        x, A, B, ids, v, scaling = ctx.saved_tensors
        dx, dA, dB = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling, dx=torch.zeros_like(x))
        return dx, dA, dB, None, dy, None


class LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens):
        logp, entropy, lse, _, _ = qwq4.logprobs(logits, tokens)
        ctx.save_for_backward(logits, tokens, lse, entropy)
        return logp, entropy

    @staticmethod
    def backward(ctx, dlogp, dentropy):
        logits, tokens, lse, entropy = ctx.saved_tensors
        return qwq4.logprobs_backward(logits, tokens, lse, entropy, dlogp.contiguous(), dentropy.contiguous()), None


class Train:
    """norm + residual -> adapters over a frozen projection's rows -> log probabilities, and all their gradients"""

    def __init__(self, seed, T, H, V, R, L, t, gpu):
        g = torch.Generator().manual_seed(seed)
        rnd = lambda *s: torch.randn(*s, generator=g).to(t).to(gpu)  # noqa: E731
        self.x, self.res, self.w, self.y0, self.dh = rnd(T, H), rnd(T, H), rnd(H), rnd(T, V), rnd(T, H)
        self.A, self.B = rnd(L, R, H) * H**-0.5, rnd(L, V, R) * R**-0.5
        self.scaling = (0.5 + torch.rand(L, generator=g)).to(gpu)
        self.ids = torch.randint(-1, L, (T,), generator=g).to(torch.int32).to(gpu)
        self.tokens = torch.randint(-1, V, (T,), generator=g).to(torch.int32).to(gpu)
        self.dlogp, self.dentropy = (torch.randn(T, generator=g).to(gpu) for _ in range(2))
        self.sizes = T, H, V, R, L, gpu

    def fill(self, seed):
        T, H, V, R, L, gpu = self.sizes
        other = Train(seed, T, H, V, R, L, self.x.dtype, gpu)
        for name in ("x", "res", "y0", "ids", "tokens", "dlogp", "dentropy", "dh"):
            getattr(self, name).copy_(getattr(other, name))

    def run(self):
        n, h = qwq4.rms_norm(self.x, self.w, EPS, residual=self.res)
        v = torch.zeros(n.shape[0], self.A.shape[1], device=n.device)
        y = qwq4.lora(n, self.A, self.B, self.ids, self.y0, scaling=self.scaling, out=torch.empty_like(self.y0), v=v)
        logp, entropy, lse, _, _ = qwq4.logprobs(y, self.tokens)
        dy = qwq4.logprobs_backward(y, self.tokens, lse, entropy, self.dlogp, self.dentropy)
        dn, dA, dB = qwq4.lora_backward(dy, n, self.A, self.B, self.ids, v, scaling=self.scaling, dx=torch.zeros_like(n))
        dx, dw = qwq4.rms_norm_backward(dn, h, self.w, EPS, dres=self.dh)
        return n, h, v, y, logp, entropy, lse, dy, dn, dA, dB, dx, dw


TRAIN = [(1, 64, 200, 8, 1), (37, 520, 1032, 16, 4), (300, 256, 2048, 40, 3), (1100, 128, 520, 64, 2)]


@pytest.mark.parametrize("T,H,V,R,L", TRAIN)
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_training_step(gpu, T, H, V, R, L, t):
    s = Train(T, T, H, V, R, L, t, gpu)
    n, h, v, y, logp, entropy, lse, dy, dn, dA, dB, dx, dw = s.run()
    _, _, wn, bn = ref.norm(s.x, s.w, EPS, s.res)
    assert_close(n, wn, bn)
    _, _, wy, by = ref.lora(n, s.A, s.B, s.ids, s.y0, s.scaling)
    assert_close(y, wy, by)
    (wlp, went, wlse, _, _), (blp, bent, blse) = ref.logprobs(y, s.tokens)
    for got, want, bound in zip((logp, entropy, lse), (wlp, went, wlse), (blp, bent, blse)):
        assert_close(got, want, bound)
    wdy, bdy = ref.logprobs_grad(y, s.tokens, lse, entropy, s.dlogp, s.dentropy)
    assert_close(dy, wdy, bdy)
    (wdn, bdn), wA, bA, wB, bB = ref.lora_grad(dy, n, s.A, s.B, s.ids, v, s.scaling, torch.zeros_like(n))
    for got, want, bound in ((dn, wdn, bdn), (dA, wA, bA), (dB, wB, bB)):
        assert_close(got, want, bound)
    wdx, bdx, wdw, bdw = ref.norm_grad(dn, h, s.w, EPS, s.dh)
    assert_close(dx, wdx, bdx)
    assert_close(dw, wdw, bdw)

    # under autograd: the same calls, the same bits
    leaves = [p.clone().requires_grad_() for p in (s.x, s.w, s.res, s.A, s.B, s.y0)]
    ln, lh = Norm.apply(*leaves[:3])
    ly = Adapters.apply(ln, leaves[3], leaves[4], s.ids, leaves[5], s.scaling)
    llp, lent = LogProbs.apply(ly, s.tokens)
    torch.autograd.backward((llp, lent, lh), (s.dlogp, s.dentropy, s.dh))
    for leaf, want in zip(leaves, (dx, dw, dx, dA, dB, dy)):
        assert torch.equal(leaf.grad, want.to(t))


@pytest.mark.parametrize("T,H,V,R,L", TRAIN)
def test_training_step_streams_and_graph(gpu, T, H, V, R, L):
    a, b = Train(1, T, H, V, R, L, torch.bfloat16, gpu), Train(2, T, H, V, R, L, torch.float16, gpu)
    want = [a.run(), b.run()]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, stream in zip((a, b), streams):
            with torch.cuda.stream(stream):
                got.append(s.run())
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for g, w in zip(got, want) for x, y in zip(g, w))
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = a.run()
    with torch.cuda.graph(other):
        captured_b = b.run()
    for seed in (3, 4, 5, 6):
        a.fill(seed)
        b.fill(seed + 50)
        graph.replay()
        other.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured + captured_b]
        eager = a.run() + b.run()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(got, eager))


# ------------------------------------------------------------- long batches
@pytest.mark.parametrize("T,K,N,R,L", [(16500, 72, 136, 16, 3), (33000, 64, 72, 64, 2), (70000, 64, 72, 8, 2),
                                       (263000, 8, 8, 8, 2)])
@pytest.mark.parametrize("t", [torch.bfloat16, torch.float16])
def test_adapters_of_long_batches(gpu, T, K, N, R, L, t):
    """Two and four tiles of tokens a block, and parts of more tokens than are listed at once."""
    print(f"lora T={T} K={K} N={N} R={R} L={L} {t}", flush=True)
    g = torch.Generator().manual_seed(T)
    rnd = lambda *s: torch.randn(*s, generator=g).to(t).to(gpu)  # noqa: E731
    x, A, B, y, dy, dx = rnd(T, K), rnd(L, R, K) * K**-0.5, rnd(L, N, R) * R**-0.5, rnd(T, N), rnd(T, N), rnd(T, K)
    ids = torch.randint(-1, L, (T,), generator=g).to(torch.int32).to(gpu)
    v = torch.zeros(T, R, device=gpu)
    got = qwq4.lora(x, A, B, ids, y, out=torch.empty_like(y), v=v)
    wv, bv, want, bound = ref.lora(x, A, B, ids, y)
    assert_close(v, wv, bv, "v")
    assert_close(got, want, bound, "out")
    out, dA, dB = qwq4.lora_backward(dy, x, A, B, ids, v, dx=dx, dx_out=torch.empty_like(dx))
    (wx, bx), wA, bA, wB, bB = ref.lora_grad(dy, x, A, B, ids, v, None, dx)
    assert_close(out, wx, bx, "dx")
    assert_close(dA, wA, bA, "dA")
    assert_close(dB, wB, bB, "dB")
