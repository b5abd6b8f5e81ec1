"""qw_lora and qw_lora_backward against 64 bits."""
import pytest
import torch

import qwq4
import _projection_ref as ref
from _projection_ref import TYPES, assert_close, f64

pytestmark = pytest.mark.gpu
GUARD = 77.0


def make(seed, T, K, N, R, L, t, gpu, kind="mixed"):
    g = torch.Generator().manual_seed(seed)
    dt = TYPES[t]
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x, A, B = rnd(T, K), rnd(L, R, K) * K**-0.5, rnd(L, N, R) * R**-0.5
    if kind == "runs":  # requests one after another
        ids = torch.sort(torch.randint(-1, L, (T,), generator=g)).values
    elif kind == "none":
        ids = torch.full((T,), -1)
    elif kind == "one":
        ids = torch.full((T,), L - 1)
    else:
        ids = torch.randint(-1, L + 1, (T,), generator=g)
        ids[::11] = -(2**31)
        ids[5::13] = 2**31 - 1
    scaling = 0.5 + torch.rand(L, generator=g)
    to = lambda v, d=dt: v.to(d).to(gpu)  # noqa: E731
    return to(x), to(A), to(B), ids.to(torch.int32).to(gpu), scaling.to(gpu), g


CASES = [(1, 64, 64, 16, 1, "one"), (1, 4096, 256, 16, 8, "one"), (2, 8, 8, 8, 2, "mixed"), (15, 136, 72, 24, 3, "mixed"),
         (16, 64, 1032, 32, 4, "runs"), (17, 520, 264, 40, 2, "mixed"), (37, 1536, 640, 16, 32, "mixed"),
         (63, 640, 328, 64, 5, "mixed"), (64, 72, 64, 128, 3, "runs"), (65, 2560, 320, 120, 2, "mixed"),
         (130, 256, 200, 16, 64, "mixed"), (601, 264, 520, 16, 4, "runs"), (1030, 128, 136, 8, 3, "runs"),
         (40, 64, 64, 16, 3, "none"), (300, 4096, 64, 56, 1, "one")]


@pytest.mark.parametrize("T,K,N,R,L,kind", CASES)
@pytest.mark.parametrize("t,y", [("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32"), ("f16", "bf16")])
def test_lora(gpu, T, K, N, R, L, kind, t, y):
    print(f"lora T={T} K={K} N={N} R={R} L={L} {kind} {t} {y}", flush=True)
    x, A, B, ids, scaling, g = make(T + K + R, T, K, N, R, L, t, gpu, kind)
    ys = torch.randn(T, N, generator=g).to(TYPES[y]).to(gpu)
    v = torch.full((T, R), GUARD, device=gpu)
    out = torch.full((T, N + 8), GUARD, dtype=ys.dtype, device=gpu)
    got = qwq4.lora(x, A, B, ids, ys, scaling=scaling, out=out[:, :N], v=v)
    wv, bv, want, bound = ref.lora(x, A, B, ids, ys, scaling)
    has = ((ids >= 0) & (ids < L)).cpu()
    assert_close(v[has.to(gpu)], wv[has], bv[has], "v")
    assert (v[~has.to(gpu)] == GUARD).all()
    assert_close(got, want, bound, "out")
    assert torch.equal(got[~has.to(gpu)], ys[~has.to(gpu)]) and (out[:, N:] == GUARD).all()
    same = ys.clone()
    assert qwq4.lora(x, A, B, ids, same, scaling=scaling) is same and torch.equal(same, got)
    ones = qwq4.lora(x, A, B, ids, ys.clone())
    assert torch.equal(ones, qwq4.lora(x, A, B, ids, ys.clone(), scaling=torch.ones_like(scaling)))


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_rows_do_not_depend_on_the_batch(gpu, t):
    T, K, N, R, L = 300, 1544, 392, 32, 6
    x, A, B, ids, scaling, g = make(1, T, K, N, R, L, t, gpu)
    for y in ("f32", t):
        ys = torch.randn(T, N, generator=g).to(TYPES[y]).to(gpu)
        whole = qwq4.lora(x, A, B, ids, ys, scaling=scaling, out=torch.empty_like(ys))
        for at in ([0], [7, 8], list(range(100, 137)), list(range(299, -1, -1))):
            i = torch.tensor(at, device=gpu)
            part = qwq4.lora(x[i], A, B, ids[i], ys[i], scaling=scaling)
            assert torch.equal(part, whole[i])


def test_strided_rows(gpu):
    T, K, N, R, L = 50, 128, 96, 16, 3
    x, A, B, ids, scaling, g = make(2, T, K, N, R, L, "bf16", gpu)
    wide_x, wide_y = torch.zeros(T, K + 24, dtype=x.dtype, device=gpu), torch.zeros(T, 3 * N, device=gpu)
    wide_x[:, 8:8 + K] = x
    wide_y[:] = torch.randn(T, 3 * N, generator=g).to(gpu)
    before = wide_y.clone()
    qwq4.lora(wide_x[:, 8:8 + K], A, B, ids, wide_y[:, N:2 * N], scaling=scaling)  # one slice of a fused projection
    assert torch.equal(wide_y[:, N:2 * N], qwq4.lora(x, A, B, ids, before[:, N:2 * N].contiguous(), scaling=scaling))
    assert torch.equal(wide_y[:, :N], before[:, :N]) and torch.equal(wide_y[:, 2 * N:], before[:, 2 * N:])


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_bad_values_stay_with_their_token(gpu, t):
    """A NaN or an infinity in one token's row, or in the weights of its adapter, reaches no other token."""
    T, K, N, R, L = 40, 128, 128, 16, 4
    x, A, B, ids, scaling, g = make(3, T, K, N, R, L, t, gpu)
    ids[:] = torch.arange(T) % 3  # (tokens of three adapters in every tile, none of the fourth)
    for y in (t, "f32"):
        ys = torch.randn(T, N, generator=g).to(TYPES[y]).to(gpu)
        clean = qwq4.lora(x, A, B, ids, ys, scaling=scaling, out=torch.empty_like(ys))
        x2, A2, B2 = x.clone(), A.clone(), B.clone()
        x2[4, 5], x2[7, 0] = float("nan"), float("inf")
        A2[2, 3, 9], B2[2, 11, 2], B2[3] = float("nan"), float("inf"), float("nan")
        got = qwq4.lora(x2, A2, B2, ids, ys, scaling=scaling, out=torch.empty_like(ys))
        good = (ids != 2) & (torch.arange(T, device=gpu) != 4) & (torch.arange(T, device=gpu) != 7)
        assert torch.equal(got[good], clean[good]) and torch.isnan(got[4]).all()
        dy, dx = torch.randn(T, N, generator=g).to(x.dtype).to(gpu), torch.randn(T, K, generator=g).to(x.dtype).to(gpu)
        v = torch.zeros(T, R, device=gpu)
        qwq4.lora(x, A, B, ids, ys.clone(), v=v)
        want = qwq4.lora_backward(dy, x, A, B, ids, v, dx=dx, dx_out=torch.empty_like(dx))
        back = qwq4.lora_backward(dy, x2, A2, B2, ids, v, dx=dx, dx_out=torch.empty_like(dx))
        clean_t = ids != 2
        assert torch.equal(back[0][clean_t], want[0][clean_t])
        assert torch.equal(back[1][0], want[1][0]) and torch.equal(back[2][:2], want[2][:2]) and (back[1][3] == 0).all()


def test_fp16_over_its_range(gpu):
    """v beyond fp16's range and far below its smallest step: the product still is the sum of 64 bits."""
    T, K, N, R, L = 33, 256, 64, 16, 2
    x, A, B, ids, scaling, g = make(4, T, K, N, R, L, "f16", gpu, "one")
    for by in (3000.0, 2.0**-14):
        xs = (x.float() * by).half()
        ys = torch.zeros(T, N, device=gpu)
        v = torch.empty(T, R, device=gpu)
        out = qwq4.lora(xs, A * 8 if by > 1 else A, B, ids, ys, out=torch.empty_like(ys), v=v)
        assert by < 1 or float(v.abs().max()) > 65504
        _, _, want, bound = ref.lora(xs, A * 8 if by > 1 else A, B, ids, ys)
        assert_close(out, want, bound)
    big = qwq4.lora((x.float() * 3000).half(), A * 8, B, ids, torch.zeros(T, N, dtype=torch.float16, device=gpu))
    assert torch.isfinite(big).all() and float(big.abs().max()) == 65504


GRAD_CASES = [(1, 64, 64, 16, 1, "one"), (2, 8, 8, 8, 2, "mixed"), (17, 520, 264, 40, 2, "mixed"),
              (37, 640, 1032, 16, 32, "mixed"), (64, 72, 64, 128, 3, "runs"), (130, 256, 200, 24, 3, "mixed"),
              (601, 264, 520, 64, 2, "runs"), (2500, 128, 136, 16, 3, "runs"), (40, 64, 64, 16, 3, "none"),
              (4100, 64, 72, 8, 1, "one"), (300, 1536, 640, 16, 4, "runs")]


@pytest.mark.parametrize("T,K,N,R,L,kind", GRAD_CASES)
@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_lora_backward(gpu, T, K, N, R, L, kind, t):
    print(f"lora_backward T={T} K={K} N={N} R={R} L={L} {kind} {t}", flush=True)
    x, A, B, ids, scaling, g = make(T + N + R, T, K, N, R, L, t, gpu, kind)
    dy, dx = (torch.randn(T, n, generator=g).to(x.dtype).to(gpu) for n in (N, K))
    v = torch.full((T, R), float("nan"), device=gpu)  # (rows without an adapter are not read)
    qwq4.lora(x, A, B, ids, torch.zeros(T, N, device=gpu), v=v)
    out, dA, dB = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling, dx=dx, dx_out=torch.empty_like(dx))
    (wx, bx), wA, bA, wB, bB = ref.lora_grad(dy, x, A, B, ids, torch.nan_to_num(v), scaling, dx)
    assert_close(out, wx, bx, "dx")
    assert_close(dA, wA, bA, "dA")
    assert_close(dB, wB, bB, "dB")
    same = dx.clone()
    a, b, c = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling, dx=same, need_weights=False)
    assert a is same and torch.equal(a, out) and b is None and c is None
    a, b, c = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling)
    assert a is None and torch.equal(b, dA) and torch.equal(c, dB)


def test_one_gradient_alone(gpu):
    """dA or dB alone through the C call, the other side's inputs not given."""
    T, K, N, R, L = 70, 128, 648, 16, 2
    x, A, B, ids, scaling, g = make(9, T, K, N, R, L, "bf16", gpu)
    dy = torch.randn(T, N, generator=g).to(x.dtype).to(gpu)
    v = torch.zeros(T, R, device=gpu)
    qwq4.lora(x, A, B, ids, torch.zeros(T, N, device=gpu), v=v)
    _, dA, dB = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling)
    lib, s = qwq4.lib(), torch.cuda.current_stream().cuda_stream
    n = qwq4.lora_backward_workspace_size(T, K, N, R, L)
    ws, a, b = torch.empty(n, dtype=torch.uint8, device=gpu), torch.empty_like(dA), torch.empty_like(dB)
    p = lambda t: t.data_ptr()  # noqa: E731
    for want_a in (True, False):
        rc = lib.qw_lora_backward(p(dy), N, p(x) if want_a else None, K, 0, p(A), p(B), p(ids), None if want_a else p(v),
                                  p(scaling), T, K, N, R, L, None, 0, None, 0, p(a) if want_a else None,
                                  None if want_a else p(b), p(ws), n, s)
        assert rc == 0, lib.qw_q4_last_error()
    assert torch.equal(a, dA) and torch.equal(b, dB)


def test_backward_is_the_derivative(gpu):
    """Along random directions, against central differences of the adapters in 64 bits."""
    T, K, N, R, L, step = 21, 64, 72, 8, 2, 1e-4
    x, A, B, ids, scaling, g = make(10, T, K, N, R, L, "bf16", gpu)
    dy = torch.randn(T, N, generator=g).to(x.dtype).to(gpu)
    v = torch.zeros(T, R, device=gpu)
    y0 = torch.zeros(T, N, device=gpu)
    qwq4.lora(x, A, B, ids, y0.clone(), v=v)
    dx0 = torch.zeros(T, K, dtype=x.dtype, device=gpu)
    dx, dA, dB = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling, dx=dx0)
    (_, bx), _, bA, _, bB = ref.lora_grad(dy, x, A, B, ids, v, scaling, torch.zeros_like(dx0))
    for seed in range(4):
        d = [torch.randn(t.shape, generator=g).double() for t in (x, A, B)]
        f = lambda s: float((ref.lora(*(f64(t) + s * e for t, e in zip((x, A, B), d)), ids, y0, scaling)[2] * f64(dy)).sum())  # noqa: E731
        # (the function is a cubic along a line: the difference's error is its third coefficient times step^2)
        slope = (f(step) - f(-step)) / (2 * step)
        third = abs((f(1.0) - f(-1.0)) / 2 - slope)
        got = sum(float((f64(t) * e).sum()) for t, e in zip((dx, dA, dB), d))
        # (dx is rounded to 16 bits, the other two to fp32)
        limit = sum(float(((b + h * f64(t).abs()) * e.abs()).sum()) for t, e, b, h in zip(
            (dx, dA, dB), d, (bx, bA, bB), (2.0**-8, ref.U, ref.U))) + third * step**2 * 2 + 1e-8 * abs(slope)
        assert abs(got - slope) <= limit, (got, slope, limit)


def test_fp16_gradient_overflows(gpu):
    T, K, N, R, L = 3, 64, 64, 16, 1
    x, A, B, ids, scaling, g = make(11, T, K, N, R, L, "f16", gpu, "one")
    dy = torch.zeros(T, N, dtype=torch.float16, device=gpu)
    dy[1] = 60000
    v = torch.zeros(T, R, device=gpu)
    dx, dA, _ = qwq4.lora_backward(dy, x, A * 100, B * 100, ids, v, dx=torch.zeros_like(x))
    assert torch.isinf(dx[1]).any() and (dx[0] == 0).all() and torch.isfinite(dA).all()


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("R", [16, 40, 64, 128])
def test_rows_do_not_depend_on_a_long_batch(gpu, t, R):
    """Long batches share weights among waves, several tiles to a block; short ones do not: the same bits, forward and
    back, in any order of the tokens."""
    T, K, N, L = 2100, 520, 1032, 2
    x, A, B, ids, scaling, g = make(R, T, K, N, R, L, t, gpu)
    dy, dx = (torch.randn(T, n, generator=g).to(x.dtype).to(gpu) for n in (N, K))
    for y in ("f32", t):
        ys = torch.randn(T, N, generator=g).to(TYPES[y]).to(gpu)
        v = torch.zeros(T, R, device=gpu)
        whole = qwq4.lora(x, A, B, ids, ys, scaling=scaling, out=torch.empty_like(ys), v=v)
        back = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling, dx=dx, dx_out=torch.empty_like(dx), need_weights=False)[0]
        for at in ([5], list(range(60, 97)), list(range(400, 527)), torch.randperm(T, generator=g).tolist()):
            i = torch.tensor(at, device=gpu)
            w = torch.zeros(len(at), R, device=gpu)
            assert torch.equal(qwq4.lora(x[i], A, B, ids[i], ys[i], scaling=scaling, v=w), whole[i])
            assert torch.equal(w, v[i])
            assert torch.equal(qwq4.lora_backward(dy[i], x[i], A, B, ids[i], w, scaling=scaling, dx=dx[i])[0], back[i])


def test_offsets_past_32_bits(gpu):
    """Rows 2^23 elements apart: the last ones lie behind 2^32 elements. The same bits as side by side."""
    T, K, N, R, L, ld = 530, 64, 72, 16, 2, 1 << 23
    x, A, B, ids, scaling, g = make(20, T, K, N, R, L, "bf16", gpu)
    flat = torch.empty(T * ld, dtype=x.dtype, device=gpu)  # (9 GB: every row holds x, y, out, dy, dx and dx_out)
    far = lambda at, n: flat.as_strided((T, n), (ld, 1), at)  # noqa: E731
    ys, dy, dx = (torch.randn(T, n, generator=g).to(x.dtype).to(gpu) for n in (N, N, K))
    views = [far(1024 * i, t.shape[1]) for i, t in enumerate((x, ys, ys, dy, dx, dx))]
    for view, t in zip(views, (x, ys, ys, dy, dx, dx)):
        view.copy_(t)
    fx, fy, fout, fdy, fdx, fdxo = views
    v, w = torch.zeros(T, R, device=gpu), torch.zeros(T, R, device=gpu)
    want = qwq4.lora(x, A, B, ids, ys, scaling=scaling, out=torch.empty_like(ys), v=v)
    qwq4.lora(fx, A, B, ids, fy, scaling=scaling, out=fout, v=w)
    assert torch.equal(fout, want) and torch.equal(v, w)
    want = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling, dx=dx, dx_out=torch.empty_like(dx))
    got = qwq4.lora_backward(fdy, fx, A, B, ids, w, scaling=scaling, dx=fdx, dx_out=fdxo)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def two_kinds(T, K, N, R, L, t, gpu, small, large):
    """Every other token's rows scaled by `small`, the others' by `large` and zero in the first 16 columns of x and dy:
    there the weights' gradients are sums of the small tokens' products alone."""
    x, A, B, ids, scaling, g = make(30, T, K, N, R, L, t, gpu, "one")
    dy = torch.randn(T, N, generator=g).to(x.dtype).to(gpu)
    big = (torch.arange(T, device=gpu) % 2 == 0)[:, None]
    by = torch.where(big, large, small)
    x, dy = (x.float() * by).to(x.dtype), (dy.float() * by).to(x.dtype)
    x[::2, :16] = 0
    dy[::2, :16] = 0
    return x, A, B, ids, scaling, dy


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("T,R", [(60, 16), (700, 16), (300, 64)])
@pytest.mark.parametrize("small,large", [(2.0**-8, 2.0**4), (2.0**-12, 2.0**12)])
def test_small_tokens_beside_large_ones(gpu, t, T, R, small, large):
    """Factors far below the largest of their rank: the sums that only they reach are as exact as any."""
    K, N, L = 136, 264, 2
    x, A, B, ids, scaling, dy = two_kinds(T, K, N, R, L, t, gpu, small, large)
    v = torch.zeros(T, R, device=gpu)
    qwq4.lora(x, A, B, ids, torch.zeros(T, N, device=gpu), v=v)
    _, dA, dB = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling)
    _, wA, bA, wB, bB = ref.lora_grad(dy, x, A, B, ids, v, scaling)
    assert_close(dA, wA, bA, "dA")
    assert_close(dB, wB, bB, "dB")


@pytest.mark.parametrize("t", ["bf16", "f16"])
@pytest.mark.parametrize("T", [300, 2500])
def test_growing_tokens(gpu, t, T):
    """Factors that grow a hundredfold and more every 64 tokens of an adapter, and shrink again."""
    K, N, R, L = 72, 136, 24, 2
    x, A, B, ids, scaling, g = make(31, T, K, N, R, L, t, gpu)
    dy = torch.randn(T, N, generator=g).to(x.dtype).to(gpu)
    by = torch.tensor([2.0**-9, 2.0**-2, 2.0**6, 2.0**9, 1.0], device=gpu)[torch.arange(T, device=gpu) // 128 % 5][:, None]
    x, dy = (x.float() * by).to(x.dtype), (dy.float() * by).to(x.dtype)
    v = torch.zeros(T, R, device=gpu)
    qwq4.lora(x, A, B, ids, torch.zeros(T, N, device=gpu), v=v)
    _, dA, dB = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling)
    _, wA, bA, wB, bB = ref.lora_grad(dy, x, A, B, ids, v, scaling)
    assert_close(dA, wA, bA, "dA")
    assert_close(dB, wB, bB, "dB")


@pytest.mark.parametrize("t", ["bf16", "f16"])
def test_infinite_rows_in_the_weights_gradients(gpu, t):
    """An infinity or a NaN of a token's row reaches its column of its adapter only, and shows there."""
    T, K, N, R, L = 70, 64, 136, 16, 2
    x, A, B, ids, scaling, g = make(32, T, K, N, R, L, t, gpu)
    ids[:] = torch.arange(T) % 2
    dy, v = torch.randn(T, N, generator=g).to(x.dtype).to(gpu), torch.randn(T, R, generator=g).to(gpu)
    _, cA, cB = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling)
    x2, dy2 = x.clone(), dy.clone()
    x2[4, 5], x2[6, 9] = float("inf"), float("nan")
    _, dA, _ = qwq4.lora_backward(dy, x2, A, B, ids, v, scaling=scaling)
    assert not torch.isfinite(dA[0, :, 5]).any() and torch.isnan(dA[0, :, 9]).all()
    dA[0, :, 5], dA[0, :, 9] = cA[0, :, 5], cA[0, :, 9]
    assert torch.equal(dA, cA)
    dy2[4, 5], dy2[6, 9] = float("-inf"), float("nan")
    _, _, dB = qwq4.lora_backward(dy2, x, A, B, ids, v, scaling=scaling)
    assert not torch.isfinite(dB[0, 5]).any() and torch.isnan(dB[0, 9]).all()
    dB[0, 5], dB[0, 9] = cB[0, 5], cB[0, 9]
    assert torch.equal(dB, cB)


@pytest.mark.parametrize("T", [40, 1000])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_scaling_of_an_adapter_without_tokens(gpu, T, bad):
    """A free slot's scaling may hold anything: its gradients are zeros, in one part of the batch or several."""
    K, N, R, L = 64, 72, 16, 3
    x, A, B, ids, scaling, g = make(33, T, K, N, R, L, "bf16", gpu)
    ids[ids == 1] = 2
    dy, v = torch.randn(T, N, generator=g).to(x.dtype).to(gpu), torch.randn(T, R, generator=g).to(gpu)
    dx = torch.zeros(T, K, dtype=x.dtype, device=gpu)
    want = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling, dx=dx.clone())
    scaling[1] = bad
    got = qwq4.lora_backward(dy, x, A, B, ids, v, scaling=scaling, dx=dx.clone())
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and (got[1][1] == 0).all() and (got[2][1] == 0).all()
