"""qw_rms_norm, qw_rms_norm_i8 and their gradients against 64 bits."""
import numpy as np
import pytest
import torch

import qwq4
import _projection_ref as ref
from _projection_ref import TYPES, assert_close, f64

pytestmark = pytest.mark.gpu
EPS = 1e-6
GUARD = 77.0


def rows(seed, T, H, t, gpu, pad=0, off=0):
    """[T][H] with `pad` elements between rows, `off` elements from an aligned start."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T * (H + pad) + off, generator=g)
    x[::37] *= 8
    buf = x.to(TYPES[t]).to(gpu)
    return buf[off:].view(T, H + pad)[:, :H]


def like(T, H, t, gpu, pad=0):
    """Rows to write to inside a guarded buffer."""
    buf = torch.full((T, H + pad), GUARD, dtype=t, device=gpu)
    return buf[:, :H], buf


SIZES = [(1, 1), (1, 7), (3, 8), (1, 4096), (5, 256), (4, 512), (6, 520), (37, 2560), (3, 2049), (2, 4097), (9, 4104),
         (5, 8192), (2, 8200), (2, 20000), (700, 640), (130, 33), (67, 1023)]


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("x,res,y", [("bf16", None, "bf16"), ("bf16", "bf16", "bf16"), ("f16", "f32", "f16"),
                                     ("f32", "f32", "bf16"), ("f16", "f16", "f32"), ("f32", None, "f32")])
def test_norm(gpu, T, H, x, res, y):
    print(f"rms_norm T={T} H={H} {x} {res} {y}", flush=True)
    xs, w = rows(T + H, T, H, x, gpu), rows(5, 1, H, "f32" if T % 2 else x, gpu)[0]
    rs = rows(T * H, T, H, res, gpu) if res else None
    out, buf = like(T, H, TYPES[y], gpu, pad=3)
    got = qwq4.rms_norm(xs, w, EPS, residual=rs, y=out)
    h, _, want, bound = ref.norm(xs, w, EPS, rs)
    if res:
        assert got[0] is out
        assert_close(got[1], h, U_of(h), "residual")
    assert_close(out, want, bound, "y")
    assert (buf[:, H:] == GUARD).all()
    again = qwq4.rms_norm(xs, w, EPS, residual=rs, y_dtype=TYPES[y])
    assert torch.equal(again[0] if res else again, out)


@pytest.mark.parametrize("y", sorted(TYPES))
@pytest.mark.parametrize("w", sorted(TYPES))
@pytest.mark.parametrize("res", [None, *sorted(TYPES)])
@pytest.mark.parametrize("x", sorted(TYPES))
def test_types(gpu, x, res, w, y):
    """Every combination of types, vectors and single elements; those that are no types of the call are refused."""
    for H in (8, 1000, 1001):
        xs, ws = rows(H, 3, H, x, gpu), rows(5, 1, H, w, gpu)[0]
        rs = rows(H + 1, 3, H, res, gpu) if res else None
        if w not in (x, "f32") or res not in (None, x, "f32"):
            with pytest.raises(RuntimeError, match="x's type"):
                qwq4.rms_norm(xs, ws, EPS, residual=rs, y_dtype=TYPES[y])
            continue
        got = qwq4.rms_norm(xs, ws, EPS, residual=rs, y_dtype=TYPES[y])
        h, _, want, bound = ref.norm(xs, ws, EPS, rs)
        assert_close(got[0] if res else got, want, bound)
        if res:
            assert_close(got[1], h, U_of(h))
        q, s, *_ = qwq4.rms_norm_i8(xs, ws, EPS, residual=rs)
        u = (xs.float() + (rs.float() if res else 0)) * ws.float()
        assert torch.equal(q, qwq4.quant_tokens_i8(u)[0]) if H % 16 == 0 else int(q.abs().max()) == 127
        if res is None and w in (y, "f32") and x in (y, "f32"):  # (y the type of dy)
            dy = rows(H + 2, 3, H, y, gpu)
            dx, dw = qwq4.rms_norm_backward(dy, xs, ws, EPS)
            want = ref.norm_grad(dy, xs, ws, EPS)
            assert_close(dx, want[0], want[1])
            assert_close(dw, want[2], want[3])


def U_of(h):
    return h.abs() * 2 * ref.U


@pytest.mark.parametrize("T,H", SIZES)
@pytest.mark.parametrize("x,res", [("bf16", "bf16"), ("f16", "f32"), ("f32", None)])
def test_norm_i8(gpu, T, H, x, res):
    """The 8-bit values are those of h w in fp32, bit for bit; the scale is within its roundings."""
    print(f"rms_norm_i8 T={T} H={H} {x} {res}", flush=True)
    xs, w = rows(T + 3 * H, T, H, x, gpu), rows(6, 1, H, x, gpu)[0]
    rs = rows(T * H + 1, T, H, res, gpu) if res else None
    q, scale, *more = qwq4.rms_norm_i8(xs, w, EPS, residual=rs)
    h, r, _, _ = ref.norm(xs, w, EPS, rs)
    u = (xs.float() + (rs.float() if res else 0)).cpu().numpy() * w.float().cpu().numpy()
    top = np.abs(u).max(1)
    step = np.where(top > 0, np.maximum(top / np.float32(127), np.float32(2.0**-126)), np.float32(1))
    assert np.array_equal(q.cpu().numpy(), np.rint(u * (np.float32(1) / step)[:, None]).astype(np.int8))
    want = torch.from_numpy(step.astype(np.float64)) * r[:, 0]
    assert_close(scale, want, want.abs() * ref.U * (ref.norm_chain(H) / 2 + 8), "scale")
    if res:
        assert_close(more[0], h, U_of(h), "residual")


def test_norm_i8_feeds_the_product(gpu):
    """q is the quantiser's for the rows h w, so the product of either is the same up to the scale's roundings."""
    xs, w = rows(3, 33, 4096, "f32", gpu), rows(4, 1, 4096, "f32", gpu)[0]
    q, scale = qwq4.rms_norm_i8(xs, w, EPS)
    q2, step = qwq4.quant_tokens_i8(xs * w)
    assert torch.equal(q, q2)
    r = ref.norm(xs, w, EPS)[1][:, 0]
    assert_close(scale, f64(step) * r, f64(step) * r * ref.U * (ref.norm_chain(4096) / 2 + 8))


@pytest.mark.parametrize("T,H", [(1, 8), (3, 640), (2, 4096), (2, 9000), (5, 2051)])
def test_in_place(gpu, T, H):
    for x, res in (("bf16", "bf16"), ("f32", "f32")):
        xs, rs, w = rows(1, T, H, x, gpu), rows(2, T, H, res, gpu), rows(3, 1, H, x, gpu)[0]
        y, r = qwq4.rms_norm(xs, w, EPS, residual=rs)
        r2 = rs.clone()
        y2, same = qwq4.rms_norm(xs, w, EPS, residual=r2, residual_out=r2)
        assert same is r2 and torch.equal(r, r2) and torch.equal(y, y2)
        x3 = xs.clone()
        assert torch.equal(qwq4.rms_norm(x3, w, EPS, y=x3), qwq4.rms_norm(xs, w, EPS))
        r4 = rs.clone()
        q, s, _ = qwq4.rms_norm_i8(xs, w, EPS, residual=rs)
        q4, s4, _ = qwq4.rms_norm_i8(xs, w, EPS, residual=r4, residual_out=r4)
        assert torch.equal(q, q4) and torch.equal(s, s4) and torch.equal(r4, r)
        dy, dres = rows(7, T, H, x, gpu), rows(8, T, H, x, gpu)
        dx, dw = qwq4.rms_norm_backward(dy, xs, w, EPS, dres=dres)
        for i in range(3):
            ins = [dy.clone(), xs.clone(), dres.clone()]
            dx2, dw2 = qwq4.rms_norm_backward(ins[0], ins[1], w, EPS, dres=ins[2], dx=ins[i])
            assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@pytest.mark.parametrize("off,pad", [(1, 0), (0, 1), (4, 4), (8, 8), (0, 5)])
def test_strides_and_alignment(gpu, off, pad):
    """Rows at any element, of any stride: the same bits as rows on their own."""
    T, H = 9, 1160
    xs, rs, w = rows(1, T, H, "bf16", gpu, pad, off), rows(2, T, H, "f32", gpu, pad, off), rows(3, 1, H, "bf16", gpu)[0]
    dy = rows(4, T, H, "bf16", gpu, pad, off)
    y, r = qwq4.rms_norm(xs.contiguous(), w, EPS, residual=rs.contiguous())
    y2, r2 = qwq4.rms_norm(xs, w, EPS, residual=rs, y=like(T, H, y.dtype, gpu, pad)[0])
    h, _, want, bound = ref.norm(xs, w, EPS, rs)
    assert torch.equal(r, r2)
    assert_close(y2, want, bound)
    q = torch.full((T, H + pad), 99, dtype=torch.int8, device=gpu)
    q1, _, _ = qwq4.rms_norm_i8(xs.contiguous(), w, EPS, residual=rs.contiguous())
    qwq4.rms_norm_i8(xs, w, EPS, residual=rs, q=q[:, :H])
    assert torch.equal(q[:, :H], q1) and (q[:, H:] == 99).all()
    dx, dw = qwq4.rms_norm_backward(dy, rs, w, EPS, dres=rs, dx=like(T, H, rs.dtype, gpu, pad)[0])
    want = ref.norm_grad(dy, rs, w, EPS, rs)
    assert_close(dx, want[0], want[1])
    assert_close(dw, want[2], want[3])


def test_special_rows(gpu):
    """Zeros, infinities and NaN stay in their rows; fp16 saturates, a row of zeros has step 1 in 8 bits."""
    for H in (64, 1001, 4096, 9000):
        xs = rows(1, 6, H, "f32", gpu).contiguous()
        xs[1] = 0
        xs[2, H // 2] = float("inf")
        xs[3, H - 1] = float("nan")
        w = torch.full((H,), 1.0, device=gpu)
        y = qwq4.rms_norm(xs, w, EPS)
        clean = qwq4.rms_norm(xs[[0, 4, 5]].contiguous(), w, EPS)
        assert torch.equal(y[[0, 4, 5]], clean)
        assert (y[1] == 0).all() and torch.isnan(y[2, H // 2]) and torch.isnan(y[3]).all()
        q, s = qwq4.rms_norm_i8(xs, w, EPS)
        assert (q[1:4] == 0).all() and torch.isnan(s[2]) and torch.isnan(s[3])
        assert float(s[1]) == pytest.approx(1 / EPS**0.5, rel=1e-5)
        big = torch.full((H,), 60000.0, device=gpu)
        assert (qwq4.rms_norm(xs[:1], big, EPS, y_dtype=torch.float16).abs() <= 65504).all()


GRAD_SIZES = [(1, 1), (1, 4096), (3, 8), (5, 7), (33, 512), (2, 520), (601, 2560), (1100, 640), (4, 2049), (3, 4104),
              (2, 8192), (5, 8193), (3, 16384), (2, 16383), (1030, 256)]


@pytest.mark.parametrize("T,H", GRAD_SIZES)
@pytest.mark.parametrize("dy,h,dres", [("bf16", "bf16", True), ("f16", "f16", False), ("f32", "f32", True),
                                       ("bf16", "f32", False)])
def test_norm_backward(gpu, T, H, dy, h, dres):
    print(f"rms_norm_backward T={T} H={H} {dy} {h} {dres}", flush=True)
    d, hs, w = rows(1, T, H, dy, gpu), rows(2, T, H, h, gpu), rows(3, 1, H, "f32" if T % 2 else dy, gpu)[0]
    rs = rows(4, T, H, h, gpu) if dres else None
    dx, dw = qwq4.rms_norm_backward(d, hs, w, EPS, dres=rs)
    want, bound, wdw, bdw = ref.norm_grad(d, hs, w, EPS, rs)
    assert_close(dx, want, bound, "dx")
    assert_close(dw, wdw, bdw, "dw")
    only, none = qwq4.rms_norm_backward(d, hs, w, EPS, dres=rs, need_dw=False)
    assert none is None and torch.equal(only, dx)


def test_backward_is_the_derivative(gpu):
    """Along random directions, against central differences of the norm in 64 bits."""
    T, H, step = 7, 320, 1e-5
    dy, hs, w = rows(1, T, H, "f32", gpu), rows(2, T, H, "f32", gpu), rows(3, 1, H, "f32", gpu)[0]
    dx, dw = qwq4.rms_norm_backward(dy, hs, w, EPS)
    want = ref.norm_grad(dy, hs, w, EPS)
    for seed in range(5):
        vh, vw = f64(rows(50 + seed, T, H, "f32", gpu)), f64(rows(60 + seed, 1, H, "f32", gpu)[0])
        f = lambda s: float((ref.norm(f64(hs) + s * vh, f64(w) + s * vw, EPS)[2] * f64(dy)).sum())  # noqa: E731
        slope = (f(step) - f(-step)) / (2 * step)
        got = float((f64(dx) * vh).sum() + (f64(dw) * vw).sum())
        # the kernel's bounds along the direction; the differences' own error is of the third derivative, times step^2
        limit = float((want[1] * vh.abs()).sum() + (want[3] * vw.abs()).sum()) + 2 * ref.U * float(
            (f64(dx) * vh).abs().sum() + (f64(dw) * vw).abs().sum()) + 1e-6 * float((f64(dy).abs()).sum())
        assert abs(got - slope) <= limit, (got, slope, limit)


def test_fp16_gradient_overflows(gpu):
    hs, w = torch.ones(2, 64, dtype=torch.float16, device=gpu), torch.full((64,), 60000.0, device=gpu)
    dy = torch.zeros(2, 64, dtype=torch.float16, device=gpu)
    dy[0, 0] = 10.0
    dx, _ = qwq4.rms_norm_backward(dy, hs, w, EPS)
    assert torch.isinf(dx[0, 0]) and torch.isfinite(dx[1]).all()


def test_offsets_past_32_bits(gpu):
    """The last rows of more than 2^32 bytes."""
    T, H = 300000, 4096
    xs = torch.zeros(T, H, dtype=torch.bfloat16, device=gpu)
    xs[-3:] = rows(1, 3, H, "bf16", gpu)
    w = rows(2, 1, H, "bf16", gpu)[0]
    y = qwq4.rms_norm(xs, w, EPS)
    assert torch.equal(y[-3:], qwq4.rms_norm(xs[-3:], w, EPS)) and (y[:5] == 0).all()
    del y
    dx, _ = qwq4.rms_norm_backward(xs, xs, w, EPS)
    assert torch.equal(dx[-3:], qwq4.rms_norm_backward(xs[-3:], xs[-3:], w, EPS)[0])


@pytest.mark.parametrize("T,H", [(40001, 64), (20000, 100), (9001, 129), (9000, 256), (4100, 384), (3001, 1000), (1500, 1032),
                                 (2100, 2048), (700, 2047), (600, 5120), (300, 12288)])
@pytest.mark.parametrize("dy,h,dres", [("bf16", "bf16", True), ("f16", "f32", False), ("f32", "f32", False)])
def test_many_rows(gpu, T, H, dy, h, dres):
    """Every way of sharing rows among lanes, waves and blocks with more rows than are taken at once."""
    test_norm_backward(gpu, T, H, dy, h, dres)
    test_norm(gpu, T, H, dy, "f32" if h == "f32" else None, dy)


@pytest.mark.parametrize("x", sorted(TYPES))
@pytest.mark.parametrize("H", [8, 16, 1000, 1008, 1001, 2560, 9000])
def test_i8_of_every_type(gpu, x, H):
    """Every combination of types that the 8-bit call takes: the bits of q, the scale and the residual, against the
    host's arithmetic in fp32."""
    xs = rows(H, 5, H, x, gpu)
    for w in {x, "f32"}:
        ws = rows(5, 1, H, w, gpu)[0]
        for res in {None, x, "f32"}:
            rs = rows(H + 1, 5, H, res, gpu) if res else None
            q, scale, *more = qwq4.rms_norm_i8(xs, ws, EPS, residual=rs)
            h = xs.float().cpu().numpy() + (rs.float().cpu().numpy() if res else np.float32(0))
            u = h * ws.float().cpu().numpy()
            step = np.maximum(np.abs(u).max(1) / np.float32(127), np.float32(2.0**-126))
            assert u.dtype == step.dtype == np.float32
            assert np.array_equal(q.cpu().numpy(), np.rint(u * (np.float32(1) / step)[:, None]).astype(np.int8)), (w, res)
            r = ref.norm(xs, ws, EPS, rs)[1][:, 0]
            want = torch.from_numpy(step.astype(np.float64)) * r
            assert_close(scale, want, want.abs() * ref.U * (ref.norm_chain(H) / 2 + 8), f"scale {w} {res}")
            if res:
                assert torch.equal(more[0].cpu(), torch.from_numpy(h).to(TYPES[res])), (w, res)


@pytest.mark.parametrize("H", [64, 520, 1160, 2048, 2047, 2560, 4100, 9000, 16384])
@pytest.mark.parametrize("dy,h", [("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f32", "f32")])
def test_bits_do_not_depend_on_the_place(gpu, H, dy, h):
    """Rows side by side on 16 bytes, rows at odd elements and strides, and a single row out of them: the same bits,
    forward and back."""
    T = 7
    for off, pad in ((0, 8), (1, 0), (3, 5)):
        d, hs, rs = rows(1, T, H, dy, gpu, pad, off), rows(2, T, H, h, gpu, pad, off), rows(3, T, H, h, gpu, pad, off)
        w = rows(4, 1, H, dy, gpu)[0]
        out = like(T, H, hs.dtype, gpu, pad + 1)[0]
        dx, dw = qwq4.rms_norm_backward(d.contiguous(), hs.contiguous(), w, EPS, dres=rs.contiguous())
        dx2, dw2 = qwq4.rms_norm_backward(d, hs, w, EPS, dres=rs, dx=out)
        assert torch.equal(dx, dx2) and torch.equal(dw, dw2), (off, pad)
        for t in (0, T - 1):
            one, _ = qwq4.rms_norm_backward(d[t:t + 1], hs[t:t + 1], w, EPS, dres=rs[t:t + 1])
            assert torch.equal(one, dx[t:t + 1]), (off, pad, t)
        ws = w if dy == h else w.float()
        y, r = qwq4.rms_norm(hs.contiguous(), ws, EPS, residual=rs.contiguous())
        y2, r2 = qwq4.rms_norm(hs, ws, EPS, residual=rs, y=like(T, H, hs.dtype, gpu, pad + 1)[0])
        assert torch.equal(y, y2) and torch.equal(r, r2), (off, pad)
        q, s, _ = qwq4.rms_norm_i8(hs.contiguous(), ws, EPS, residual=rs.contiguous())
        q2, s2, _ = qwq4.rms_norm_i8(hs, ws, EPS, residual=rs, q=torch.empty(T, H + 3, dtype=torch.int8, device=gpu)[:, :H])
        assert torch.equal(q, q2) and torch.equal(s, s2), (off, pad)
