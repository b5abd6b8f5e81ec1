"""What the operators around a projection refuse, each with a message and nothing
launched (host-side checks: no GPU needed)."""
import ctypes

import pytest

import qwq4

P, Q = ctypes.c_void_p(4096), ctypes.c_void_p(8192)  # aligned, never read: every call below is refused first
ODD, TWO, EIGHT = (ctypes.c_void_p(4096 + n) for n in (1, 2, 8))
BIG = 1 << 40
MANY = (1 << 23) + 1
NAN = float("nan")


def norm(x=P, xt=1, ldx=64, r=Q, rt=1, ldr=64, ro=Q, ldro=64, w=P, wt=0, eps=1e-6, T=4, H=64, y=P, yt=1, ldy=64):
    return "qw_rms_norm", (x, xt, ldx, r, rt, ldr, ro, ldro, w, wt, eps, T, H, y, yt, ldy, None)


def norm_i8(x=P, xt=1, ldx=64, r=None, rt=0, ldr=0, ro=None, ldro=0, w=P, wt=0, eps=1e-6, T=4, H=64, q=Q, ldq=64, s=P):
    return "qw_rms_norm_i8", (x, xt, ldx, r, rt, ldr, ro, ldro, w, wt, eps, T, H, q, ldq, s, None)


def norm_grad(dy=P, dt=1, lddy=64, h=Q, ht=1, ldh=64, w=P, wt=0, eps=1e-6, dres=None, lddr=0, T=4, H=64, dx=Q, lddx=64,
              dw=P, ws=P, wb=BIG):
    return "qw_rms_norm_backward", (dy, dt, lddy, h, ht, ldh, w, wt, eps, dres, lddr, T, H, dx, lddx, dw, ws, wb, None)


def lora(x=P, ldx=64, f16=0, A=P, B=P, ids=P, s=None, T=4, K=64, N=32, R=16, L=2, v=P, y=P, ldy=32, out=P, ldo=32, yt=1):
    return "qw_lora", (x, ldx, f16, A, B, ids, s, T, K, N, R, L, v, y, ldy, out, ldo, yt, None)


def lora_grad(dy=P, lddy=32, x=P, ldx=64, A=P, B=P, ids=P, v=P, s=None, T=4, K=64, N=32, R=16, L=2, dx=P, lddx=64,
              dxo=P, lddxo=64, dA=P, dB=P, ws=P, wb=BIG):
    return "qw_lora_backward", (dy, lddy, x, ldx, 0, A, B, ids, v, s, T, K, N, R, L, dx, lddx, dxo, lddxo, dA, dB, ws,
                                wb, None)


def logprobs(l=P, t=1, ld=100, tok=P, T=1, V=100, top=3, lp=P, h=P, lse=P, ti=P, tv=P, ws=P, wb=BIG):
    return "qw_logprobs", (l, t, ld, tok, T, V, top, lp, h, lse, ti, tv, ws, wb, None)


def logprobs_grad(l=P, t=1, ld=100, tok=P, lse=P, h=P, g=P, gh=P, T=2, V=100, d=Q, ldd=100):
    return "qw_logprobs_backward", (l, t, ld, tok, lse, h, g, gh, T, V, d, ldd, None)


CALLS = {
    "norm null x": norm(x=None), "norm null w": norm(w=None), "norm null y": norm(y=None), "norm no rows": norm(T=0),
    "norm negative rows": norm(T=-1), "norm no columns": norm(H=0), "norm too many rows": norm(T=MANY),
    "norm rows too long": norm(H=(1 << 28) + 1, T=1), "norm x type": norm(xt=3), "norm w type": norm(wt=2),
    "norm w type unknown": norm(wt=-1), "norm residual type": norm(rt=2), "norm y type": norm(yt=4),
    "norm ldx": norm(ldx=63), "norm ldr": norm(ldr=63), "norm ldro": norm(ldro=63, ro=P), "norm ldy": norm(ldy=60),
    "norm x odd": norm(x=ODD), "norm fp32 w at 2": norm(w=TWO), "norm no res_out": norm(ro=None),
    "norm res_out alone": norm(r=None), "norm residual in place, other stride": norm(ldro=72),
    "norm y on x, other type": norm(yt=2), "norm y on x, other stride": norm(ldy=72), "norm y on the residual": norm(y=Q),
    "norm eps negative": norm(eps=-1.0), "norm eps nan": norm(eps=NAN), "norm eps infinite": norm(eps=float("inf")),
    "i8 null q": norm_i8(q=None), "i8 null scale": norm_i8(s=None), "i8 ldq": norm_i8(ldq=63), "i8 no rows": norm_i8(T=0),
    "i8 x type": norm_i8(xt=5), "i8 scale odd": norm_i8(s=TWO), "i8 residual without res_out": norm_i8(r=P, rt=1, ldr=64),
    "i8 q on x": norm_i8(q=P), "i8 q on the residual": norm_i8(r=Q, rt=1, ldr=64, ro=Q, ldro=64),
    "norm res_out on x, other type": norm(ro=P, rt=0, y=EIGHT), "norm res_out on x, other stride": norm(ro=P, ldro=72, ldr=72, y=EIGHT),
    "grad null dy": norm_grad(dy=None), "grad null h": norm_grad(h=None), "grad null w": norm_grad(w=None),
    "grad null dx": norm_grad(dx=None), "grad no rows": norm_grad(T=0), "grad rows too long": norm_grad(H=16385),
    "grad h type": norm_grad(ht=2), "grad w type": norm_grad(wt=2), "grad dy type": norm_grad(dt=7),
    "grad lddy": norm_grad(lddy=63), "grad ldh": norm_grad(ldh=63), "grad lddx": norm_grad(lddx=63),
    "grad lddr": norm_grad(dres=P, lddr=63), "grad dx on dy, other type": norm_grad(ht=0, dx=P),
    "grad dx on h, other stride": norm_grad(lddx=72), "grad no workspace": norm_grad(ws=None),
    "grad workspace short": norm_grad(wb=1023), "grad workspace at 8": norm_grad(ws=EIGHT), "grad dw odd": norm_grad(dw=TWO),
    "grad eps": norm_grad(eps=NAN),
    "lora null x": lora(x=None), "lora null A": lora(A=None), "lora null B": lora(B=None), "lora null ids": lora(ids=None),
    "lora null v": lora(v=None), "lora null y": lora(y=None), "lora null out": lora(out=None), "lora no rows": lora(T=0),
    "lora too many rows": lora(T=(1 << 20) + 1), "lora K 60": lora(K=60), "lora N 30": lora(N=30), "lora K 0": lora(K=0),
    "lora N 0": lora(N=0), "lora R 0": lora(R=0), "lora R 12": lora(R=12), "lora R 136": lora(R=136), "lora L 0": lora(L=0),
    "lora L 4097": lora(L=4097), "lora ldx": lora(ldx=60), "lora ldx 68": lora(ldx=68), "lora ldx too wide": lora(ldx=(1 << 23) + 8), "lora ldy": lora(ldy=24),
    "lora ldy 36": lora(ldy=36, ldo=36), "lora fp32 ldy 34": lora(yt=0, ldy=34, ldo=34), "lora ldo 36": lora(out=Q, ldo=36),
    "lora in place, other stride": lora(ldo=40), "lora y type": lora(yt=3), "lora x at 8": lora(x=EIGHT),
    "lora A at 8": lora(A=EIGHT), "lora B at 8": lora(B=EIGHT), "lora v at 8": lora(v=EIGHT), "lora y at 8": lora(y=EIGHT),
    "lora ids odd": lora(ids=TWO), "lora scaling odd": lora(s=TWO), "lora K too large": lora(K=(1 << 20) + 8),
    "lora too much": lora(T=1 << 20, N=1 << 17, ldy=1 << 17, ldo=1 << 17),
    "lora grad null dy": lora_grad(dy=None), "lora grad null x": lora_grad(x=None), "lora grad null v": lora_grad(v=None),
    "lora grad nothing asked": lora_grad(dx=None, dxo=None, dA=None, dB=None), "lora grad dx alone": lora_grad(dxo=None),
    "lora grad dx_out alone": lora_grad(dx=None), "lora grad in place, other stride": lora_grad(lddxo=72),
    "lora grad lddy": lora_grad(lddy=24), "lora grad lddx 68": lora_grad(lddx=68, lddxo=68), "lora grad dA at 8": lora_grad(dA=EIGHT),
    "lora grad dB at 8": lora_grad(dB=EIGHT), "lora grad no workspace": lora_grad(ws=None),
    "lora grad workspace short": lora_grad(wb=100), "lora grad workspace at 8": lora_grad(ws=EIGHT), "lora grad R": lora_grad(R=4),
    "logprobs null logits": logprobs(l=None), "logprobs null tokens": logprobs(tok=None), "logprobs no rows": logprobs(T=0),
    "logprobs no vocabulary": logprobs(V=0), "logprobs too many rows": logprobs(T=MANY), "logprobs V too large": logprobs(V=(1 << 28) + 1),
    "logprobs type": logprobs(t=3), "logprobs ld": logprobs(T=2, ld=99), "logprobs logits odd": logprobs(l=ODD),
    "logprobs tokens odd": logprobs(tok=TWO), "logprobs top -1": logprobs(top=-1), "logprobs top 65": logprobs(top=65),
    "logprobs top over V": logprobs(V=2, ld=2), "logprobs null logp": logprobs(lp=None), "logprobs null entropy": logprobs(h=None),
    "logprobs null lse": logprobs(lse=None), "logprobs null top_ids": logprobs(ti=None), "logprobs null top_logp": logprobs(tv=None),
    "logprobs no workspace": logprobs(V=1 << 17, ld=1 << 17, ws=None), "logprobs workspace short": logprobs(V=1 << 17, ld=1 << 17, wb=8),
    "logprobs workspace at 8": logprobs(V=1 << 17, ld=1 << 17, ws=EIGHT), "logprobs output odd": logprobs(lp=TWO),
    "logprobs grad null lse": logprobs_grad(lse=None), "logprobs grad null tokens": logprobs_grad(tok=None),
    "logprobs grad null dlogits": logprobs_grad(d=None), "logprobs grad nothing given": logprobs_grad(g=None, gh=None),
    "logprobs grad no entropy": logprobs_grad(h=None), "logprobs grad ldd": logprobs_grad(ldd=99),
    "logprobs grad in place, other stride": logprobs_grad(d=P, ldd=101), "logprobs grad type": logprobs_grad(t=-1),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refused(lib, name):
    fn, args = CALLS[name]
    assert getattr(lib, fn)(*args) == -1
    assert lib.qw_q4_last_error().decode().startswith(fn + ": ")


def test_workspace_sizes(lib):
    assert lib.qw_rms_norm_backward_workspace_size(0, 64) == 0 == lib.qw_rms_norm_backward_workspace_size(4, -1)
    assert lib.qw_rms_norm_backward_workspace_size(4, 64) == 4 * 64 * 4
    assert lib.qw_logprobs_workspace_size(0, 100, 1) == 0 == lib.qw_logprobs_workspace_size(4096, 151936, 20)
    assert lib.qw_logprobs_workspace_size(1, 151936, 20) > lib.qw_logprobs_workspace_size(1, 151936, 0) > 0
    assert lib.qw_lora_backward_workspace_size(0, 64, 64, 16, 1) == 0
    assert lib.qw_lora_backward_workspace_size(1, 64, 32, 16, 2) >= 16 * 4  # (dv)


@pytest.mark.parametrize("K,N,R,L", [(64, 72, 8, 1), (4096, 12288, 16, 4), (4096, 4096, 64, 63), (2560, 4096, 128, 3),
                                     (512, 512, 32, 1023), (1 << 20, 8, 16, 1), (4096, 4096, 128, 4096)])
def test_lora_workspace_is_bounded(lib, K, N, R, L):
    """dv, and sums of parts of the batch below 256 MB with their counts, however long the batch."""
    for T in (1, 129, 5000, 1 << 20):
        size = lib.qw_lora_backward_workspace_size(T, K, N, R, L)
        assert T * R * 4 <= size < T * R * 4 + (256 << 20) + 64 * 4 * min(L, 2048) + 1024


def test_logprobs_workspace_of_many_rows(lib):
    assert lib.qw_logprobs_workspace_size(511, 151936, 20) > 0
    for T in (512, 513, 2047, 1 << 23):
        for V in (1, 151936, 1 << 28):
            assert lib.qw_logprobs_workspace_size(T, V, min(V, 64)) == 0


def test_python_checks():
    """What the binding itself refuses, on CPU tensors of shapes that the C call never sees."""
    import torch
    x, w = torch.zeros(4, 64), torch.zeros(64)
    for call, error in [
        (lambda: qwq4.rms_norm(x, w[:60]), "w is"), (lambda: qwq4.rms_norm(x, w, residual=x[:3]), "residual is"),
        (lambda: qwq4.rms_norm(x, w, residual_out=x), "without a residual"), (lambda: qwq4.rms_norm(x[0], w), "x is"),
        (lambda: qwq4.rms_norm(x.t(), torch.zeros(4)), "contiguous"), (lambda: qwq4.rms_norm(x, w), "on the GPU"),
        (lambda: qwq4.rms_norm_i8(x, w, q=torch.zeros(4, 64)), "q is"),
        (lambda: qwq4.rms_norm_backward(x, x, w, dres=x.half()), "dres is"),
        (lambda: qwq4.rms_norm(x.requires_grad_(), w), "requires grad"),
    ]:
        with pytest.raises((ValueError, TypeError, RuntimeError), match=error):
            call()
    h = torch.bfloat16
    rows, A, B = torch.zeros(4, 64, dtype=h), torch.zeros(2, 16, 64, dtype=h), torch.zeros(2, 32, 16, dtype=h)
    ids, y, v = torch.zeros(4, dtype=torch.int32), torch.zeros(4, 32), torch.zeros(4, 16)
    for call, error in [
        (lambda: qwq4.lora(rows.float(), A, B, ids, y), "bfloat16 or float16"), (lambda: qwq4.lora(rows, A.half(), B, ids, y), "A is"),
        (lambda: qwq4.lora(rows, A[0], B, ids, y), "A is"), (lambda: qwq4.lora(rows, A, B[:1], ids, y), "B is"),
        (lambda: qwq4.lora(rows[:, :32], A, B, ids, y), "x is"), (lambda: qwq4.lora(rows, A, B, ids.long(), y), "ids is"),
        (lambda: qwq4.lora(rows, A, B, ids[:3], y), "ids is"), (lambda: qwq4.lora(rows, A, B, ids, y[:, :16]), "y is"),
        (lambda: qwq4.lora(rows, A, B, ids, y, out=y.half()), "out is"), (lambda: qwq4.lora(rows, A, B, ids, y, v=v[:, :8]), "v is"),
        (lambda: qwq4.lora(rows, A, B, ids, y, scaling=torch.zeros(3)), "scaling is"), (lambda: qwq4.lora(rows, A, B, ids, y), "on the GPU"),
        (lambda: qwq4.lora_backward(y.to(h), rows, A, B, ids, v, dx_out=rows), "without dx"),
        (lambda: qwq4.lora_backward(y, rows, A, B, ids, v), "dy is"), (lambda: qwq4.lora_backward(y.to(h)[:3], rows, A, B, ids, v), "dy"),
        (lambda: qwq4.lora_backward(y.to(h), rows, A, B, ids, v, dA=v), "dA is"),
        (lambda: qwq4.lora(rows, A, B.clone().requires_grad_(), ids, y), "requires grad"),
    ]:
        with pytest.raises((ValueError, TypeError, RuntimeError), match=error):
            call()
    l, tok, f = torch.zeros(4, 100), torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    for call, error in [
        (lambda: qwq4.logprobs(l, tok.long()), "tokens is"), (lambda: qwq4.logprobs(l, tok, top=65), "top = 65"),
        (lambda: qwq4.logprobs(l[:, :2], tok, top=3), "top = 3"), (lambda: qwq4.logprobs(l.double(), tok), "element type"),
        (lambda: qwq4.logprobs(l, tok), "on the GPU"), (lambda: qwq4.logprobs_backward(l, tok, f[:3], f, f), "lse is"),
        (lambda: qwq4.logprobs_backward(l, tok, f, f, f, dlogits=l.half()), "dlogits is"),
    ]:
        with pytest.raises((ValueError, TypeError, RuntimeError), match=error):
            call()
