"""What the W8A8 products and the expert-row calls refuse, each with a message
and nothing launched (host-side checks: no GPU needed)."""
import ctypes

import pytest

import qwq4

P = ctypes.c_void_p(4096)      # aligned, never read: every call below is refused first
ODD = ctypes.c_void_p(4096 + 1)
EIGHT = ctypes.c_void_p(4096 + 8)
BIG = 1 << 40


def quant(x=P, t=1, ldx=64, T=4, K=64, q=P, ldq=64, s=P):
    return "qw_quant_tokens_i8", (x, t, ldx, T, K, q, ldq, s, None)


def gemm(W=P, ldw=64, sw=P, q=P, ldq=64, sx=P, T=4, Y=P, ldy=32, yt=1, N=32, K=64):
    return "qw_w8a8_gemm", (W, ldw, sw, q, ldq, sx, T, Y, ldy, yt, N, K, None)


def linear(W=P, ldw=64, sw=P, x=P, xt=1, ldx=64, T=4, Y=P, ldy=32, yt=1, N=32, K=64, ws=P, wb=BIG):
    return "qw_w8a8_linear", (W, ldw, sw, x, xt, ldx, T, Y, ldy, yt, N, K, ws, wb, None)


def experts(w=(P,) * 6, E=8, H=64, F=32, lists=(P,) * 5, x=P, xt=1, T=4, k=2, h=P, yp=P, yt=2, ws=P, wb=BIG):
    return "qw_moe_experts_w8a8", (*w, E, H, F, *lists, x, xt, T, k, h, yp, yt, ws, wb, None)


def sort(e=P, T=4, E=8, k=2, tile_m=0, outs=(P,) * 6, tiles=(None,) * 3):
    return "qw_moe_sort", (e, T, E, k, tile_m, *outs, *tiles, None)


def permute(x=P, ldx=64, b=2, T=4, k=2, H=64, slot=P, xs=P, ldxs=64):
    return "qw_moe_permute", (x, ldx, b, T, k, H, slot, xs, ldxs, None)


def unpermute(yp=P, yt=1, ldyp=64, slot=P, w=P, T=4, k=2, H=64, out=P, ot=1, ldo=64):
    return "qw_moe_unpermute", (yp, yt, ldyp, slot, w, T, k, H, out, ot, ldo, None)


def grad(dout=P, dt=1, ldd=64, yp=P, yt=1, ldyp=64, slot=P, w=P, T=4, k=2, H=64, dyp=P, lddyp=64, dw=P):
    return "qw_moe_unpermute_backward", (dout, dt, ldd, yp, yt, ldyp, slot, w, T, k, H, dyp, lddyp, dw, None)


CALLS = {
    "quant null x": quant(x=None), "quant null q": quant(q=None), "quant null scale": quant(s=None),
    "quant type": quant(t=3), "quant K 40": quant(K=40, ldx=40, ldq=48), "quant K 0": quant(K=0),
    "quant K past the limit": quant(K=131072, ldx=131072, ldq=131072), "quant no rows": quant(T=0),
    "quant negative rows": quant(T=-1), "quant ldx": quant(ldx=63), "quant ldq": quant(ldq=72),
    "quant ldq short": quant(ldq=48), "quant q at 8": quant(q=EIGHT), "quant x odd": quant(x=ODD),
    "quant fp32 x at 2": quant(t=0, x=ctypes.c_void_p(4098)), "quant too many rows": quant(T=(1 << 23) + 1),
    "gemm null W": gemm(W=None), "gemm null sw": gemm(sw=None), "gemm null q": gemm(q=None), "gemm null sx": gemm(sx=None),
    "gemm null Y": gemm(Y=None), "gemm K 24": gemm(K=24), "gemm ldw": gemm(ldw=72), "gemm ldw short": gemm(ldw=48),
    "gemm W at 8": gemm(W=EIGHT), "gemm ldq": gemm(ldq=56), "gemm y type": gemm(yt=4), "gemm ldy": gemm(ldy=31),
    "gemm no rows": gemm(T=0), "gemm no columns": gemm(N=0), "gemm Y odd": gemm(Y=ODD),
    "gemm fp32 Y at 2": gemm(yt=0, Y=ctypes.c_void_p(4098)),
    "gemm too many outputs": gemm(T=1 << 20, N=1 << 20, ldy=1 << 20),
    "linear null x": linear(x=None), "linear x type": linear(xt=-1), "linear no workspace": linear(ws=None),
    "linear small workspace": linear(wb=256), "linear workspace at 8": linear(ws=EIGHT), "linear ldx": linear(ldx=60),
    "linear null W": linear(W=None),
    **{f"experts null weights {i}": experts(w=tuple(None if j == i else P for j in range(6))) for i in range(6)},
    **{f"experts null list {i}": experts(lists=tuple(None if j == i else P for j in range(5))) for i in range(5)},
    "experts E": experts(E=1025), "experts no expert": experts(E=0), "experts H": experts(H=72), "experts F": experts(F=40),
    "experts F 0": experts(F=0), "experts topk": experts(k=65), "experts topk 0": experts(k=0), "experts no token": experts(T=0),
    "experts slots": experts(T=1 << 22, k=4), "experts grid": experts(T=1 << 20, k=8, H=16384),
    "experts weights at 8": experts(w=(P, P, P, P, EIGHT, P)), "experts null h": experts(h=None),
    "experts null yp": experts(yp=None), "experts yp type": experts(yt=3), "experts small workspace": experts(wb=1023),
    "experts no workspace": experts(ws=None), "experts x type": experts(xt=7), "experts yp odd": experts(yp=ODD),
    "sort null": sort(e=None), "sort null output": sort(outs=(P, P, None, P, P, P)), "sort E": sort(E=1025),
    "sort E 0": sort(E=0), "sort T": sort(T=0), "sort topk": sort(k=65), "sort topk 0": sort(k=0),
    "sort pairs": sort(T=1 << 25, k=64), "sort tiles": sort(tile_m=-32), "sort tile_m": sort(tile_m=4096, tiles=(P,) * 3),
    "permute null x": permute(x=None), "permute null slot": permute(slot=None), "permute null xs": permute(xs=None),
    "permute 8 bytes": permute(b=8), "permute 3 bytes": permute(b=3), "permute ldx": permute(ldx=63),
    "permute ldxs": permute(ldxs=63), "permute H": permute(H=0), "permute T": permute(T=0),
    "permute odd 16-bit rows": permute(x=ODD), "permute many": permute(T=(1 << 23) + 1), "permute topk": permute(k=65),
    "unpermute null yp": unpermute(yp=None), "unpermute null out": unpermute(out=None), "unpermute null slot": unpermute(slot=None),
    "unpermute yp type": unpermute(yt=5), "unpermute out type": unpermute(ot=-1), "unpermute ldyp": unpermute(ldyp=63),
    "unpermute ldo": unpermute(ldo=63), "unpermute T": unpermute(T=0), "unpermute weights at 1": unpermute(w=ODD),
    "grad null dout": grad(dout=None), "grad nothing wanted": grad(dyp=None, dw=None), "grad dw without yp": grad(yp=None),
    "grad dout type": grad(dt=3), "grad yp type": grad(yt=3), "grad ldd": grad(ldd=63), "grad ldyp": grad(ldyp=63),
    "grad lddyp": grad(lddyp=63), "grad topk": grad(k=0), "grad null slot": grad(slot=None), "grad H": grad(H=-1),
}


@pytest.mark.parametrize("name", sorted(CALLS))
def test_refused(lib, name):
    fn, args = CALLS[name]
    assert getattr(lib, fn)(*args) == -1
    message = lib.qw_q4_last_error().decode()
    assert message.startswith(fn + ":"), message


def test_sizes(lib):
    assert lib.qw_w8a8_workspace_size(0, 64) == 0 and lib.qw_w8a8_workspace_size(4, 0) == 0
    assert lib.qw_w8a8_workspace_size(4096, 4096) >= 4096 * 4096 + 4096 * 4
    assert lib.qw_moe_w8a8_workspace_size(0, 8, 64, 64) == 0
    assert lib.qw_moe_w8a8_workspace_size(4096, 8, 4096, 1536) >= 4096 * 4096 + 4096 * 8 * 1536
    # sizes whose products pass 32 bits
    assert lib.qw_w8a8_workspace_size(1 << 20, 131056) >= (1 << 20) * 131056


def test_binding_refusals():
    """Shapes, types and tensors off the GPU, before any library call."""
    import torch
    W, sw = torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8)
    x, slot = torch.zeros(3, 32), torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="on the GPU"):
        qwq4.linear_w8a8(W, sw, x)
    with pytest.raises(ValueError, match="W is"):
        qwq4.linear_w8a8(W, sw, torch.zeros(3, 48))
    with pytest.raises(TypeError, match="W is"):
        qwq4.linear_w8a8(W.float(), sw, x)
    with pytest.raises(ValueError, match="sw is"):
        qwq4.linear_w8a8(W, sw[:7], x)
    with pytest.raises(ValueError, match="contiguous"):
        qwq4.linear_w8a8(W, sw, torch.zeros(32, 3).t())
    with pytest.raises(ValueError, match="contiguous"):
        qwq4.linear_w8a8(W, torch.zeros(16)[::2], x)
    with pytest.raises(TypeError, match="element type"):
        qwq4.linear_w8a8(W, sw, x.double())
    with pytest.raises(TypeError, match="the output is"):
        qwq4.linear_w8a8(W, sw, x, Y=torch.zeros(3, 8), y_dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="the output is"):
        qwq4.linear_w8a8(W, sw, x, Y=torch.zeros(3, 9))
    with pytest.raises(RuntimeError, match="on the GPU"):
        qwq4.quant_tokens_i8(x)
    with pytest.raises(TypeError, match="q is"):
        qwq4.gemm_w8a8(W, sw, x, torch.zeros(3))
    with pytest.raises(ValueError, match="sx is"):
        qwq4.gemm_w8a8(W, sw, torch.zeros(3, 32, dtype=torch.int8), torch.zeros(4))
    with pytest.raises(TypeError, match="top_e is"):
        qwq4.moe_sort(slot.long(), 4)
    with pytest.raises(ValueError, match="top_e is"):
        qwq4.moe_sort(slot.flatten(), 4)
    with pytest.raises(RuntimeError, match="on the GPU"):
        qwq4.moe_sort(slot, 4)
    with pytest.raises(ValueError, match="x is"):
        qwq4.moe_permute(torch.zeros(4, 32), slot)
    with pytest.raises(ValueError, match="xs is"):
        qwq4.moe_permute(x, slot, xs=torch.zeros(5, 32))
    with pytest.raises(TypeError, match="xs is"):
        qwq4.moe_permute(x, slot, xs=torch.zeros(6, 32).half())
    with pytest.raises(RuntimeError, match="on the GPU"):
        qwq4.moe_permute(x, slot)
    with pytest.raises(ValueError, match="yp is"):
        qwq4.moe_unpermute(torch.zeros(5, 32), slot)
    with pytest.raises(TypeError, match="tok_w is"):
        qwq4.moe_unpermute(torch.zeros(6, 32), slot, torch.zeros(3, 2).half())
    with pytest.raises(ValueError, match="dout is"):
        qwq4.moe_unpermute_backward(torch.zeros(3, 31), torch.zeros(6, 32), slot)
    with pytest.raises(TypeError, match="dyp is"):
        qwq4.moe_unpermute_backward(x, torch.zeros(6, 32), slot, dyp=torch.zeros(6, 32).half())
    with pytest.raises(RuntimeError, match="on the GPU"):
        qwq4.moe_unpermute_backward(x, torch.zeros(6, 32), slot)


def test_binding_wants_the_current_device(monkeypatch):
    """A tensor of another GPU than the current one is refused: its call would go to the wrong device's stream."""
    import types

    import torch
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda d: 70 + d, raising=False)
    on = lambda d: types.SimpleNamespace(is_cuda=True, get_device=lambda: d)  # noqa: E731
    assert qwq4._here("f", on(0), None, on(0)) == 70
    with pytest.raises(RuntimeError, match="f: a tensor is on GPU 1"):
        qwq4._here("f", on(0), on(1))
    with pytest.raises(RuntimeError, match="on the GPU"):
        qwq4._here("f", types.SimpleNamespace(is_cuda=False))


def test_experts_binding_refusals():
    import torch
    E, F, H, T, k = 4, 32, 48, 3, 2
    w = lambda *s: torch.zeros(s, dtype=torch.int8)  # noqa: E731
    gate, down = (w(E, F, H), torch.zeros(E, F)), (w(E, H, F), torch.zeros(E, H))
    route = qwq4.Route(T, E, k, "cpu", tile_m=qwq4.moe_w8a8_tile_m())
    x = torch.zeros(T, H)
    with pytest.raises(RuntimeError, match="on the GPU"):
        qwq4.moe_experts_w8a8(gate, gate, down, route, x)
    with pytest.raises(ValueError, match="tile list"):
        qwq4.moe_experts_w8a8(gate, gate, down, qwq4.Route(T, E, k, "cpu"), x)
    with pytest.raises(ValueError, match="down is"):
        qwq4.moe_experts_w8a8(gate, gate, gate, route, x)
    with pytest.raises(ValueError, match="up scales is"):
        qwq4.moe_experts_w8a8(gate, (gate[0], torch.zeros(E, H)), down, route, x)
    with pytest.raises(TypeError, match="gate is"):
        qwq4.moe_experts_w8a8((gate[0].float(), gate[1]), gate, down, route, x)
    with pytest.raises(ValueError, match="x is"):
        qwq4.moe_experts_w8a8(gate, gate, down, route, torch.zeros(T + 1, H))
    with pytest.raises(TypeError, match="h is"):
        qwq4.moe_experts_w8a8(gate, gate, down, route, x, h=torch.zeros(T * k, F))
    with pytest.raises(TypeError, match="yp is"):
        qwq4.moe_experts_w8a8(gate, gate, down, route, x, yp=torch.zeros(T * k, H), yp_dtype=torch.float16)
    with pytest.raises(ValueError, match="contiguous"):
        qwq4.moe_experts_w8a8(gate, gate, down, route, torch.zeros(H, T).t())


WIDE = {"permute": permute(H=(1 << 28) + 1, ldx=1 << 29, ldxs=1 << 29),
        "unpermute": unpermute(H=(1 << 28) + 1, ldyp=1 << 29, ldo=1 << 29),
        "grad": grad(H=(1 << 28) + 1, ldd=1 << 29, ldyp=1 << 29, lddyp=1 << 29)}


@pytest.mark.parametrize("name", sorted(WIDE))
def test_rows_too_wide(lib, name):
    fn, args = WIDE[name]
    assert getattr(lib, fn)(*args) == -1
    assert "2^28" in lib.qw_q4_last_error().decode()


def test_binding_refuses_what_passes_32_bits():
    """Sizes and strides that a 32-bit argument would cut, and workspaces with holes."""
    import torch
    big = 2**32 + 32
    wide = torch.empty_strided((3, 32), (big, 1), dtype=torch.float32, device="meta")
    slot = torch.zeros(3, 2, dtype=torch.int32)
    W, sw, x = torch.zeros(8, 32, dtype=torch.int8), torch.zeros(8), torch.zeros(3, 32)
    for call in (lambda: qwq4.quant_tokens_i8(wide), lambda: qwq4.linear_w8a8(W, sw, wide),
                 lambda: qwq4.moe_permute(wide, slot), lambda: qwq4.moe_unpermute_backward(wide, x.repeat(2, 1), slot),
                 lambda: qwq4.quant_tokens_i8(torch.empty((big, 16), device="meta")),
                 lambda: qwq4.quant_tokens_i8(torch.empty((1, big), device="meta"))):
        with pytest.raises(ValueError, match="2\\^31"):
            call()
    with pytest.raises(ValueError, match="2\\^30"):
        qwq4.moe_permute(torch.empty((big, 1), device="meta"), torch.empty((big, 1), dtype=torch.int32, device="meta"))
    for e, E in ((torch.empty((2**30, 1), dtype=torch.int32, device="meta"), 4), (slot, 1025), (slot, 0)):
        with pytest.raises(ValueError, match="need T \\* k below"):
            qwq4.moe_sort(e, E)
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        qwq4._space("f", torch.zeros(1, dtype=torch.uint8).expand(4096))
    assert qwq4._space("f", torch.zeros(8, 2)) == 64


def test_workspace_of_few_rows(lib):
    """One and two rows need no workspace as long as they fit a block; longer ones and more rows do."""
    assert lib.qw_w8a8_workspace_size(1, 4096) == 0 and lib.qw_w8a8_workspace_size(2, 32768) == 0
    assert lib.qw_w8a8_workspace_size(2, 32784) >= 2 * 32784 + 8 and lib.qw_w8a8_workspace_size(3, 64) >= 3 * 64 + 12
    for T, K in ((3, 64), (2, 32784)):
        fn, args = linear(T=T, K=K, ldw=K, ldx=K, ws=None, wb=0)
        assert getattr(lib, fn)(*args) == -1 and "workspace needs" in lib.qw_q4_last_error().decode()


def _combine_route(T=3, E=4, k=2):
    import torch
    r = qwq4.Route(T, E, k, "cpu")
    r.tok_slot.copy_(torch.arange(T * k, dtype=torch.int32).view(T, k))
    r.top_w.fill_(0.5)
    return r


@pytest.mark.parametrize("dtype", ["bfloat16", "float64", "int16", "int8"])
def test_combine_refuses_rows_it_would_misread(dtype):
    """moe_combine knows fp32 and fp16 rows: others (the bf16 yp that moe_experts_w8a8 can write) are refused, as the
    expert rows and as the shared ones, before anything is launched."""
    import torch
    r, bad, good = _combine_route(), torch.zeros(6, 8, dtype=getattr(torch, dtype)), torch.zeros(6, 8)
    with pytest.raises(TypeError, match="moe_combine: yp is torch." + dtype):
        qwq4.moe_combine(bad, r, 8)
    with pytest.raises(TypeError, match="moe_combine: shared is torch." + dtype):
        qwq4.moe_combine(good, r, 8, shared=bad[:3])
    for t in (torch.float32, torch.float16):  # (these go on to the check of the device)
        with pytest.raises(RuntimeError, match="on the GPU"):
            qwq4.moe_combine(good.to(t), r, 8, shared=good[:3].to(t))


def permute_grad(dxs=P, dt=1, lddxs=64, slot=P, T=4, k=2, H=64, dx=P, xt=1, lddx=64):
    return "qw_moe_permute_backward", (dxs, dt, lddxs, slot, T, k, H, dx, xt, lddx, None)


PERMUTE_GRAD = {
    "null dxs": permute_grad(dxs=None), "null dx": permute_grad(dx=None), "null slot": permute_grad(slot=None),
    "dxs type": permute_grad(dt=3), "dx type": permute_grad(xt=-1), "lddxs": permute_grad(lddxs=63),
    "lddx": permute_grad(lddx=63), "T": permute_grad(T=0), "topk": permute_grad(k=65), "H": permute_grad(H=0),
    "too wide": permute_grad(H=(1 << 28) + 1, lddxs=1 << 29, lddx=1 << 29), "dx odd": permute_grad(dx=ODD),
}


@pytest.mark.parametrize("name", sorted(PERMUTE_GRAD))
def test_permute_gradient_refused(lib, name):
    fn, args = PERMUTE_GRAD[name]
    assert getattr(lib, fn)(*args) == -1
    assert lib.qw_q4_last_error().decode().startswith("qw_moe_permute_backward:")


def test_permute_gradient_binding_refusals():
    import torch
    slot = torch.zeros(3, 2, dtype=torch.int32)
    with pytest.raises(ValueError, match="moe_permute_backward: dxs is"):
        qwq4.moe_permute_backward(torch.zeros(5, 32), slot)
    with pytest.raises(TypeError, match="element type"):
        qwq4.moe_permute_backward(torch.zeros(6, 32, dtype=torch.int8), slot)
    with pytest.raises(TypeError, match="moe_permute_backward: the output is"):
        qwq4.moe_permute_backward(torch.zeros(6, 32), slot, dx=torch.zeros(3, 32), dx_dtype=torch.float16)
    with pytest.raises(RuntimeError, match="moe_permute_backward: all tensors must be on the GPU"):
        qwq4.moe_permute_backward(torch.zeros(6, 32), slot)


def test_sort_into_a_route_keeps_the_routers_buffers(monkeypatch):
    """moe_sort(out=route) shows the given choices as route.top_e; the next moe_route into it writes the route's own
    buffers again, not the caller's choices, and a Route that moe_sort made has none to write."""
    import types

    import torch
    calls = []
    stub = types.SimpleNamespace(qw_moe_sort=lambda *a: calls.append(("sort", a)) or 0,
                                 qw_moe_route=lambda *a: calls.append(("route", a)) or 0)
    monkeypatch.setattr(qwq4, "lib", lambda: stub)
    monkeypatch.setattr(qwq4, "_here", lambda *a: None)
    monkeypatch.setattr(qwq4, "_dev", lambda *a: None)
    monkeypatch.setattr(qwq4, "_stream", lambda: None)
    T, E, k = 5, 4, 2
    r = qwq4.Route(T, E, k, "cpu")
    own_e, own_w, logits = r.top_e, r.top_w, torch.zeros(T, E)
    for _ in range(2):
        for e in (torch.zeros(T, k, dtype=torch.int32), torch.ones(T, k, dtype=torch.int32)):
            assert qwq4.moe_sort(e, E, out=r) is r and r.top_e is e and r.top_w is None
        r.top_w = torch.ones(T, k)  # (the caller's weights of these choices)
        assert qwq4.moe_route(logits, k, out=r) is r and r.top_e is own_e and r.top_w is own_w
        assert calls[-1][0] == "route" and calls[-1][1][5:7] == (own_e.data_ptr(), own_w.data_ptr())
    w = torch.ones(T, k)
    r.top_w = w  # (buffers that a caller put there stay: no sort came between)
    assert qwq4.moe_route(logits, k, out=r).top_w is w
    n, made = len(calls) + 1, qwq4.moe_sort(own_e, E)
    made.top_w = torch.ones(T, k)
    with pytest.raises(ValueError, match="moe_route: out was made by moe_sort"):
        qwq4.moe_route(logits, k, out=made)
    assert len(calls) == n and made.top_e is own_e


def test_combine_of_a_sorted_route_wants_weights(monkeypatch):
    """A route of given choices has no router's weights: moe_combine takes them as tok_w (fp32 [T][k]), and without
    any says what is missing."""
    import types

    import torch
    r, yp, w = _combine_route(), torch.zeros(6, 8), torch.ones(3, 2)
    r.top_w = None
    with pytest.raises(ValueError, match="moe_combine: the route has no weights"):
        qwq4.moe_combine(yp, r, 8)
    with pytest.raises(ValueError, match="tok_w is"):
        qwq4.moe_combine(yp, r, 8, tok_w=torch.ones(3, 3))
    with pytest.raises(TypeError, match="tok_w is"):
        qwq4.moe_combine(yp, r, 8, tok_w=w.half())
    with pytest.raises(ValueError, match="tok_w must be contiguous"):
        qwq4.moe_combine(yp, r, 8, tok_w=torch.ones(2, 3).t())
    with pytest.raises(RuntimeError, match="on the GPU"):
        qwq4.moe_combine(yp, r, 8, tok_w=w)
    seen = []
    monkeypatch.setattr(qwq4, "lib", lambda: types.SimpleNamespace(qw_moe_combine=lambda *a: seen.append(a[3]) or 0))
    monkeypatch.setattr(qwq4, "_dev", lambda *a: None)
    monkeypatch.setattr(qwq4, "_stream", lambda: None)
    qwq4.moe_combine(yp, r, 8, tok_w=w)
    r.top_w = torch.ones(3, 2)  # (a router's, or set by the caller; tok_w goes before it)
    qwq4.moe_combine(yp, r, 8)
    qwq4.moe_combine(yp, r, 8, tok_w=w)
    assert seen == [w.data_ptr(), r.top_w.data_ptr(), w.data_ptr()]


def test_expert_rows_refuse_what_autograd_follows():
    """A result that is cut off from its inputs would train nothing and say nothing."""
    import torch
    x, yp, w = (torch.zeros(*s, requires_grad=True) for s in ((3, 32), (6, 32), (3, 2)))
    slot = torch.zeros(3, 2, dtype=torch.int32)
    calls = (("moe_permute", lambda: qwq4.moe_permute(x, slot)), ("moe_unpermute", lambda: qwq4.moe_unpermute(yp, slot)),
             ("moe_unpermute", lambda: qwq4.moe_unpermute(yp.detach(), slot, w)))
    for fn, call in calls:
        with pytest.raises(RuntimeError, match=fn + ": an input requires grad.*" + fn + "_backward"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="on the GPU"):  # (goes on to the check of the device)
            call()


def test_lists_of_any_object(monkeypatch):
    """moe_route and moe_sort write into any object that has a Route's lists."""
    import types

    import torch
    calls = []
    stub = types.SimpleNamespace(qw_moe_sort=lambda *a: calls.append(a) or 0, qw_moe_route=lambda *a: calls.append(a) or 0)
    monkeypatch.setattr(qwq4, "lib", lambda: stub)
    monkeypatch.setattr(qwq4, "_here", lambda *a: None)
    monkeypatch.setattr(qwq4, "_dev", lambda *a: None)
    monkeypatch.setattr(qwq4, "_stream", lambda: None)
    like = types.SimpleNamespace(**vars(qwq4.Route(3, 4, 2, "cpu")))
    own_e, own_w, e = like.top_e, like.top_w, torch.zeros(3, 2, dtype=torch.int32)
    assert qwq4.moe_route(torch.zeros(3, 4), 2, out=like) is like
    assert qwq4.moe_sort(e, 4, out=like) is like and like.top_e is e
    assert qwq4.moe_route(torch.zeros(3, 4), 2, out=like).top_e is own_e and like.top_w is own_w and len(calls) == 3
