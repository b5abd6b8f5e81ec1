"""The W8A8 products (qw_quant_tokens_i8, qw_w8a8_gemm, qw_w8a8_linear and the
routed experts qw_moe_experts_w8a8) against plain numpy. The sums are of whole
numbers and every rounding is defined, so quantised rows, scales and products
are compared bit for bit; h alone has a tolerance, for its exponential."""
import numpy as np
import pytest

import qwq4
import _w8a8_ref as ref
from _gpu_util import host, to_dev

pytestmark = pytest.mark.gpu

GUARD = 12345.0


def _types():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _rows(seed, T, K, t, gpu, pad=0):
    """(device rows of type t with a stride of K + pad, their fp32 values)."""
    import torch
    v = np.random.default_rng(seed).standard_normal((T, K + pad)).astype(np.float32)
    v[:, ::37] *= 8
    d = torch.from_numpy(v).to(gpu).to(_types()[t])
    return d[:, :K], host(d).astype(np.float32)[:, :K]


def _weights(seed, N, K, gpu, pad=0):
    r = np.random.default_rng(seed)
    W = r.integers(-128, 128, (N, K + pad), dtype=np.int8)
    sw = ((0.5 + r.random(N)) / (73 * K**0.5)).astype(np.float32)
    return to_dev(W, gpu)[:, :K], to_dev(sw, gpu), W[:, :K], sw


def _same(y, want):
    y, want = np.asarray(host(y), np.float32), np.asarray(want, np.float32)
    assert y.shape == want.shape
    assert np.array_equal(np.isnan(y), np.isnan(want))
    assert np.array_equal(y[~np.isnan(y)], want[~np.isnan(want)])


# ------------------------------------------------------------- quantiser
@pytest.mark.parametrize("t", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T,K,pad", [(1, 16, 0), (3, 48, 0), (5, 4096, 0), (37, 1040, 3), (66, 2560, 8), (2, 20000, 0)])
def test_quant_tokens(gpu, t, T, K, pad):
    x, v = _rows(1, T, K, t, gpu, pad)
    q, sc = qwq4.quant_tokens_i8(x)
    qr, sr = ref.quant(v)
    assert np.array_equal(host(q).astype(np.float64), qr)
    assert np.array_equal(host(sc).view(np.uint32), sr.view(np.uint32))


def test_quant_tokens_extreme_rows(gpu):
    """Zeros, the smallest and largest numbers, ties at half a step, infinities and NaN, each in a row of its own."""
    import torch
    K = 64
    v = np.random.default_rng(2).standard_normal((9, K)).astype(np.float32)
    v[0] = 0
    v[1] = 0
    v[1, 5] = 1e-45
    v[2] *= np.float32(1e-38)
    v[3] = np.float32(3.3e38) * np.sign(v[3])
    v[4] = np.arange(K) * 0.5
    v[4, 0] = 127.0
    v[5, 7] = np.inf
    v[6, 60] = np.nan
    v[7] = -0.0
    v[7, 3] = -1.0
    q, sc = qwq4.quant_tokens_i8(torch.from_numpy(v).to(gpu))
    qr, sr = ref.quant(v)
    assert np.array_equal(host(q).astype(np.float64), qr)
    assert np.array_equal(np.isnan(host(sc)), np.isnan(sr)) and np.isnan(host(sc)).sum() == 2
    assert np.array_equal(host(sc)[~np.isnan(sr)], sr[~np.isnan(sr)])
    # 16-bit subnormals
    h = torch.full((1, K), 6e-8, dtype=torch.float16, device=gpu)
    b = torch.full((1, K), 1e-40, dtype=torch.bfloat16, device=gpu)
    for d in (h, b):
        q, sc = qwq4.quant_tokens_i8(d)
        qr, sr = ref.quant(host(d).astype(np.float32))
        assert np.array_equal(host(q).astype(np.float64), qr) and np.array_equal(host(sc), sr)


def test_quant_tokens_strided_q(gpu):
    """Rows of q apart; what lies between them is not written."""
    import torch
    x, v = _rows(3, 6, 80, "bf16", gpu)
    wide = torch.full((6, 112), 99, dtype=torch.int8, device=gpu)
    qwq4.quant_tokens_i8(x, q=wide[:, :80])
    assert np.array_equal(host(wide)[:, :80].astype(np.float64), ref.quant(v)[0])
    assert (host(wide)[:, 80:] == 99).all()


# --------------------------------------------------------------- products
@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 33, 64, 65, 100, 129, 257, 600, 1030])
@pytest.mark.parametrize("N,K", [(1, 16), (33, 144), (100, 2064), (257, 1024), (1000, 400)])
def test_gemm_bits(gpu, T, N, K):
    """Every size around the tiles' edges: ragged rows, columns and K."""
    print(f"gemm_w8a8 T={T} N={N} K={K}", flush=True)
    Wd, swd, W, sw = _weights(10 * N + K, N, K, gpu)
    x, v = _rows(T, T, K, "bf16", gpu)
    q, sx = ref.quant(v)
    for t in (("f32",) if T % 2 else ("bf16", "f16")):
        y = qwq4.gemm_w8a8(Wd, swd, *qwq4.quant_tokens_i8(x), y_dtype=_types()[t])
        _same(y, ref.ROUND[t](ref.product(q, sx, W, sw)))


@pytest.mark.parametrize("xt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("T", [1, 2, 4, 6, 12, 37, 130, 1100])
@pytest.mark.parametrize("N,K", [(384, 4096), (75, 336), (2000, 128)])
def test_linear_is_quantiser_and_product(gpu, xt, T, N, K):
    print(f"linear_w8a8 T={T} N={N} K={K} {xt}", flush=True)
    Wd, swd, W, sw = _weights(5, N, K, gpu)
    x, v = _rows(6 + T, T, K, xt, gpu)
    for t in ("f32", "bf16", "f16"):
        _same(qwq4.linear_w8a8(Wd, swd, x, y_dtype=_types()[t]),
              ref.ROUND[t](ref.product(*ref.quant(v), W, sw)))


@pytest.mark.parametrize("T", [1, 3, 20, 70, 300])
def test_strides_and_guards(gpu, T):
    """Weights, rows and outputs inside wider matrices (rows of x and y at odd strides, not 16-byte aligned); nothing
    is written beside the outputs."""
    import torch
    N, K = 129, 272
    Wd, swd, W, sw = _weights(8, N, K, gpu, pad=48)
    for xt, pad in (("bf16", 3), ("f32", 1), ("f16", 8)):
        x, v = _rows(9, T, K, xt, gpu, pad=pad)
        want = ref.product(*ref.quant(v), W, sw)
        for yt in ("f32", "bf16"):
            wide = torch.full((T + 2, N + 7), GUARD, dtype=_types()[yt], device=gpu)
            keep = host(wide).copy()
            qwq4.linear_w8a8(Wd, swd, x, Y=wide[1:T + 1, 3:3 + N])
            got = host(wide)
            _same(wide[1:T + 1, 3:3 + N], ref.ROUND[yt](want))
            got = got.copy()
            got[1:T + 1, 3:3 + N] = keep[1:T + 1, 3:3 + N]
            assert np.array_equal(got, keep)


@pytest.mark.parametrize("T", [1, 5, 40, 150])
def test_bad_rows_stay_alone(gpu, T):
    """A row with a NaN or an infinity is NaN in the output; the others are what they are without it."""
    import torch
    N, K = 70, 256
    Wd, swd, W, sw = _weights(11, N, K, gpu)
    x, v = _rows(12, T, K, "f32", gpu)
    v = v.copy()
    v[T // 2, 200] = np.inf
    if T > 2:
        v[T - 1, 0] = np.nan
        v[0] = 0
    y = qwq4.linear_w8a8(Wd, swd, torch.from_numpy(v).to(gpu))
    _same(y, ref.product(*ref.quant(v), W, sw))


@pytest.mark.parametrize("T", [1, 9, 200])
def test_largest_sums(gpu, T):
    """K at its limit with every int8 at -128: the largest sum there is, just inside int32; and a fp16 output beyond
    its range."""
    import torch
    K, N = 131056, 5
    W = torch.full((N, K), -128, dtype=torch.int8, device=gpu)
    W[1] = 127
    q = torch.full((T, K), -128, dtype=torch.int8, device=gpu)
    sw = torch.tensor([1.0, 1.0, 1e-5, -1.0, 0.0], device=gpu)
    sx = torch.full((T,), 0.5, device=gpu)
    want = ref.product(np.full((T, K), -128.0), np.full(T, 0.5, np.float32), host(W), host(sw))
    _same(qwq4.gemm_w8a8(W, sw, q, sx, y_dtype=torch.float32), want)
    got = host(qwq4.gemm_w8a8(W, sw, q, sx, y_dtype=torch.float16)).astype(np.float32)
    assert np.array_equal(got, ref.f16(want)) and got.max() == 65504 and got.min() == -65504


@pytest.mark.parametrize("T", [6, 300])
def test_rows_do_not_depend_on_the_batch(gpu, T):
    import torch
    Wd, swd, _, _ = _weights(14, 513, 1168, gpu)
    x, _ = _rows(15, T, 1168, "f16", gpu)
    whole = qwq4.linear_w8a8(Wd, swd, x)
    for lo, hi in ((0, 1), (T - 1, T), (1, 4), (2, T)):
        assert torch.equal(whole[lo:hi], qwq4.linear_w8a8(Wd, swd, x[lo:hi]))


def test_outputs_past_32_bits(gpu):
    """More than 2^31 output elements: the last rows are where they belong."""
    import torch
    T, N, K = 66000, 33000, 16
    Wd, swd, W, sw = _weights(16, N, K, gpu)
    x, v = _rows(17, T, K, "f16", gpu)
    y = qwq4.linear_w8a8(Wd, swd, x)
    for rows in (slice(0, 2), slice(65070, 65080), slice(T - 3, T)):
        _same(y[rows], ref.f16(ref.product(*ref.quant(v[rows]), W, sw)))


# ----------------------------------------------------------------- experts
def _experts(seed, E, H, F, gpu):
    r = np.random.default_rng(seed)
    out = []
    for n, k in ((F, H), (F, H), (H, F)):
        W = r.integers(-127, 128, (E, n, k), dtype=np.int8)
        s = ((0.5 + r.random((E, n))) * 1.5 / (73 * k**0.5)).astype(np.float32)
        out.append(((to_dev(W, gpu), to_dev(s, gpu)), (W, s)))
    return [o[0] for o in out], [o[1] for o in out]


def _choices(seed, T, E, k, kind):
    r = np.random.default_rng(seed)
    e = np.argsort(r.random((T, E)), axis=1)[:, :k].astype(np.int32)
    if kind == "one":      # every token to the same expert first
        e[:, 0] = E - 1
        e[:, 1:] = np.where(e[:, 1:] == E - 1, 0, e[:, 1:])
    if kind == "dropped":  # experts elsewhere, some tokens without any
        e[r.random((T, k)) < 0.4] = -1
        e[:: 3] = E + 5
    if kind == "repeated":
        e[:] = e[:, :1]
    return e


def _check_experts(gpu, T, E, k, H, F, xt, yt, kind, seed=21):
    import torch
    (g, u, d), (gr, ur, dr) = _experts(seed, E, H, F, gpu)
    x, v = _rows(seed + 1, T, H, xt, gpu)
    e = _choices(seed + 2, T, E, k, kind)
    r = qwq4.moe_sort(to_dev(e, gpu), E, tile_m=qwq4.moe_w8a8_tile_m())
    h = torch.full((T * k, F), GUARD, dtype=torch.float16, device=gpu)
    yp = torch.full((T * k, H), GUARD, dtype=_types()[yt], device=gpu)
    qwq4.moe_experts_w8a8(g, u, d, r, x, h=h, yp=yp)
    hs, ys = host(h).astype(np.float32), np.asarray(host(yp), np.float32)
    _, offsets, _, tok = ref.sort(e, E)
    q, sx = ref.quant(v)
    for i in range(E):
        at = slice(offsets[i], offsets[i + 1])
        t = tok[at]
        if not len(t):
            continue
        gate = ref.product(q[t], sx[t], gr[0][i], gr[1][i]).astype(np.float64)
        up = ref.product(q[t], sx[t], ur[0][i], ur[1][i]).astype(np.float64)
        want = gate / (1 + np.exp(-gate)) * up
        # fp16's half step 2^-11; sigmoid and the products in fp32: the exponential's argument and result
        # are off by at most about (|gate| + 4) 2^-24 (|gate| < 64 here) and five roundings follow: below 2^-16 together
        assert np.abs(gate).max() < 64
        assert np.all(np.abs(hs[at] - want) <= np.abs(want) * (2.0**-11 + 2.0**-16) + 2.0**-25)
        # from the h that the call wrote, the down projection's bits
        qh, sh = ref.quant(hs[at])
        assert np.array_equal(ys[at], ref.ROUND[yt](ref.product(qh, sh, dr[0][i], dr[1][i])))
    guard = np.float32(ref.ROUND[yt](np.float32(GUARD)))
    assert (hs[offsets[E]:] == np.float16(GUARD)).all() and (ys[offsets[E]:] == guard).all()


@pytest.mark.parametrize("T", [1, 2, 7, 33, 100, 700])
@pytest.mark.parametrize("E,k,H,F,xt,yt", [(8, 2, 272, 144, "bf16", "f32"), (16, 4, 512, 384, "f16", "f16"),
                                           (60, 8, 128, 80, "f32", "bf16")])
def test_experts(gpu, T, E, k, H, F, xt, yt):
    print(f"experts_w8a8 T={T} E={E} k={k} H={H} F={F}", flush=True)
    _check_experts(gpu, T, E, k, H, F, xt, yt, "spread")


@pytest.mark.parametrize("kind", ["one", "dropped", "repeated"])
@pytest.mark.parametrize("T", [1, 6, 45, 400])
def test_experts_uneven(gpu, T, kind):
    """All tokens on one expert (many tiles of it), choices without a slot, the same expert twice."""
    print(f"experts_w8a8 {kind} T={T}", flush=True)
    _check_experts(gpu, T, 12, 3, 160, 208, "bf16", "bf16", kind)


def test_experts_no_slot_at_all(gpu):
    _check_experts(gpu, 5, 4, 2, 64, 64, "bf16", "f16", "spread", seed=31)
    import torch
    (g, u, d), _ = _experts(1, 4, 64, 64, gpu)
    r = qwq4.moe_sort(torch.full((5, 2), -1, dtype=torch.int32, device=gpu), 4, tile_m=qwq4.moe_w8a8_tile_m())
    yp = torch.full((10, 64), GUARD, device=gpu)
    qwq4.moe_experts_w8a8(g, u, d, r, torch.randn(5, 64, device=gpu), yp=yp)
    assert (yp == GUARD).all()


def test_experts_route_and_bad_rows(gpu):
    """A route of qw_moe_route serves as well; a NaN row touches its own slots only."""
    import torch
    T, E, k, H, F = 50, 8, 2, 256, 128
    (g, u, d), _ = _experts(41, E, H, F, gpu)
    x, _ = _rows(42, T, H, "bf16", gpu)
    logits = torch.from_numpy(np.random.default_rng(43).standard_normal((T, E)).astype(np.float32)).to(gpu)
    r = qwq4.moe_route(logits, k, tile_m=qwq4.moe_w8a8_tile_m())
    h, yp = qwq4.moe_experts_w8a8(g, u, d, r, x)
    s = qwq4.moe_sort(r.top_e, E, tile_m=qwq4.moe_w8a8_tile_m())
    for name in ("counts", "offsets", "tok_slot", "pair_tok", "n_active", "n_tiles"):
        assert torch.equal(getattr(r, name), getattr(s, name)), name
    assert torch.equal(yp, qwq4.moe_experts_w8a8(g, u, d, s, x)[1])
    x2 = x.clone()
    x2[7, 3] = float("nan")
    _, yp2 = qwq4.moe_experts_w8a8(g, u, d, r, x2)
    mine = torch.zeros(T * k, dtype=torch.bool, device=gpu)
    mine[r.tok_slot[7].long()] = True
    assert torch.isnan(yp2[mine]).all() and torch.equal(yp2[~mine], yp[~mine])


def test_experts_rows_do_not_depend_on_the_batch(gpu):
    import torch
    T, E, k, H, F = 90, 6, 2, 400, 176
    (g, u, d), _ = _experts(51, E, H, F, gpu)
    x, _ = _rows(52, T, H, "f16", gpu)
    e = to_dev(_choices(53, T, E, k, "spread"), gpu)

    def rows(lo, hi):
        r = qwq4.moe_sort(e[lo:hi].contiguous(), E, tile_m=qwq4.moe_w8a8_tile_m())
        yp = qwq4.moe_experts_w8a8(g, u, d, r, x[lo:hi])[1]
        return yp[r.tok_slot.long()]
    whole = rows(0, T)
    for lo, hi in ((0, 1), (40, 43), (10, 75)):
        assert torch.equal(whole[lo:hi], rows(lo, hi))


# ------------------------------------------------ a layer, streams, graphs
def test_layer_graph_and_streams(gpu):
    """sort -> experts -> unpermute and a projection, together as a decode layer runs them: on a stream of its own,
    and captured and replayed with new inputs between eager calls; every replay gives the eager call's bits."""
    import torch
    T, E, k, H, F, N = 6, 16, 4, 512, 256, 640
    (g, u, d), _ = _experts(61, E, H, F, gpu)
    Wd, swd, _, _ = _weights(62, N, H, gpu)
    x = torch.empty((T, H), dtype=torch.bfloat16, device=gpu)
    e = torch.empty((T, k), dtype=torch.int32, device=gpu)
    w = torch.empty((T, k), device=gpu)
    ws = torch.empty(qwq4.moe_w8a8_workspace_size(T, k, H, F), dtype=torch.uint8, device=gpu)
    ws2 = torch.empty(qwq4.w8a8_workspace_size(T, H), dtype=torch.uint8, device=gpu)

    def layer(xi, ei, wi, a, b):
        r = qwq4.moe_sort(ei, E, tile_m=qwq4.moe_w8a8_tile_m())
        h, yp = qwq4.moe_experts_w8a8(g, u, d, r, xi, workspace=a)
        out = qwq4.moe_unpermute(yp, r.tok_slot, wi, out_dtype=torch.bfloat16)
        return qwq4.linear_w8a8(Wd, swd, out, y_dtype=torch.float32, workspace=b)

    def fill(seed):
        r = np.random.default_rng(seed)
        x.copy_(torch.from_numpy(r.standard_normal((T, H)).astype(np.float32)))
        e.copy_(torch.from_numpy(_choices(seed, T, E, k, "dropped" if seed % 2 else "spread")))
        w.copy_(torch.from_numpy(r.random((T, k)).astype(np.float32)))

    fill(0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        on_side = layer(x, e, w, ws, ws2)
    torch.cuda.synchronize()
    assert torch.equal(on_side, layer(x, e, w, ws, ws2))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = layer(x, e, w, ws, ws2)
    for seed in (1, 2, 3, 4):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = captured.clone()
        eager = layer(x.clone(), e.clone(), w.clone(), None, None)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)


# -------------------------------------------------- edges of the kernels' choice
@pytest.mark.parametrize("T", [3, 8, 9, 15, 16, 17, 24])
@pytest.mark.parametrize("E,k", [(3, 2), (40, 5)])
def test_experts_few_tokens(gpu, T, E, k):
    """Around the number of tokens up to which the weights are streamed, with few and many slots per expert."""
    print(f"experts_w8a8 T={T} E={E} k={k}", flush=True)
    _check_experts(gpu, T, E, k, 208, 336, "f16", "bf16", "spread", seed=71)


@pytest.mark.parametrize("xt", ["bf16", "f32"])
@pytest.mark.parametrize("T", [1, 8, 40])
def test_experts_buffers_at_any_address(gpu, T, xt):
    """Rows, h and yp that start at their element's alignment only."""
    import torch
    E, k, H, F = 6, 2, 144, 80
    (g, u, d), _ = _experts(81, E, H, F, gpu)
    x, _ = _rows(82, T, H, xt, gpu)
    r = qwq4.moe_sort(to_dev(_choices(83, T, E, k, "spread"), gpu), E, tile_m=qwq4.moe_w8a8_tile_m())

    def odd(shape, dtype):
        return torch.empty(shape[0] * shape[1] + 1, dtype=dtype, device=gpu)[1:].view(shape)
    x1 = odd((T, H), x.dtype)
    x1.copy_(x)
    h, yp = qwq4.moe_experts_w8a8(g, u, d, r, x, yp_dtype=torch.bfloat16)
    h1, yp1 = qwq4.moe_experts_w8a8(g, u, d, r, x1, h=odd((T * k, F), torch.float16),
                                    yp=odd((T * k, H), torch.bfloat16))
    assert torch.equal(h, h1) and torch.equal(yp, yp1)


@pytest.mark.parametrize("T,K", [(1, 65536), (2, 32768), (3, 16384), (4, 16384), (4, 16400), (1, 65552)])
def test_gemv_longest_rows(gpu, T, K):
    """The longest rows that are staged whole, and the next longer ones."""
    Wd, swd, W, sw = _weights(91, 40, K, gpu)
    x, v = _rows(92, T, K, "bf16", gpu)
    _same(qwq4.linear_w8a8(Wd, swd, x), ref.bf16(ref.product(*ref.quant(v), W, sw)))


@pytest.mark.parametrize("T", [1, 2, 8])
def test_experts_longest_rows(gpu, T):
    _check_experts(gpu, T, 2, 1, 8192, 48, "bf16", "f32", "spread", seed=95)
    _check_experts(gpu, T, 2, 1, 8208, 48, "bf16", "f32", "spread", seed=96)
    _check_experts(gpu, T, 2, 1, 48, 8192, "bf16", "f32", "spread", seed=97)


def test_two_streams_at_once(gpu):
    """Calls in flight on two streams, each with its own workspace."""
    import torch
    T, N, K, E, k, H, F = 300, 700, 1024, 8, 2, 256, 192
    Wd, swd, _, _ = _weights(101, N, K, gpu)
    x, _ = _rows(102, T, K, "bf16", gpu)
    (g, u, d), _ = _experts(103, E, H, F, gpu)
    xe, _ = _rows(104, T, H, "f16", gpu)
    r = qwq4.moe_sort(to_dev(_choices(105, T, E, k, "spread"), gpu), E, tile_m=qwq4.moe_w8a8_tile_m())
    want_y, (_, want_yp) = qwq4.linear_w8a8(Wd, swd, x), qwq4.moe_experts_w8a8(g, u, d, r, xe)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = []
    for _ in range(4):
        with torch.cuda.stream(a):
            y = qwq4.linear_w8a8(Wd, swd, x)
        with torch.cuda.stream(b):
            yp = qwq4.moe_experts_w8a8(g, u, d, r, xe)[1]
        got.append((y, yp))
    torch.cuda.synchronize()
    for y, yp in got:
        assert torch.equal(y, want_y) and torch.equal(yp, want_yp)


@pytest.mark.parametrize("T", [4, 5, 9, 16, 17])
@pytest.mark.parametrize("F", [2048, 2032])
def test_large_experts_few_tokens(gpu, T, F):
    """Large experts stream their weights for more tokens than small ones; both sides of the edge."""
    print(f"experts_w8a8 T={T} F={F}", flush=True)
    _check_experts(gpu, T, 3, 2, 2048, F, "bf16", "f16", "uneven", seed=111)
    _check_experts(gpu, T, 3, 2, 2048, F, "f16", "f32", "one", seed=115)


@pytest.mark.parametrize("K", [16, 64, 128, 144, 256, 272, 384, 400])
@pytest.mark.parametrize("T,N", [(20, 300), (60, 9000), (100, 20000), (300, 25000)])
def test_fewer_stages_than_buffers(gpu, T, N, K):
    """Rows of one to four stages: loads that nobody reads must have landed before their buffers are used again."""
    print(f"gemm_w8a8 T={T} N={N} K={K}", flush=True)
    Wd, swd, W, sw = _weights(121, N, K, gpu)
    r = np.random.default_rng(122)
    q, sx = r.integers(-127, 128, (T, K), dtype=np.int8), (r.random(T) + 0.5).astype(np.float32)
    _same(qwq4.gemm_w8a8(Wd, swd, to_dev(q, gpu), to_dev(sx, gpu)), ref.bf16(ref.product(q, sx, W, sw)))


@pytest.mark.parametrize("H,F", [(16, 16), (128, 128), (64, 256), (256, 112), (272, 400)])
@pytest.mark.parametrize("T", [40, 700])
def test_experts_of_few_stages(gpu, T, H, F):
    """The same for the experts, whose blocks run several tiles in the same buffers."""
    print(f"experts_w8a8 T={T} H={H} F={F}", flush=True)
    _check_experts(gpu, T, 4, 2, H, F, "bf16", "bf16", "one", seed=131)


@pytest.mark.parametrize("K", [496, 512, 528, 1040, 1168, 1552, 2064])
@pytest.mark.parametrize("T,N", [(3, 8191), (3, 8193), (32, 10001), (33, 4096), (33, 4128), (64, 8192), (64, 8193), (45, 7003)])
def test_split_tiles(gpu, T, N, K):
    """Waves that split K, with even and uneven shares, one or two tiles side by side, and the next larger tiles."""
    print(f"gemm_w8a8 T={T} N={N} K={K}", flush=True)
    Wd, swd, W, sw = _weights(141, N, K, gpu)
    r = np.random.default_rng(142)
    q, sx = r.integers(-128, 128, (T, K), dtype=np.int8), (r.random(T) + 0.5).astype(np.float32)
    want = ref.product(q, sx, W, sw)
    for t in ("bf16", "f32"):
        _same(qwq4.gemm_w8a8(Wd, swd, to_dev(q, gpu), to_dev(sx, gpu), y_dtype=_types()[t]), ref.ROUND[t](want))


@pytest.mark.parametrize("T", [1, 2])
def test_few_rows_without_workspace(gpu, T):
    import torch
    Wd, swd, W, sw = _weights(151, 70, 528, gpu)
    x, v = _rows(152, T, 528, "bf16", gpu)
    want = ref.bf16(ref.product(*ref.quant(v), W, sw))
    for ws in (None, torch.empty(0, dtype=torch.uint8, device=gpu), torch.empty(4096, dtype=torch.uint8, device=gpu)):
        _same(qwq4.linear_w8a8(Wd, swd, x, workspace=ws), want)
