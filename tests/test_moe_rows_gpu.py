"""Tokens sorted by expert and back (qw_moe_sort, qw_moe_permute, qw_moe_unpermute,
qw_moe_unpermute_backward) against plain numpy. Lists and moved rows are compared
exactly; sums against float64 within the roundings they are made of."""
import numpy as np
import pytest

import qwq4
import _w8a8_ref as ref
from _gpu_util import host, to_dev

pytestmark = pytest.mark.gpu

GUARD = 77.0
HALF = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}  # half a step, relative
SMALLEST = {"f32": 2.0**-150, "bf16": 2.0**-134, "f16": 2.0**-25}  # half the smallest step


def _types():
    import torch
    return {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def _choices(seed, T, E, k, kind="spread"):
    r = np.random.default_rng(seed)
    e = r.integers(0, E, (T, k)).astype(np.int32)
    if kind == "dropped":
        e[r.random((T, k)) < 0.3] = -1
        e[r.random((T, k)) < 0.1] = E
        e[r.random((T, k)) < 0.05] = np.iinfo(np.int32).min
        e[r.random((T, k)) < 0.05] = np.iinfo(np.int32).max
    if kind == "none":
        e[:] = -1
    if kind == "one":
        e[:] = E - 1
    return e


def _floats(seed, shape, t, gpu, pad=0):
    import torch
    v = np.random.default_rng(seed).standard_normal((shape[0], shape[1] + pad)).astype(np.float32)
    d = torch.from_numpy(v).to(gpu).to(_types()[t])
    return d[:, :shape[1]], host(d).astype(np.float64)[:, :shape[1]]


# ------------------------------------------------------------------- sort
@pytest.mark.parametrize("kind", ["spread", "dropped", "none", "one"])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 256, 8), (3, 5, 2), (8, 1024, 64), (65, 60, 6), (257, 512, 10),
                                   (700, 3, 1), (5000, 256, 8), (40001, 1024, 3)])
def test_sort(gpu, T, E, k, kind):
    """Choices repeat experts within a token (drawn with replacement), from one pair to more than a block's turn."""
    print(f"moe_sort T={T} E={E} k={k} {kind}", flush=True)
    e = _choices(T + k, T, E, k, kind)
    for tile_m in (0, 32, -32):
        r = qwq4.moe_sort(to_dev(e, gpu), E, tile_m=tile_m)
        counts, offsets, slot, tok = ref.sort(e, E)
        assert np.array_equal(host(r.counts), counts)
        assert np.array_equal(host(r.offsets), offsets)
        assert np.array_equal(host(r.tok_slot), slot)
        assert np.array_equal(host(r.pair_tok), tok)
        n = int(host(r.n_active)[0])
        assert np.array_equal(host(r.active)[:n], np.nonzero(counts)[0])
        if tile_m:
            want = ref.tiles(counts, tile_m)
            assert int(host(r.n_tiles)[0]) == len(want)
            got = np.stack([host(r.tile_e), host(r.tile_m0)], 1)[:len(want)]
            assert np.array_equal(got, np.array(want).reshape(-1, 2))


def test_sort_is_the_routing_of_its_choices(gpu):
    import torch
    logits = torch.from_numpy(np.random.default_rng(5).standard_normal((333, 64)).astype(np.float32)).to(gpu)
    a = qwq4.moe_route(logits, 6, tile_m=-32)
    b = qwq4.moe_sort(a.top_e, 64, tile_m=-32)
    for name in ("counts", "offsets", "tok_slot", "pair_tok", "n_active", "n_tiles"):
        assert torch.equal(getattr(a, name), getattr(b, name)), name


def test_sort_into_a_route(gpu):
    import torch
    out = qwq4.Route(20, 16, 3, gpu, tile_m=-32)
    for seed in (1, 2):
        e = _choices(seed, 20, 16, 3, "dropped")
        assert qwq4.moe_sort(to_dev(e, gpu), 16, tile_m=-32, out=out) is out
        assert np.array_equal(host(out.tok_slot), ref.sort(e, 16)[2])


# ---------------------------------------------------------------- permute
@pytest.mark.parametrize("T,k,H,pad", [(1, 1, 1, 0), (1, 8, 4096, 0), (5, 3, 7, 1), (37, 10, 2560, 0), (64, 2, 130, 6),
                                       (301, 8, 1023, 0), (700, 1, 640, 8)])
@pytest.mark.parametrize("t", ["i8", "bf16", "f32"])
def test_permute(gpu, T, k, H, pad, t):
    """Rows of 1, 2 and 4 bytes an element at any stride; rows without a choice and the space between rows stay."""
    import torch
    print(f"moe_permute T={T} k={k} H={H} pad={pad} {t}", flush=True)
    r = np.random.default_rng(T)
    wide = torch.from_numpy(r.integers(-99, 100, (T, H + pad)).astype(np.int8)).to(gpu)
    wide = wide if t == "i8" else wide.to(_types()[t])
    x = wide[:, :H]
    e = _choices(T + H, T, 9, k, "dropped")
    _, offsets, slot, tok = ref.sort(e, 9)
    keep = int(GUARD)
    buf = torch.full((T * k, H + pad), keep, dtype=wide.dtype, device=gpu)
    qwq4.moe_permute(x, to_dev(slot.astype(np.int32), gpu), xs=buf[:, :H])
    got, n = host(buf).astype(np.float32), int(offsets[-1])
    assert np.array_equal(got[:n, :H], host(wide).astype(np.float32)[tok[:n], :H])
    assert (got[n:] == keep).all() and (got[:, H:] == keep).all()


def test_slots_outside_are_skipped(gpu):
    """Slots that no sort gives (beyond T*k) are not written to and not read."""
    import torch
    T, k, H = 4, 3, 96
    slot = np.array([[0, 12, 5], [11, -7, 2**31 - 1], [1, 2, 3], [-2**31, 100, 4]], np.int32)
    fine = (slot >= 0) & (slot < T * k)
    x, v = _floats(1, (T, H), "f32", gpu)
    xs = torch.full((T * k, H), GUARD, device=gpu)
    qwq4.moe_permute(x, to_dev(slot, gpu), xs=xs)
    want = np.full((T * k, H), GUARD)
    for t, i in zip(*np.nonzero(fine)):
        want[slot[t, i]] = v[t]
    assert np.array_equal(host(xs), want.astype(np.float32))
    out = host(qwq4.moe_unpermute(xs, to_dev(slot, gpu)))
    assert np.allclose(out, fine.sum(1)[:, None] * v, rtol=4 * 2.0**-24, atol=0)
    dyp = torch.full((T * k, H), GUARD, device=gpu)
    _, dw = qwq4.moe_unpermute_backward(x, xs, to_dev(slot, gpu), dyp=dyp)
    assert np.array_equal(host(dyp), want.astype(np.float32)) and (host(dw)[~fine] == 0).all()


# -------------------------------------------------------------- unpermute
SIZES = [(1, 1, 1, 0), (1, 8, 4096, 0), (2, 64, 48, 0), (5, 3, 7, 1), (37, 10, 2560, 0), (64, 2, 130, 6),
         (301, 8, 1023, 0), (530, 5, 264, 8)]


@pytest.mark.parametrize("T,k,H,pad", SIZES)
@pytest.mark.parametrize("yt,ot,weights", [("f32", "f32", True), ("bf16", "bf16", True), ("f16", "f32", False),
                                           ("f32", "f16", False), ("f16", "bf16", True)])
def test_unpermute(gpu, T, k, H, pad, yt, ot, weights):
    import torch
    print(f"moe_unpermute T={T} k={k} H={H} pad={pad} {yt} {ot} {weights}", flush=True)
    e = _choices(T + k, T, 11, k, "dropped")
    slot = ref.sort(e, 11)[2]
    yp, y = _floats(T, (T * k, H), yt, gpu, pad)
    w = np.random.default_rng(T).standard_normal((T, k)).astype(np.float32)
    buf = torch.full((T, H + pad), GUARD, dtype=_types()[ot], device=gpu)
    qwq4.moe_unpermute(yp, to_dev(slot.astype(np.int32), gpu), to_dev(w, gpu) if weights else None, out=buf[:, :H])
    got = host(buf).astype(np.float64)
    parts = np.where((slot >= 0)[..., None], y[np.maximum(slot, 0)], 0.0)
    parts = parts * w[..., None] if weights else parts
    want = parts.sum(1)
    # k products and k sums in fp32, each off by at most 2^-24 of the sum of magnitudes; then the output's rounding
    bound = 2 * k * 2.0**-24 * np.abs(parts).sum(1)
    bound += (np.abs(want) + bound) * HALF[ot] + SMALLEST[ot]
    assert np.all(np.abs(got[:, :H] - want) <= bound)
    assert (got[:, H:] == GUARD).all()


def test_unpermute_saturates_and_passes_nan(gpu):
    import torch
    yp = torch.full((4, 8), 60000.0, device=gpu)
    yp[2, 1], yp[3, 2] = float("inf"), float("nan")
    slot = torch.tensor([[0, 1], [2, -1], [-1, -1]], dtype=torch.int32, device=gpu)
    slot4 = torch.cat([slot[:2]])
    out = host(qwq4.moe_unpermute(yp, slot4, out_dtype=torch.float16)).astype(np.float32)
    assert (out[0] == 65504).all() and np.isinf(out[1, 1]) and (np.delete(out[1], 1) == 60000).all()
    # the row of slot 3 (a NaN) has no choice: it reaches nothing, not even with a weight of zero beside it
    assert not np.isnan(out).any()


def test_rows_without_slots_are_zero(gpu):
    import torch
    slot = torch.full((3, 4), -1, dtype=torch.int32, device=gpu)
    yp = torch.full((12, 33), float("nan"), dtype=torch.bfloat16, device=gpu)
    w = torch.full((3, 4), float("nan"), device=gpu)
    assert (host(qwq4.moe_unpermute(yp, slot, w)) == 0).all()
    dyp = torch.full((12, 33), GUARD, dtype=torch.bfloat16, device=gpu)
    _, dw = qwq4.moe_unpermute_backward(torch.ones(3, 33, device=gpu), yp, slot, w, dyp=dyp)
    assert (host(dw) == 0).all() and (host(dyp) == GUARD).all()


def test_unpermute_agrees_with_combine(gpu):
    import torch
    logits = torch.from_numpy(np.random.default_rng(6).standard_normal((70, 32)).astype(np.float32)).to(gpu)
    r = qwq4.moe_route(logits, 4)
    yp, y = _floats(7, (280, 512), "f32", gpu)
    a = host(qwq4.moe_combine(yp, r, 512, out_dtype=torch.float32)).astype(np.float64)
    b = host(qwq4.moe_unpermute(yp, r.tok_slot, r.top_w)).astype(np.float64)
    mags = (np.abs(y[host(r.tok_slot)]) * host(r.top_w)[..., None]).sum(1)
    assert np.all(np.abs(a - b) <= 2 * 8 * 2.0**-24 * mags)  # either is within 2 k 2^-24 of the sum


# --------------------------------------------------------------- gradients
@pytest.mark.parametrize("T,k,H,pad", SIZES)
@pytest.mark.parametrize("dt,yt,weights", [("f32", "f32", True), ("bf16", "bf16", True), ("f16", "f32", True),
                                           ("f32", "f16", False), ("bf16", "f16", True)])
def test_unpermute_backward(gpu, T, k, H, pad, dt, yt, weights):
    import torch
    print(f"moe_unpermute_backward T={T} k={k} H={H} pad={pad} {dt} {yt} {weights}", flush=True)
    e = _choices(T + k, T, 11, k, "dropped")
    _, offsets, slot, tok = ref.sort(e, 11)
    n = int(offsets[-1])
    yp, y = _floats(T, (T * k, H), yt, gpu, pad)
    dout, d = _floats(T + 1, (T, H), dt, gpu, pad)
    w = np.random.default_rng(T).standard_normal((T, k)).astype(np.float32)
    buf = torch.full((T * k, H + pad), GUARD, dtype=_types()[yt], device=gpu)
    _, dw = qwq4.moe_unpermute_backward(dout, yp, to_dev(slot.astype(np.int32), gpu), to_dev(w, gpu) if weights else None,
                                        dyp=buf[:, :H])
    got, dw = host(buf).astype(np.float32), host(dw).astype(np.float64)
    # one fp32 product and its rounding to the type: bit for bit
    want = np.full((T * k, H), GUARD, np.float32)
    t, i = np.nonzero(slot >= 0)
    rows = d[t].astype(np.float32) * (w[t, i][:, None] if weights else np.float32(1))
    want[slot[t, i]] = ref.ROUND[yt](rows)
    assert np.array_equal(got[:, :H], want) and (got[:, H:] == GUARD).all()
    # H products and H sums in any order: 2 H 2^-24 of the sum of magnitudes
    part = np.zeros((T, k, H))
    part[t, i] = y[slot[t, i]] * d[t]
    assert np.all(np.abs(dw - part.sum(-1)) <= 2 * H * 2.0**-24 * np.abs(part).sum(-1))
    assert (dw[slot < 0] == 0).all() and n == len(t)


@pytest.mark.parametrize("T,k,H", [(3, 2, 5), (40, 4, 96)])
def test_gradients_against_differences(gpu, T, k, H):
    """<dout, f(a + d) - f(a - d)> / 2 = <gradient, d> for each input of the two forwards: the functions are linear in
    each, so a difference of any size is exact but for roundings (values of magnitude about 1; every compared number is
    a sum of at most T k H = 15360 products whose own error is below 2 (k + 1) 2^-24 of its size)."""
    import torch
    r = np.random.default_rng(T)
    e = _choices(T, T, 6, k, "dropped")
    slot = to_dev(ref.sort(e, 6)[2].astype(np.int32), gpu)
    n = int((host(slot) >= 0).sum())
    new = lambda *s: torch.from_numpy(r.standard_normal(s).astype(np.float32)).to(gpu)  # noqa: E731
    yp, w, dout, x, dxs = new(T * k, H), new(T, k), new(T, H), new(T, H), new(T * k, H)
    dot = lambda a, b: float((a.double() * b.double()).sum())  # noqa: E731
    dyp = torch.zeros_like(yp)
    _, dw = qwq4.moe_unpermute_backward(dout, yp, slot, w, dyp=dyp)
    up = lambda y_, w_: qwq4.moe_unpermute(y_, slot, w_)  # noqa: E731
    # (the terms' magnitudes: at most 4 each, of products of three normals)
    bound = 2 * (k + 2) * 2.0**-24 * 64 * T * k * H
    d = new(T * k, H)
    assert abs(dot(dout, up(yp + d, w).double() - up(yp - d, w).double()) / 2 - dot(dyp, d)) <= bound
    d = new(T, k)
    assert abs(dot(dout, up(yp, w + d).double() - up(yp, w - d).double()) / 2 - dot(dw, d)) <= bound
    # permute: rows without a choice are not part of its output
    dx = qwq4.moe_permute_backward(dxs, slot)
    d = new(T, H)
    xs = lambda v: qwq4.moe_permute(v, slot)[:n].double()  # noqa: E731
    assert abs(dot(dxs[:n], xs(x + d) - xs(x - d)) / 2 - dot(dx, d)) <= bound


def test_backward_parts(gpu):
    """Either gradient alone gives the bits it has beside the other."""
    import torch
    T, k, H = 21, 4, 200
    slot = to_dev(ref.sort(_choices(1, T, 7, k, "dropped"), 7)[2].astype(np.int32), gpu)
    yp, _ = _floats(2, (T * k, H), "bf16", gpu)
    dout, _ = _floats(3, (T, H), "bf16", gpu)
    w = torch.rand(T, k, device=gpu)
    a, b = torch.zeros_like(yp), torch.zeros_like(yp)
    _, dw = qwq4.moe_unpermute_backward(dout, yp, slot, w, dyp=a)
    none, dw2 = qwq4.moe_unpermute_backward(dout, yp, slot, w, need_dyp=False)
    _, none2 = qwq4.moe_unpermute_backward(dout, yp, slot, w, dyp=b, need_dw=False)
    assert none is None and none2 is None and torch.equal(dw, dw2) and torch.equal(a, b)


def test_round_trip_and_graph(gpu):
    """sort -> permute -> unpermute -> both gradients as one step, captured and replayed between eager steps."""
    import torch
    T, E, k, H = 45, 12, 4, 320
    e = torch.empty((T, k), dtype=torch.int32, device=gpu)
    x, dout = torch.empty((T, H), dtype=torch.bfloat16, device=gpu), torch.empty((T, H), device=gpu)
    w = torch.empty((T, k), device=gpu)

    def step(e, x, w, dout):
        r = qwq4.moe_sort(e, E)
        xs = torch.zeros((T * k, H), dtype=torch.bfloat16, device=gpu)
        dyp = torch.zeros((T * k, H), dtype=torch.bfloat16, device=gpu)
        qwq4.moe_permute(x, r.tok_slot, xs=xs)
        out = qwq4.moe_unpermute(xs, r.tok_slot, w, out_dtype=torch.float32)
        _, dw = qwq4.moe_unpermute_backward(dout, xs, r.tok_slot, w, dyp=dyp)
        return xs, out, dyp, dw, qwq4.moe_permute_backward(dyp, r.tok_slot, dx_dtype=torch.float32)

    def fill(seed):
        g = np.random.default_rng(seed)
        e.copy_(torch.from_numpy(_choices(seed, T, E, k, "dropped" if seed % 2 else "spread")))
        x.copy_(torch.from_numpy(g.standard_normal((T, H)).astype(np.float32)))
        dout.copy_(torch.from_numpy(g.standard_normal((T, H)).astype(np.float32)))
        w.copy_(torch.from_numpy(g.random((T, k)).astype(np.float32)))

    fill(0)
    step(e, x, w, dout)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(e, x, w, dout)
    for seed in (1, 2, 3, 4):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in captured]
        eager = step(e.clone(), x.clone(), w.clone(), dout.clone())
        torch.cuda.synchronize()
        for a, b in zip(got, eager):
            assert torch.equal(a, b)


def test_offsets_past_32_bits(gpu):
    """More than 2^31 elements in the sorted rows: the last ones are where they belong, there and back."""
    import torch
    T, k, H = 66000, 8, 4100
    e = torch.from_numpy(np.random.default_rng(9).integers(0, 64, (T, k)).astype(np.int32)).to(gpu)
    r = qwq4.moe_sort(e, 64)
    x = torch.randint(-99, 100, (T, H), dtype=torch.int8, device=gpu).to(torch.float16)
    xs = qwq4.moe_permute(x, r.tok_slot)
    at = torch.tensor([0, 1, 523770, 523777, T * k - 2, T * k - 1], device=gpu)
    assert torch.equal(xs[at], x[r.pair_tok[at].long()])
    out = qwq4.moe_unpermute(xs, r.tok_slot)
    assert torch.equal(out[-300:], x[-300:] * k)  # (sums of small whole numbers: exact)
    dyp, dw = qwq4.moe_unpermute_backward(x, xs, r.tok_slot)
    assert torch.equal(dyp[at], xs[at])
    assert torch.equal(dw[-3:], (x[-3:].float() ** 2).sum(1)[:, None].expand(3, k))


# fp16 beside and beyond its largest value 65504: 65519.996 rounds down to it, 65520 is the tie that rounds to infinity
EDGE = [65504.0, 65519.996, 65520.0, -65520.0, 70000.0, -1e6, 3.0, float("inf")]


@pytest.mark.parametrize("pad", [0, 1])
def test_fp16_gradients_overflow(gpu, pad):
    """Gradients that fp16 cannot hold are infinite, as a plain rounding makes them (a loss scaler looks for those);
    the forward saturates. Whole 16-byte pieces, and one element at a time."""
    import torch
    H = len(EDGE)
    d = torch.zeros(2, H + pad, device=gpu)[:, :H]
    d[0], d[1] = torch.tensor(EDGE, device=gpu), 30000.0
    slot = torch.tensor([[0, 2], [1, 3]], dtype=torch.int32, device=gpu)
    w = torch.tensor([[1.0, 2.0], [2.0, 3.0]], device=gpu)
    yp = torch.ones(4, H + pad, dtype=torch.float16, device=gpu)[:, :H]
    dyp, _ = qwq4.moe_unpermute_backward(d, yp, slot, w)
    with np.errstate(over="ignore"):
        want = np.stack([host(d[0]), 2 * host(d[1]), 2 * host(d[0]), 3 * host(d[1])]).astype(np.float16)
        want_dx = np.stack([host(d[0]), 2 * host(d[1])]).astype(np.float16)
    assert np.array_equal(host(dyp), want)
    assert np.isinf(want).any() and (want[3] == np.inf).all()
    # its other choice's row is of zeros: the sum is the edge itself
    dxs = torch.zeros(4, H + pad, device=gpu)[:, :H]
    dxs[0], dxs[1], dxs[3] = d[0], d[1], d[1]
    dx = torch.full((2, H + pad), GUARD, dtype=torch.float16, device=gpu)[:, :H]
    assert np.array_equal(host(qwq4.moe_permute_backward(dxs, slot, dx=dx)), want_dx)
    half = torch.full((4, H), 40000.0, dtype=torch.float16, device=gpu)  # (a sum of two: 80000)
    assert (host(qwq4.moe_permute_backward(half, slot)) == np.inf).all()
    assert (host(qwq4.moe_unpermute(half, slot)) == 65504).all()


@pytest.mark.parametrize("t", ["i8", "u16", "e4m3", "bf16", "f32"])
def test_new_rows_are_defined(gpu, t):
    """Sorted rows and dyp that a call allocates are zero where no choice has a slot (a product over all of them, such as
    an expert's weight gradient, must not meet what the memory held before)."""
    import torch
    T, k, H = 96, 4, 512
    dtype = {"i8": torch.int8, "u16": torch.uint16, "e4m3": torch.float8_e4m3fn, "bf16": torch.bfloat16,
             "f32": torch.float32}[t]
    e = _choices(17, T, 9, k, "dropped")
    _, offsets, slot, tok = ref.sort(e, 9)
    n, slots = int(offsets[-1]), to_dev(slot.astype(np.int32), gpu)
    assert 0 < n < T * k
    x = torch.from_numpy(np.random.default_rng(18).integers(1, 99, (T, H)).astype(np.int8)).to(gpu)
    x = x.repeat(1, dtype.itemsize).view(dtype)

    def used():  # the allocator's block that the call below takes, full of ones (a NaN in any float type)
        block = torch.full((T * k, H * dtype.itemsize), 255, dtype=torch.uint8, device=gpu)
        torch.cuda.synchronize()
        return block.data_ptr()
    torch.cuda.empty_cache()
    at = used()
    xs = qwq4.moe_permute(x, slots)
    print(f"moe_permute {t}: block taken again: {at == xs.data_ptr()}", flush=True)
    bits = host(xs.view(torch.uint8))
    assert np.array_equal(bits[:n], host(x.view(torch.uint8))[tok[:n]]) and (bits[n:] == 0).all()
    if t not in ("bf16", "f32"):
        return
    yp, dout = torch.ones(T * k, H, dtype=dtype, device=gpu), torch.ones(T, H, device=gpu)
    del xs
    used()
    dyp, _ = qwq4.moe_unpermute_backward(dout, yp, slots)
    assert (host(dyp)[:n] == 1).all() and (host(dyp)[n:] == 0).all()


@pytest.mark.parametrize("T,k,H", [(1, 1, 8), (37, 4, 96), (130, 8, 257)])
def test_functions_of_the_guide(gpu, T, k, H):
    """The integration guide's autograd Functions around a user's own expert (a product per column): they run, and
    their gradients are the formula's."""
    import os
    import re

    import torch
    guide = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "INTEGRATION.md")).read()
    code, = (b for b in re.findall(r"```python\n(.*?)```", guide, flags=re.S) if "class Unpermute" in b)
    names = {"torch": torch, "qwq4": qwq4}
    exec(code, names)
    r = np.random.default_rng(T)
    slot = ref.sort(_choices(T + k, T, 7, k, "dropped" if T > 1 else "spread"), 7)[2]
    x, w, a, m = (r.standard_normal(s).astype(np.float32) for s in ((T, H), (T, k), (H,), (T, H)))
    leaf = [torch.from_numpy(v).to(gpu).requires_grad_() for v in (x, w)]
    s = to_dev(slot.astype(np.int32), gpu)
    out = names["Unpermute"].apply(names["Permute"].apply(leaf[0], s) * to_dev(a, gpu), s, leaf[1])
    (out * to_dev(m, gpu)).sum().backward()
    x, w, a, m = (v.astype(np.float64) for v in (x, w, a, m))
    kept = slot >= 0
    each = np.where(kept[..., None], (w[..., None] * m[:, None]) * a, 0.0)
    # w m, its product with a, and k sums: k + 2 roundings of 2^-24 of the sum of magnitudes
    assert np.all(np.abs(host(leaf[0].grad) - each.sum(1)) <= (k + 2) * 2.0**-24 * np.abs(each).sum(1))
    # x a, H products and H sums
    part = np.where(kept[..., None], ((x * a) * m)[:, None], 0.0)
    assert np.all(np.abs(host(leaf[1].grad) - part.sum(-1)) <= (2 * H + 1) * 2.0**-24 * np.abs(part).sum(-1))
    only, = torch.autograd.grad(names["Unpermute"].apply(torch.ones(T * k, H, device=gpu), s, leaf[1]).sum(), leaf[1])
    assert np.array_equal(host(only), np.where(kept, H, 0).astype(np.float32))
