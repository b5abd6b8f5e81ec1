"""An MoE layer of W8A8 experts as a model runs it, over choices that another
router made: sorted, multiplied, and combined with a shared expert's rows."""
import numpy as np
import pytest

import qwq4
import test_w8a8_gpu as base
import _w8a8_ref as ref
from _gpu_util import host, to_dev

pytestmark = pytest.mark.gpu

HALF = {"f32": 2.0**-24, "bf16": 2.0**-8, "f16": 2.0**-11}  # half a step, relative
SMALLEST = {"f32": 2.0**-150, "bf16": 2.0**-134, "f16": 2.0**-25}


@pytest.mark.parametrize("kind", ["spread", "dropped", "repeated"])
@pytest.mark.parametrize("yt,st,ot", [("f32", "f32", "bf16"), ("f16", "f16", "f16"), ("f16", None, "f32")])
@pytest.mark.parametrize("T", [1, 2, 9, 130])
def test_combined_with_the_shared_expert(gpu, T, yt, st, ot, kind):
    import torch
    print(f"layer T={T} {yt} {st} {ot} {kind}", flush=True)
    E, k, H, F = 12, 4, 272, 144
    types = base._types()
    (g, u, d), _ = base._experts(301, E, H, F, gpu)
    x, _ = base._rows(302, T, H, "bf16", gpu)
    e = base._choices(303, T, E, k, kind)
    w = np.random.default_rng(304).random((T, k)).astype(np.float32)
    shared = None if st is None else base._rows(305, T, H, st, gpu)[0].contiguous()
    r = qwq4.moe_sort(to_dev(e, gpu), E, tile_m=qwq4.moe_w8a8_tile_m())
    yp = qwq4.moe_experts_w8a8(g, u, d, r, x, yp_dtype=types[yt])[1]
    out = qwq4.moe_combine(yp, r, H, shared=shared, out_dtype=types[ot], tok_w=to_dev(w, gpu))
    slot = ref.sort(e, E)[2]
    y = host(yp).astype(np.float64)[np.maximum(slot, 0)] * w[..., None]
    y = np.where((slot >= 0)[..., None], y, 0.0)
    sh = np.zeros((T, H)) if shared is None else host(shared).astype(np.float64)
    want = sh + y.sum(1)
    # k products and k sums in fp32, each off by at most 2^-24 of the sum of magnitudes; then the output's rounding
    bound = 2 * k * 2.0**-24 * (np.abs(sh) + np.abs(y).sum(1))
    bound += (np.abs(want) + bound) * HALF[ot] + SMALLEST[ot]
    assert np.all(np.abs(host(out).astype(np.float64) - want) <= bound)
    # without a shared expert the same rows by the other call, within either's bound
    if shared is None:
        again = host(qwq4.moe_unpermute(yp, r.tok_slot, to_dev(w, gpu), out_dtype=torch.float32)).astype(np.float64)
        assert np.all(np.abs(again - want) <= bound)


def test_a_route_used_in_turn(gpu):
    """One Route for a router's choices and for given ones in turn: each call's lists and weights are its own, and a
    sort of what the router chose with some taken out leaves the tensors it was given alone."""
    import torch
    T, E, k = 70, 16, 4
    logits = torch.from_numpy(np.random.default_rng(311).standard_normal((T, E)).astype(np.float32)).to(gpu)
    want = qwq4.moe_route(logits, k)
    r = qwq4.Route(T, E, k, gpu)
    given = torch.where(want.top_e % 2 == 0, want.top_e, torch.full_like(want.top_e, -1))
    kept = given.clone()
    for _ in range(2):
        assert qwq4.moe_sort(given, E, out=r) is r
        assert np.array_equal(host(r.tok_slot), ref.sort(host(kept), E)[2])
        qwq4.moe_route(logits, k, out=r)
        for name in ("top_e", "top_w", "offsets", "tok_slot", "pair_tok"):
            assert torch.equal(getattr(r, name), getattr(want, name)), name
        assert torch.equal(given, kept)
