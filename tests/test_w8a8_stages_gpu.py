"""The W8A8 products over many stages of K: the steady turns of every tile's
main loop, in which each buffer is used again and again, with even, odd and
ragged numbers of stages. Sums are of whole numbers: compared bit for bit."""
import numpy as np
import pytest

import qwq4
import test_w8a8_gpu as base
import _w8a8_ref as ref
from _gpu_util import to_dev

pytestmark = pytest.mark.gpu


def _choices(seed, T, E, k, kind):
    """k different experts per token: all alike, the last of them always, or with loads that fall by half from one
    expert to the next."""
    r = np.random.default_rng(seed)
    v = r.gumbel(size=(T, E))
    if kind == "one":
        v[:, E - 1] += 1e6
    elif kind == "uneven":
        v -= np.log(2) * np.arange(E)
    elif kind != "spread":
        raise ValueError(kind)
    return np.argsort(-v, axis=1)[:, :k].astype(np.int32)


@pytest.fixture
def check_experts(monkeypatch):
    monkeypatch.setattr(base, "_choices", _choices)
    return base._check_experts


# stages of 128: 9 and 17 (the last of 16 columns), 10, 32
@pytest.mark.parametrize("K", [1040, 1280, 2064, 4096])
@pytest.mark.parametrize("T,N", [(300, 25000), (100, 20000), (60, 9000)])
def test_dense_tiles(gpu, T, N, K):
    """Tiles of 256, 128 and 64 rows."""
    print(f"gemm_w8a8 T={T} N={N} K={K}", flush=True)
    Wd, swd, W, sw = base._weights(201, N, K, gpu)
    r = np.random.default_rng(202)
    q, sx = r.integers(-128, 128, (T, K), dtype=np.int8), (r.random(T) + 0.5).astype(np.float32)
    want = ref.product(q, sx, W, sw)
    for t in ("bf16", "f32"):
        y = qwq4.gemm_w8a8(Wd, swd, to_dev(q, gpu), to_dev(sx, gpu), y_dtype=base._types()[t])
        base._same(y, ref.ROUND[t](want))


@pytest.mark.parametrize("kind", ["spread", "one", "uneven"])
@pytest.mark.parametrize("H,F,xt,yt", [(1296, 912, "bf16", "f32"), (2048, 768, "f16", "bf16"),
                                       (784, 1040, "f32", "f16")])
def test_tall_expert_tiles(gpu, check_experts, H, F, xt, yt, kind):
    """More than 24 slots an expert: 128 and 64 slots a tile in three buffers, both products over 6 to 16 stages."""
    print(f"experts_w8a8 H={H} F={F} {kind}", flush=True)
    check_experts(gpu, 300, 4, 2, H, F, xt, yt, kind, seed=211)


@pytest.mark.parametrize("kind", ["spread", "one", "uneven"])
@pytest.mark.parametrize("H,F", [(1296, 912), (1024, 1168)])
def test_low_expert_tiles(gpu, check_experts, H, F, kind):
    """Up to 24 slots an expert: 64 slots a tile in two buffers, 8 to 11 stages."""
    print(f"experts_w8a8 H={H} F={F} {kind}", flush=True)
    check_experts(gpu, 100, 16, 2, H, F, "bf16", "bf16", kind, seed=221)


@pytest.mark.parametrize("T", [4, 5, 9, 16, 17])
def test_uneven_loads_of_few_tokens(gpu, check_experts, T):
    """Streamed and tiled experts of which one has nearly all slots."""
    print(f"experts_w8a8 T={T}", flush=True)
    check_experts(gpu, T, 6, 2, 2048, 2032, "bf16", "f16", "uneven", seed=231)


@pytest.mark.parametrize("T,K", [(2, 32752), (2, 32784), (1, 65520)])
def test_longest_staged_rows(gpu, T, K):
    """Around the longest rows that one and two tokens stage whole."""
    Wd, swd, W, sw = base._weights(241, 40, K, gpu)
    x, v = base._rows(242, T, K, "bf16", gpu)
    base._same(qwq4.linear_w8a8(Wd, swd, x), ref.bf16(ref.product(*ref.quant(v), W, sw)))
