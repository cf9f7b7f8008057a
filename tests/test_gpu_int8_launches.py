"""8-bit rows and products behind other launches of the library: what those write is read when it is there."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _kernels():
    from geneinfer_b200.ops import kernels
    return kernels


@pytest.mark.parametrize("D", [100, 2048, 8192, 9001, 16384, 40001])
def test_a_norms_weights_of_the_launch_before(D):
    k = _kernels()
    g = torch.Generator().manual_seed(D)
    left, right = torch.randn(D, 4096, generator=g).to(DEV), torch.randn(1, 4096, generator=g).to(DEV)
    x = torch.randn(5, D, generator=g).to(DEV)
    weight, q, scales = torch.empty(D, 1, device=DEV), torch.empty(5, k.int8_width(D), dtype=torch.int8, device=DEV), torch.empty(5, device=DEV)

    def run(wait):
        weight.zero_()
        torch.cuda.synchronize()
        k.gemm_simt(left, right, weight)
        if wait:
            torch.cuda.synchronize()
        k.rmsnorm_int8(x, weight.view(-1), q, scales, 1e-5)
        return q.clone(), scales.clone()

    want = run(True)
    assert (want[1] > 0).all()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(False), want))


@pytest.mark.parametrize("T", [3, 40, 100, 900])
@pytest.mark.parametrize("gated", [False, True])
def test_a_products_weights_of_the_launch_before(T, gated):
    """Tiles that a launch of rows in 8 bits writes (the integers of rows whose largest is 127 are the rows themselves)."""
    k = _kernels()
    g = torch.Generator(device=DEV).manual_seed(T)
    K, N = 4096, 2048
    w = k.int8_weight(torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8), torch.rand(N, generator=g, device=DEV) / 1000, gated=gated)
    assert w.constant
    whole = w.tiles.view(-1, 4096).float()
    whole[:, 0] = 127
    w = k.Int8Weight(w.tiles, w.scales, w.channels, w.width, gated)
    assert not w.constant
    a, s = torch.randint(-127, 128, (T, K), generator=g, device=DEV, dtype=torch.int8), torch.rand(T, generator=g, device=DEV) / 1000
    unused = torch.empty(whole.shape[0], device=DEV)
    h, hs = torch.empty(T, k.int8_width(w.channels), dtype=torch.int8, device=DEV), torch.empty(T, device=DEV)
    work, out = torch.empty(k.int8_gated_work(T, w), device=DEV), torch.empty(T, w.channels, device=DEV)

    def run(wait):
        w.tiles.zero_()
        torch.cuda.synchronize()
        k.quantize_rows(whole, w.tiles.view(-1, 4096), unused)
        if wait:
            torch.cuda.synchronize()
        if gated:
            k.int8_gated(a, s, w, h, hs, work)
            return h.clone(), hs.clone()
        k.int8_product(a, s, w, out)
        return (out.clone(),)

    want = run(True)
    assert torch.equal(w.tiles.view(-1, 4096).float(), whole) and all((t != 0).any() for t in want)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(run(False), want))
