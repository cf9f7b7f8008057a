"""8-bit rows and products at the ends of their ranges: plans, bounds, values near the ends of 32 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _kernels():
    from geneinfer_b200.ops import kernels
    return kernels


def _product(k, g, T, K, N):
    """A weight, rows, and the product by the roundings of the definition."""
    q, ws = torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8), 0.01 + torch.rand(N, generator=g, device=DEV)
    a = torch.zeros(T, k.int8_width(K), dtype=torch.int8, device=DEV)
    a[:, :K] = torch.randint(-127, 128, (T, K), generator=g, device=DEV, dtype=torch.int8)
    s = 0.01 + torch.rand(T, generator=g, device=DEV)
    return k.int8_weight(q, ws), a, s, ((a[:, :K].double() @ q.double().T).float() * s[:, None]) * ws


def test_more_tiles_walked_together_than_there_are():
    k = _kernels()
    w, a, s, want = _product(k, torch.Generator(device=DEV).manual_seed(1), 700, 200, 1000)
    for group in (4, 1000, 2 ** 30, 2 ** 31 - 1):
        out = torch.full((700, 1000), math.nan, device=DEV)
        k.int8_product(a, s, w, out, plan=("many", group))
        assert torch.equal(out, want), group


@pytest.mark.parametrize("D", [300, 2048, 9001, 16384, 33000])
def test_norms_with_weights_near_the_ends_of_32_bits(D):
    """Ordinary rows whose products with the weights overflow, small rows without an eps with weights as large, large rows with small weights: a norm's squares and
    its products with the weights leave the range each by itself."""
    k = _kernels()
    g = torch.Generator(device=DEV).manual_seed(D)
    for size, weight, eps in ((3.0, 1.5e38, 1e-5), (3.0, 1.5e38, 0.0), (1e-20, 1e36, 0.0), (1e-24, 1e-12, 0.0), (1e-20, 1.0, 0.0), (1e25, 1e-30, 1e-5), (1e25, 1.0, 1e-5), (1e25, 1e20, 1e-5)):
        x = torch.randn(3, D, generator=g, device=DEV) * size
        x[1] = 0
        w = (0.5 + 0.5 * torch.rand(D, generator=g, device=DEV)) * weight
        more = torch.zeros_like(x)
        q, s = torch.empty(3, k.int8_width(D), dtype=torch.int8, device=DEV), torch.empty(3, device=DEV)
        k.rmsnorm_int8(x, w, q, s, eps, add=more)
        assert float(s[1]) == 0 and not q[1].any()
        for row in (0, 2):
            want = x[row].double() / (x[row].double().square().mean() + eps).sqrt() * w.double()
            got = q[row, :D].double() * s[row].double()
            # half a step of the integers and, far below it, the 32-bit scale's and borders' roundings (a scale below 2^-126 has steps of 2^-149)
            assert float((got - want).abs().max()) <= float(want.abs().max()) / 127 * 0.501, (size, weight, eps, row)


@pytest.mark.parametrize("T", [8, 400])
def test_additions_of_values_below_the_least_normal_one(T):
    """What a product is added to, the product and the sum may be subnormal: kept by every form, so that a row's result does not depend on the others in the call."""
    k = _kernels()
    g = torch.Generator(device=DEV).manual_seed(T)
    for N in (256, 257, 130):
        _, a, s, _ = _product(k, g, T, 64, N)
        s *= 2.0 ** -15
        q = torch.randint(-127, 128, (N, 64), generator=g, device=DEV, dtype=torch.int8)
        w = k.int8_weight(q, (0.01 + torch.rand(N, generator=g, device=DEV)) * 2.0 ** -120)
        want = ((a.double() @ q.double().T).float() * s[:, None]) * w.scales
        assert float(((want != 0) & (want.abs() < 2.0 ** -126)).float().mean()) > 0.05
        for base in (torch.zeros_like(want), torch.randn(T, N, generator=g, device=DEV) * 2.0 ** -130, -want, want * 0.75):
            for plan in (None, ("few", 8, 1, 0), ("many", 1), ("many", 2)):
                for room in (0, 3):
                    out = torch.full((T, N + room), 7.0, device=DEV)
                    out[:, :N] = base
                    k.int8_product(a, s, w, out[:, :N], accumulate=True, plan=plan)
                    assert torch.equal(out[:, :N], base + want) and (out[:, N:] == 7).all(), (N, plan, room)


@pytest.mark.parametrize("activation", ["silu", "relu", "gelu_tanh", "capped_swish"])
@pytest.mark.parametrize("T,K,I", [(2048, 512, 1024), (1500, 130, 4099), (700, 777, 8200)])
def test_activated_rows_of_few_and_of_many_are_the_same(T, K, I, activation):
    """With few rows the products go through memory in 32 bits, with many the activation is the product's epilogue: the same integers and scales, to the bit."""
    k = _kernels()
    g = torch.Generator(device=DEV).manual_seed(T + I)
    q, ws = torch.randint(-127, 128, (2 * I, K), generator=g, device=DEV, dtype=torch.int8), (0.01 + torch.rand(2 * I, generator=g, device=DEV)) / (4900 * math.sqrt(K))
    w = k.int8_weight(q, ws, gated=True)
    _, a, s, _ = _product(k, g, T, K, 1)
    for bias in (None, 0.2 * torch.randn(2 * I, generator=g, device=DEV)):
        got = []
        for n in (T, 60, 1):
            out, scales = torch.full((n, k.int8_width(I)), 77, dtype=torch.int8, device=DEV), torch.full((n,), -1.0, device=DEV)
            k.int8_gated(a[:n], s[:n], w, out, scales, torch.empty(k.int8_gated_work(n, w), device=DEV), activation, 2.0, bias)
            got.append((out, scales))
            assert k._int8_plan(n, w)[0] == ("many" if n == T else "few")
        for out, scales in got[1:]:
            n = scales.numel()
            assert torch.equal(out, got[0][0][:n]) and torch.equal(scales, got[0][1][:n])


@pytest.mark.parametrize("D", [300, 9001, 33000])
def test_small_norms_with_small_weights(D):
    """Rows without an eps whose products with the weights vanish in 32 bits altogether, though the normed values do not."""
    k = _kernels()
    g = torch.Generator(device=DEV).manual_seed(D)
    x = torch.randn(2, D, generator=g, device=DEV) * 1e-30
    x[1] = 0
    w = (0.5 + 0.5 * torch.rand(D, generator=g, device=DEV)) * 1e-20
    assert not (x * w).any()
    q, s = torch.empty(2, k.int8_width(D), dtype=torch.int8, device=DEV), torch.empty(2, device=DEV)
    k.rmsnorm_int8(x, w, q, s, 0.0)
    want = x[0].double() / x[0].double().square().mean().sqrt() * w.double()
    assert float((q[0, :D].double() * s[0].double() - want).abs().max()) <= float(want.abs().max()) / 127 * 0.501
    assert float(s[1]) == 0 and not q[1].any()
