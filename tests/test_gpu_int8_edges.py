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
