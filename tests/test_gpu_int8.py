"""Rows and products in 8-bit integers against plain 64-bit arithmetic of the same definitions."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
EPS = 1e-5


def _kernels():
    from geneinfer_b200.ops import kernels
    return kernels


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _ints(v):
    """q and the largest |v| of every row of 32-bit rows, by the three operations of the definition."""
    m = v.abs().amax(1, keepdim=True)
    small = m < 2.0 ** -100
    q = torch.round(v * (torch.full_like(m, 127.0) / torch.where(small, 1.0, m)))      # (127.0 / tensor is a reciprocal and a product: two roundings)
    return torch.where(small, 0.0, q).to(torch.int8), torch.where(small, 0.0, m)[:, 0]


def _buffers(kernels, T, D):
    width = kernels.int8_width(D)
    return torch.full((T, width), 77, dtype=torch.int8, device=DEV), torch.full((T,), -1.0, device=DEV)


def _check_rows(q, scales, want_q, want_scales, D):
    """Integers equal (their three operations are exact in IEEE arithmetic), zeros behind; scales to 8 roundings of 2^-24."""
    assert torch.equal(q[:, :D], want_q)
    assert not q[:, D:].any()
    assert torch.allclose(scales.double(), want_scales, rtol=8 * 2.0 ** -24, atol=0)


WIDTHS = [1, 3, 8, 16, 20, 127, 512, 513, 1000, 2048, 2050, 4096, 4100, 5000, 8192, 9001, 16384, 20480, 32768, 40001]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", WIDTHS)
def test_rows(D, dtype):
    k = _kernels()
    for T in (1, 7, 130):
        x = (_normal(_gen(D + T), T, D) * 3).to(dtype)
        x[T // 2] = 0                                   # a row of zeros
        q, s = _buffers(k, T, D)
        k.quantize_rows(x, q, s)
        want, m = _ints(x.float())
        _check_rows(q, s, want, m.double() / 127, D)


def test_rows_that_lie_apart():
    k = _kernels()
    for D, ld, offset in ((512, 1024, 0), (100, 233, 0), (64, 200, 3), (4096, 4100, 4)):
        wide = _normal(_gen(D), 9, ld)
        for x in (wide[:, offset:offset + D], wide.to(torch.bfloat16)[:, offset:offset + D]):
            q, s = _buffers(k, 9, D)
            k.quantize_rows(x, q, s)
            want, m = _ints(x.float())
            _check_rows(q, s, want, m.double() / 127, D)


def test_normed_and_activated_rows_that_lie_apart():
    k = _kernels()
    for D, ld in ((256, 260), (100, 333), (2048, 4096)):
        g = _gen(D)
        wide, w, more = _normal(g, 6, ld), torch.ones(D, device=DEV), _normal(g, 6, D)
        keep, after = wide[:, D:].clone(), wide[:, :D] + more
        q, s = _buffers(k, 6, D)
        k.rmsnorm_int8(wide[:, :D], w, q, s, EPS, add=more)
        assert torch.equal(wide[:, :D], after) and torch.equal(wide[:, D:], keep)
        assert torch.equal(q[:, :D], _ints(after)[0]) and not q[:, D:].any()
        both = _normal(g, 6, 2 * ld)[:, 3:3 + 2 * D]
        k.gated_act_int8(both, q, s, "relu")
        _near_ints(q, s, _act64(both[:, :D], both[:, D:], "relu", 0.0), 2 * 2.0 ** -9 + 2.0 ** -18)


@pytest.mark.parametrize("add", [None, torch.float32, torch.bfloat16])
@pytest.mark.parametrize("D", WIDTHS)
def test_normed_rows(D, add):
    k = _kernels()
    g = _gen(D)
    for T in (1, 9, 133):
        x, w = _normal(g, T, D) * 2, 0.5 + torch.rand(D, generator=g, device=DEV)
        x[0] *= 1e-4
        more = None if add is None else _normal(g, T, D).to(add)
        after = x if add is None else x + more.float()
        q, s = _buffers(k, T, D)
        k.rmsnorm_int8(x, w, q, s, EPS, add=more)
        assert torch.equal(x, after)
        want, m = _ints(after * w)
        mean = after.double().square().mean(1)
        # the squares' sum: all of one sign, each rounded, in chains and trees of at most D / 32 + 20 additions
        want_s = m.double() / 127 / (mean + EPS).sqrt()
        assert torch.equal(q[:, :D], want) and not q[:, D:].any()
        assert torch.allclose(s.double(), want_s, rtol=(D / 32 + 30) * 2.0 ** -24, atol=0)


def test_normed_rows_of_extreme_values():
    """Squares and products with the weights beyond 32 bits' range, rows of zeros, infinities and NaN."""
    k = _kernels()
    for D in (300, 2048, 33000):
        g = _gen(D)
        x, w = _normal(g, 8, D), 0.5 + torch.rand(D, generator=g, device=DEV)
        x[0] *= 1e25                     # the squares overflow
        x[1] *= 1e-30                    # the squares vanish
        x[2] = 0
        x[3, D // 2] = math.inf
        x[4, D - 1] = math.nan
        x[5] = x[5].clamp(-1, 1) * 3e38  # the products with the weights overflow
        x[6] *= 2.0 ** -120              # counts as zero
        more = torch.zeros_like(x)
        q, s = _buffers(k, 8, D)
        k.rmsnorm_int8(x, w, q, s, EPS, add=more)
        for row in (3, 4):
            assert math.isnan(float(s[row])) and not q[row].any()
        for row in (2, 6):
            assert float(s[row]) == 0 and not q[row].any()
        for row in (0, 1, 5, 7):
            v = x[row].double() * w.double()
            want = v / (x[row].double().square().mean() + EPS).sqrt()
            got = q[row, :D].double() * s[row].double()
            # half a step of the integers, and the borders' roundings
            assert float((got - want).abs().max()) <= float(want.abs().max()) / 127 * 0.5001, row


def test_normed_rows_without_an_eps():
    """Rows whose squares vanish in 32 bits, with nothing beside them under the root."""
    k = _kernels()
    for D in (64, 2048, 33000):
        g = _gen(D)
        w = 0.5 + torch.rand(D, generator=g, device=DEV)
        for eps in (0.0, 1e-38):
            x = _normal(g, 4, D) * torch.tensor([[1.0], [1e-18], [1e-24], [0.0]], device=DEV)
            q, s = _buffers(k, 4, D)
            k.rmsnorm_int8(x, w, q, s, eps)
            for row in range(3):
                want = x[row].double() * w.double() / (x[row].double().square().mean() + eps).sqrt()
                got = q[row, :D].double() * s[row].double()
                assert float((got - want).abs().max()) <= float(want.abs().max()) / 127 * 0.501, (D, eps, row)
            assert float(s[3]) == 0 and not q[3].any()


def test_rows_of_extreme_values():
    k = _kernels()
    for dtype in (torch.float32, torch.bfloat16):
        x = _normal(_gen(1), 6, 777).to(dtype)
        x[0, 5], x[1, 776], x[2, 0] = math.inf, -math.inf, math.nan
        x[3] = 0
        x[4] *= 2.0 ** -110
        x[5] = x[5].clamp(-1, 1) * 3e38
        q, s = _buffers(k, 6, 777)
        k.quantize_rows(x, q, s)
        assert torch.isnan(s[:3]).all() and not q[:5].any() and (s[3:5] == 0).all()
        want, m = _ints(x[5:].float())
        _check_rows(q[5:], s[5:], want, m.double() / 127, 777)


def _act64(g, u, activation, limit):
    g, u = g.double(), u.double()
    if activation == "relu":
        return g.clamp(min=0) * u
    if activation == "gelu_tanh":
        return 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))) * u
    if activation == "capped_swish":
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
        return g * torch.sigmoid(1.702 * g) * (u + 1)
    return g * torch.sigmoid(g) * u


def _near_ints(q, s, h, slack):
    """q * s against h: half a step of the integers, and ``slack`` of the largest value (what is rounded ahead of them)."""
    m = h.abs().amax(1, keepdim=True)
    got = q.double()[:, :h.shape[1]] * s.double()[:, None]
    assert float(((got - h).abs() - m * (0.5 / 127 + slack)).max()) <= 0
    assert not q[:, h.shape[1]:].any()


@pytest.mark.parametrize("activation", ["silu", "relu", "gelu_tanh", "capped_swish"])
@pytest.mark.parametrize("I", [1, 5, 48, 512, 1027, 2048, 4096, 8192, 14336, 28672, 33001])
def test_activated_rows(I, activation):
    k = _kernels()
    g = _gen(I)
    for T, dtype, biased in ((1, torch.float32, False), (5, torch.bfloat16, True), (37, torch.float32, True)):
        x = (_normal(g, T, 2 * I) * 2).to(dtype)
        x[T // 2, :I] = 0
        bias = _normal(g, 2 * I) * 0.5 if biased else None
        both = x.float() if bias is None else x.float() + bias
        q, s = _buffers(k, T, I)
        k.gated_act_int8(x, q, s, activation, 3.0, bias)
        h = _act64(both[:, :I], both[:, I:], activation, 3.0)
        # h is rounded to bfloat16: half a step 2^-9 of a value up to the largest, twice (its own, and the scale's), and the activation's 32 bits
        _near_ints(q, s, h, 2 * 2.0 ** -9 + 2.0 ** -18)


def test_activated_rows_of_extreme_values():
    k = _kernels()
    x = _normal(_gen(3), 4, 2 * 640)
    x[0, 3], x[1, 640 + 3], x[2] = math.nan, math.inf, 0
    q, s = _buffers(k, 4, 640)
    k.gated_act_int8(x, q, s, "silu")
    assert torch.isnan(s[:2]).all() and not q[:3].any() and float(s[2]) == 0 and float(s[3]) > 0
    for activation in ("silu", "relu", "gelu_tanh", "capped_swish"):      # a NaN in either half, and none is lost to a bound
        for at in (9, 640 + 9):
            x = _normal(_gen(4), 2, 2 * 640)
            x[0, at] = math.nan
            k.gated_act_int8(x, q[:2], s[:2], activation, 2.0)
            assert math.isnan(float(s[0])) and not q[0].any() and float(s[1]) > 0, (activation, at)


def _weight(g, N, K):
    q = torch.randint(-127, 128, (N, K), generator=g, device=DEV, dtype=torch.int8)
    return q, 0.01 + torch.rand(N, generator=g, device=DEV)


def _a(k, g, T, K):
    a = torch.zeros(T, k.int8_width(K), dtype=torch.int8, device=DEV)
    a[:, :K] = torch.randint(-127, 128, (T, K), generator=g, device=DEV, dtype=torch.int8)
    return a, 0.01 + torch.rand(T, generator=g, device=DEV)


def _sums(a, q, K):
    return a[:, :K].double() @ q.double().T


def _scaled(sums, a_scales, w_scales):
    """The roundings of the kernels: the sum to 32 bits, then two products."""
    return (sums.float() * a_scales[:, None]) * w_scales


SHAPES = [(1, 16, 1), (1, 2048, 2048), (3, 100, 130), (16, 8192, 256), (17, 4096, 333), (33, 1000, 64), (64, 4096, 1000), (65, 129, 2049),
          (128, 2064, 700), (100, 300, 19100), (200, 5000, 513), (256, 2048, 4096), (257, 512, 300), (300, 4096, 1024), (511, 1040, 129), (1000, 777, 1001), (2049, 2048, 512)]


@pytest.mark.parametrize("T,K,N", SHAPES)
def test_product(T, K, N):
    """The sums are exact and the scaling is two rounded products: results equal to the bit, in every form of output."""
    k = _kernels()
    g = _gen(T + K + N)
    q, ws = _weight(g, N, K)
    a, s = _a(k, g, T, K)
    w = k.int8_weight(q, ws)
    want = _scaled(_sums(a, q, K), s, ws)
    out = torch.full((T, N), math.nan, device=DEV)
    k.int8_product(a, s, w, out)
    assert torch.equal(out, want)
    half = torch.full((T, N), math.nan, dtype=torch.bfloat16, device=DEV)
    k.int8_product(a, s, w, half)
    assert torch.equal(half, want.to(torch.bfloat16))
    base = _normal(g, T, N) * 1000
    out = base.clone()
    k.int8_product(a, s, w, out, accumulate=True)
    assert torch.equal(out, base + want)
    wide = torch.full((T, N + 5), 7.0, device=DEV)                      # rows that lie apart, at an odd place
    k.int8_product(a, s, w, wide[:, 3:3 + N])
    assert torch.equal(wide[:, 3:3 + N], want) and (wide[:, :3] == 7).all() and (wide[:, 3 + N:] == 7).all()
    for dtype in (torch.float32, torch.bfloat16):                       # rows behind the last one stay as they were
        more = torch.full((T + 300, N), 7.0, device=DEV, dtype=dtype)
        k.int8_product(a, s, w, more[:T])
        assert torch.equal(more[:T], want.to(dtype)) and (more[T:] == 7).all()


@pytest.mark.parametrize("T", [5, 100, 1000])
def test_nothing_behind_a_rows_last_channel_is_written(T):
    """Rows that lie whole 16 bytes apart and end within them: a store of whole pieces would reach into what lies behind."""
    k = _kernels()
    g = _gen(T)
    for N in (333, 334, 335, 336, 1001, 2049):
        q, ws = _weight(g, N, 200)
        a, s = _a(k, g, T, 200)
        w = k.int8_weight(q, ws)
        want = _scaled(_sums(a, q, 200), s, ws)
        for dtype in (torch.float32, torch.bfloat16):
            wide = torch.full((T, (N + 15) // 16 * 16), 7.0, device=DEV, dtype=dtype)
            for plan in (None, ("many", 1)):
                k.int8_product(a, s, w, wide[:, :N], plan=plan)
                assert torch.equal(wide[:, :N], want.to(dtype)) and (wide[:, N:] == 7).all(), (N, dtype, plan)
        wide = torch.full((T, (N + 15) // 16 * 16), 7.0, device=DEV)
        for plan in (None, ("many", 1)):
            before = wide[:, :N].clone()
            k.int8_product(a, s, w, wide[:, :N], accumulate=True, plan=plan)
            assert torch.equal(wide[:, :N], before + want) and (wide[:, N:] == 7).all(), (N, plan)


@pytest.mark.parametrize("T,K,N", [(1, 8192, 2048), (40, 2048, 1500), (100, 1300, 640), (256, 4096, 512), (700, 900, 700)])
def test_every_cut_of_a_product_gives_the_same(T, K, N):
    k = _kernels()
    g = _gen(5)
    q, ws = _weight(g, N, K)
    a, s = _a(k, g, T, K)
    w = k.int8_weight(q, ws)
    want = _scaled(_sums(a, q, K), s, ws)
    for plan in [("few", bq, splits, stages) for bq in (8, 32, 64) for splits in (1, 2, 3, 5, 8) for stages in (1, 2, 4)] + \
            [("few", 128, 1, stages) for stages in (1, 2, 4)] + [("many", group) for group in (1, 3, 8)]:
        out = torch.full((T, N), math.nan, device=DEV)
        k.int8_product(a, s, w, out, plan=plan)
        assert torch.equal(out, want), plan
        half = torch.full((T, N), math.nan, dtype=torch.bfloat16, device=DEV)
        k.int8_product(a, s, w, half, plan=plan)
        assert torch.equal(half, want.to(torch.bfloat16)), plan
        k.int8_product(a, s, w, out, accumulate=True, plan=plan)
        assert torch.equal(out, want + want), plan


def test_the_largest_sums_stay_exact():
    k = _kernels()
    K = k.INT8_WIDTH_MOST
    for T in (2, 300):
        a = torch.full((T, K), 127, dtype=torch.int8, device=DEV)
        q = torch.full((5, K), -127, dtype=torch.int8, device=DEV)
        assert 128 * 128 * K < 2 ** 31
        out = torch.empty(T, 5, device=DEV)
        k.int8_product(a, torch.ones(T, device=DEV), k.int8_weight(q, torch.ones(5, device=DEV)), out)
        assert (out == -float(127 * 127 * K)).all()


def test_rows_without_a_scale_give_nan_or_zero():
    k = _kernels()
    g = _gen(9)
    q, ws = _weight(g, 200, 300)
    for T in (4, 400):
        x = _normal(g, T, 300)
        x[1, 7], x[2] = math.inf, 0
        a, s = _buffers(k, T, 300)
        k.quantize_rows(x, a, s)
        out = torch.empty(T, 200, device=DEV)
        k.int8_product(a, s, k.int8_weight(q, ws), out)
        assert torch.isnan(out[1]).all() and (out[2] == 0).all() and torch.isfinite(out[3:]).all() and torch.isfinite(out[0]).all()


@pytest.mark.parametrize("activation", ["silu", "relu", "gelu_tanh", "capped_swish"])
@pytest.mark.parametrize("T,K,I", [(1, 2048, 1024), (8, 100, 5), (130, 500, 1027), (256, 2048, 512), (257, 2048, 512), (300, 130, 1), (600, 777, 333), (1030, 1024, 2048)])
def test_gated_product(T, K, I, activation):
    k = _kernels()
    g = _gen(T + K + I)
    q, ws = _weight(g, 2 * I, K)
    ws = ws / (70 * 70 * math.sqrt(K))
    a, s = _a(k, g, T, K)
    w = k.int8_weight(q, ws, gated=True)
    for bias in (None, _normal(g, 2 * I) * 0.2):
        both = _scaled(_sums(a, q, K), s, ws)
        both = both if bias is None else both + bias
        h = _act64(both[:, :I], both[:, I:], activation, 2.0)
        out, scales = _buffers(k, T, I)
        work = torch.empty(k.int8_gated_work(T, w), device=DEV)
        k.int8_gated(a, s, w, out, scales, work, activation, 2.0, bias)
        _near_ints(out, scales, h, 2 * 2.0 ** -9 + 2.0 ** -18)


def test_a_feed_forward_of_them():
    """Norm, gate and up, activation, down, as the decoder runs them, against the definitions one by one."""
    k = _kernels()
    for T, H, I in ((1, 256, 512), (20, 333, 700), (300, 512, 1000)):
        g = _gen(T)
        up, down = _weight(g, 2 * I, H), _weight(g, H, I)
        up, down = (up[0], up[1] / (70 * math.sqrt(H))), (down[0], down[1] / (70 * math.sqrt(I)))
        x, add, weight = _normal(g, T, H), _normal(g, T, H), 0.5 + torch.rand(H, generator=g, device=DEV)
        stream = x + add
        q, s = _buffers(k, T, H)
        hq, hs = _buffers(k, T, I)
        out = stream.clone()
        k.rmsnorm_int8(x, weight, q, s, EPS, add=add)
        w = k.int8_weight(*up, gated=True)
        k.int8_gated(q, s, w, hq, hs, torch.empty(k.int8_gated_work(T, w), device=DEV))
        k.int8_product(hq, hs, k.int8_weight(*down), out, accumulate=True)
        assert torch.equal(x, stream)
        want_q, m = _ints(stream * weight)
        assert torch.equal(q[:, :H], want_q)
        both = _scaled(_sums(q, up[0], H), s, up[1])
        _near_ints(hq, hs, _act64(both[:, :I], both[:, I:], "silu", 0.0), 2 * 2.0 ** -9 + 2.0 ** -18)
        assert torch.equal(out, stream + _scaled(_sums(hq, down[0], I), hs, down[1]))


def test_offsets_beyond_32_bits():
    """More than 2^31 values in rows, integers and results: the last rows come out as they do alone."""
    k = _kernels()
    g = _gen(12)
    T, D = 131100, 16400                                                # rows: 2.15e9 values
    x = torch.zeros(T, D, dtype=torch.bfloat16, device=DEV)
    x[-3:] = _normal(g, 3, D)
    q, s = torch.empty(T, D, dtype=torch.int8, device=DEV), torch.empty(T, device=DEV)
    k.quantize_rows(x, q, s)
    want, m = _ints(x[-3:].float())
    _check_rows(q[-3:], s[-3:], want, m.double() / 127, D)
    assert (s[:-3] == 0).all() and not q[:4].any()
    del x
    w = k.int8_weight(*_weight(g, 130, D))
    out = torch.empty(T, 130, device=DEV)
    k.int8_product(q, s, w, out)
    few = torch.empty(3, 130, device=DEV)
    k.int8_product(q[-3:], s[-3:], w, few)
    assert torch.equal(out[-3:], few) and (out[:-3] == 0).all()
    del q, out
    T, N = 70000, 32768                                                 # results: 2.29e9 values
    a, s = _a(k, g, T, 64)
    w = k.int8_weight(*_weight(g, N, 64))
    out = torch.empty(T, N, dtype=torch.bfloat16, device=DEV)
    k.int8_product(a, s, w, out)
    few = torch.empty(5, N, dtype=torch.bfloat16, device=DEV)
    k.int8_product(a[-5:], s[-5:], w, few)
    assert torch.equal(out[-5:], few)


def test_no_rows():
    k = _kernels()
    g = _gen(2)
    w, gated = k.int8_weight(*_weight(g, 64, 32)), k.int8_weight(*_weight(g, 64, 32), gated=True)
    none = torch.empty(0, 32, device=DEV)
    q, s = _buffers(k, 0, 32)
    k.quantize_rows(none, q, s)
    k.rmsnorm_int8(none, torch.ones(32, device=DEV), q, s, EPS)
    k.gated_act_int8(torch.empty(0, 64, device=DEV), q, s)
    k.int8_product(q, s, w, torch.empty(0, 64, device=DEV))
    k.int8_gated(q, s, gated, q, s, torch.empty(0, device=DEV))
    torch.cuda.synchronize()


def test_tensors_of_two_devices_are_refused():
    k = _kernels()
    a, s = _a(k, _gen(1), 3, 64)
    x, one = torch.ones(3, 64, device=DEV), torch.ones(64, device=DEV)
    w = k.int8_weight(torch.ones(8, 64, dtype=torch.int8), torch.ones(8))
    for call in (lambda: k.int8_product(a, s, w, torch.empty(3, 8, device=DEV)), lambda: k.quantize_rows(x, a, s.cpu()), lambda: k.rmsnorm_int8(x, one.cpu(), a, s, EPS),
                 lambda: k.rmsnorm_int8(x, one, a.cpu(), s, EPS), lambda: k.gated_act_int8(x, a[:, :32].cpu(), s)):
        with pytest.raises(k.KernelError, match="one device"):
            call()


def test_two_streams_at_once():
    """Nothing is shared between calls: products, rows and gated halves of two streams beside each other give what they give alone."""
    k = _kernels()
    g = _gen(21)
    jobs = []
    for T, K, N in ((5, 4096, 1024), (700, 1024, 1500), (64, 2048, 4096), (300, 512, 8000)):
        w, pair = k.int8_weight(*_weight(g, N, K)), k.int8_weight(*_weight(g, 2 * N, K), gated=True)
        x = _normal(g, T, K)
        a, s = _buffers(k, T, K)
        h, hs = _buffers(k, T, N)
        jobs.append((x, a, s, w, pair, h, hs, torch.empty(k.int8_gated_work(T, pair), device=DEV), torch.empty(T, N, device=DEV)))

    def go(x, a, s, w, pair, h, hs, work, out):
        k.rmsnorm_int8(x, torch.ones(x.shape[1], device=DEV), a, s, EPS)
        k.int8_product(a, s, w, out)
        k.int8_gated(a, s, pair, h, hs, work)

    alone = []
    for job in jobs:
        go(*job)
        torch.cuda.synchronize()
        alone.append([t.clone() for t in (job[1], job[2], job[5], job[6], job[8])])
    for job in jobs:
        for t in (job[1], job[2], job[5], job[6], job[8]):
            t.zero_()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for i, job in enumerate(jobs):
            with torch.cuda.stream(streams[i % 2]):
                go(*job)
    torch.cuda.synchronize()
    for job, want in zip(jobs, alone):
        assert all(torch.equal(t, u) for t, u in zip((job[1], job[2], job[5], job[6], job[8]), want))


def test_in_a_captured_graph_and_on_another_stream():
    k = _kernels()
    g = _gen(4)
    for T in (8, 300):
        q, ws = _weight(g, 256, 512)
        w = k.int8_weight(q, ws)
        x, weight = _normal(g, T, 512), torch.ones(512, device=DEV)
        a, s = _buffers(k, T, 512)
        out = torch.empty(T, 256, device=DEV)

        def go():
            k.rmsnorm_int8(x, weight, a, s, EPS)
            k.int8_product(a, s, w, out)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            go()
        torch.cuda.current_stream().wait_stream(side)
        first = out.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            go()
        for scale in (1.0, 3.0):
            x.copy_(_normal(g, T, 512) * scale)
            graph.replay()
            want_q, _ = _ints(x)
            assert torch.equal(a, want_q)
            assert torch.equal(out, _scaled(_sums(a, q, 512), s, ws))
        assert first.shape == out.shape and torch.isfinite(first).all()
