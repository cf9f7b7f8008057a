"""Low-rank adapters of many rows at once against the formula in 64 bits.

The bound of an element: with B = scale sum_j |up| sum_k |x| |down|, sums of K and of rank terms in 32 bits are off by at most
2^-24 (K + rank + 16) B; the values between the two products may be held as two bfloat16 pieces (2^-16 B); the output is rounded to its
type. Besides, the whole error is held to 2e-5 of the whole (32 bits), as sums of many terms err by far less than their bound.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def K_():
    from geneinfer_b200.ops import kernels
    return kernels


def dt(name):
    return torch.float32 if name == "float32" else torch.bfloat16


def make(seed, T, K, widths, rank, A, dtype, out_dtype, base=True):
    g = torch.Generator().manual_seed(seed)
    S, N = len(widths), sum(widths)
    x = torch.randn(T, K, generator=g).to(dt(dtype)).to(DEV)
    down = (torch.randn(A, S * rank, K, generator=g) / math.sqrt(K)).to(dt(dtype)).to(DEV)
    up = (torch.randn(A, N, rank, generator=g) / math.sqrt(rank)).to(dt(dtype)).to(DEV)
    scales = (0.5 + torch.rand(A, generator=g)).to(DEV)
    out = (torch.randn(T, N, generator=g) if base else torch.zeros(T, N)).to(dt(out_dtype)).to(DEV)
    ids = torch.randint(-1, A, (T,), generator=g, dtype=torch.int32).to(DEV)
    return x, down, up, scales, out, ids


def exact(x, down, up, scales, out, ids, widths):
    """(result, bound of the element's error without the output's rounding), 64 bits."""
    want, bound = out.double().clone(), torch.zeros(out.shape, dtype=torch.float64, device=DEV)
    K, r = x.shape[1], up.shape[2]
    for a in ids.unique().tolist():
        if not 0 <= a < up.shape[0]:
            continue
        rows = (ids == a).nonzero()[:, 0]
        xa, d, s = x[rows].double(), down[a].double(), float(scales[a])
        h, hb = xa @ d.T * s, xa.abs() @ d.abs().T * s
        at = 0
        for i, n in enumerate(widths):
            u = up[a, at:at + n].double()
            want[rows, at:at + n] += h[:, i * r:(i + 1) * r] @ u.T
            bound[rows, at:at + n] = hb[:, i * r:(i + 1) * r] @ u.abs().T
            at += n
    return want, bound * (2.0 ** -24 * (K + r + 16) + 2.0 ** -16)


def compare(x, down, up, scales, out, ids, widths, got):
    want, bound = exact(x, down, up, scales, out, ids, widths)
    unit = 2.0 ** -24 if out.dtype == torch.float32 else 2.0 ** -8
    error = (got.double() - want).abs()
    assert bool((error <= bound + unit * want.abs() * 1.01 + 1e-30).all()), float((error - bound - unit * want.abs()).max())
    whole = float(want.norm())
    assert float(error.norm()) <= (2e-5 if out.dtype == torch.float32 else 2.0 ** -8) * whole
    alone = ~((ids >= 0) & (ids < up.shape[0]))
    assert torch.equal(got[alone], out[alone]), "a row without an adapter was touched"


def run(x, down, up, scales, out, ids, widths):
    plan = K_().adapter_plan(ids, up.shape[0])
    got = out.clone()
    K_().adapter_product(x, down, up, scales, plan, got, widths if len(widths) > 1 else None)
    return got


TYPES = [("float32", "float32"), ("bfloat16", "float32"), ("bfloat16", "bfloat16")]


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("T,K,widths,rank,A", [
    (1, 1, (1,), 1, 1), (1, 2048, (2048,), 16, 1), (2, 33, (7,), 3, 2), (8, 2048, (2048,), 16, 8), (15, 1000, (129, 3), 5, 4), (16, 64, (40,), 4, 30),
    (17, 520, (264,), 8, 3), (64, 2048, (512, 128, 128), 16, 9), (100, 256, (96,), 64, 2), (255, 2056, (1000, 520), 12, 24), (256, 1024, (512,), 32, 40),
    (257, 1024, (512,), 32, 7), (300, 4096, (640, 128, 64, 8), 24, 5), (700, 2048, (2048,), 12, 3), (1000, 136, (264,), 128, 11), (130, 72, (24,), 256, 3),
    (1500, 328, (1028,), 16, 1), (333, 999, (257,), 7, 6), (513, 2048, (250, 250), 100, 2), (1024, 264, (72,), 8, 1000), (1025, 264, (72,), 8, 1000),
    (200, 128, (64,), 8, 1024), (200, 128, (64,), 8, 1025), (3000, 72, (40,), 4, 5000), (5000, 520, (96, 32), 16, 3), (4100, 264, (64,), 64, 9)])
def test_adapters_of_many_rows(dtype, out_dtype, T, K, widths, rank, A):
    x, down, up, scales, out, ids = make(T + K + rank, T, K, widths, rank, A, dtype, out_dtype)
    compare(x, down, up, scales, out, ids, widths, run(x, down, up, scales, out, ids, widths))


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("T", [5, 640])
def test_the_adapters_part_alone(dtype, out_dtype, T):
    """Nothing under it: the product's own precision shows."""
    x, down, up, scales, out, ids = make(3, T, 2048, (768,), 16, 4, dtype, out_dtype, base=False)
    ids.fill_(2)
    got = run(x, down, up, scales, out, ids, (768,))
    compare(x, down, up, scales, out, ids, (768,), got)
    if out_dtype == "float32":
        want, _ = exact(x, down, up, scales, out, ids, (768,))
        assert float((got.double() - want).norm()) <= 1e-5 * float(want.norm())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [40, 1000])
def test_rows_in_any_order_none_at_all_and_numbers_beyond(dtype, T):
    x, down, up, scales, out, ids = make(4, T, 264, (136,), 8, 12, dtype, "float32")
    for order in ("sorted", "reversed", "one", "last", "none", "beyond"):
        some = {"sorted": ids.sort().values, "reversed": ids.sort(descending=True).values, "one": torch.full_like(ids, 5),
                "last": torch.where(torch.arange(T, device=DEV) == T - 1, 11, -1).int(), "none": torch.full_like(ids, -1),
                "beyond": torch.where(torch.arange(T, device=DEV) % 3 == 0, 12 + ids, -5 - ids).int()}[order].contiguous()
        compare(x, down, up, scales, out, some, (136,), run(x, down, up, scales, out, some, (136,)))


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("T,K,N,offset", [(33, 200, 120, 8), (33, 200, 121, 1), (400, 201, 64, 3), (20, 256, 64, 4)])
def test_columns_of_wider_tensors(dtype, out_dtype, T, K, N, offset):
    x, down, up, scales, out, ids = make(5, T, K, (N,), 8, 3, dtype, out_dtype)
    wide_x = torch.full((T, K + 24), float("nan"), dtype=x.dtype, device=DEV)
    wide_x[:, offset:offset + K] = x
    wide_out = torch.full((T, N + 24), 7.0, dtype=out.dtype, device=DEV)
    wide_out[:, offset:offset + N] = out
    K_().adapter_product(wide_x[:, offset:offset + K], down, up, scales, K_().adapter_plan(ids, 3), wide_out[:, offset:offset + N])
    compare(x, down, up, scales, out, ids, (N,), wide_out[:, offset:offset + N])
    assert (wide_out[:, :offset] == 7).all() and (wide_out[:, offset + N:] == 7).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("T", [30, 500])
def test_what_is_not_read_does_not_show(dtype, T):
    """No number in an adapter that no row has, in rows without an adapter, in one row: only that row has none."""
    x, down, up, scales, out, ids = make(6, T, 128, (64, 32), 8, 5, dtype, "float32")
    ids[ids == 3] = 1
    ids[7], ids[8] = -1, 2
    want = run(x, down, up, scales, out, ids, (64, 32))
    down[3], up[3], scales[3] = math.nan, math.inf, math.nan
    x[7] = math.nan
    x[8, 5] = math.nan
    got = run(x, down, up, scales, out, ids, (64, 32))
    same = torch.arange(T, device=DEV) != 8
    assert torch.equal(got[same], want[same]) and torch.isnan(got[8]).all()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_same_bits_every_time_and_in_every_batch_of_a_size(dtype):
    x, down, up, scales, out, ids = make(7, 600, 1024, (512,), 16, 6, dtype, "float32")
    first = run(x, down, up, scales, out, ids, (512,))
    for _ in range(3):
        assert torch.equal(run(x, down, up, scales, out, ids, (512,)), first)
    order = torch.randperm(600, generator=torch.Generator().manual_seed(1)).to(DEV)
    assert torch.equal(run(x[order].contiguous(), down, up, scales, out[order].contiguous(), ids[order].contiguous(), (512,)), first[order])


def test_streams_buffers_and_programs():
    x, down, up, scales, out, ids = make(8, 2500, 512, (256,), 16, 4, "bfloat16", "float32")
    want = run(x, down, up, scales, out, ids, (256,))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    buffer = torch.full((K_().adapter_plan_size(2500, 4),), -7, dtype=torch.int32, device=DEV)
    got = out.clone()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side), K_().record() as rec:
        K_().adapter_product(x, down, up, scales, K_().adapter_plan(ids, 4, buffer), got)
    side.synchronize()
    assert torch.equal(got, want)
    got.copy_(out)
    rec.program.run()
    assert torch.equal(got, want) and len(rec.program) == 2


def test_a_plan_serves_every_number_of_rows_up_to_its_size():
    size = K_().adapter_plan_size(3000, 9)
    for T in (0, 1, 16, 255, 256, 257, 1023, 1024, 1025, 3000):
        plan = K_().adapter_plan(torch.arange(T, dtype=torch.int32, device=DEV) % 9, 9, torch.empty(size, dtype=torch.int32, device=DEV))
        assert plan.rows == T
    with pytest.raises(K_().KernelError):
        K_().adapter_plan(torch.zeros(3001, dtype=torch.int32, device=DEV), 9, torch.empty(3000, dtype=torch.int32, device=DEV))


def test_adapters_refuse_what_does_not_fit():
    x, down, up, scales, out, ids = make(9, 12, 64, (32, 16), 8, 3, "bfloat16", "float32")
    plan = K_().adapter_plan(ids, 3)
    good = dict(x=x, down=down, up=up, scales=scales, plan=plan, out=out, slices=(32, 16))
    K_().adapter_product(**good)
    for name, value in (("x", x.float()), ("x", x[:, :63]), ("x", x[:5]), ("x", x.cpu()), ("x", x.t().contiguous().t()), ("down", down[:, :8].contiguous()), ("down", down[:2]),
                        ("down", down.float()), ("down", down.transpose(1, 2).contiguous().transpose(1, 2)), ("up", up[:, :40].contiguous()), ("up", up[:2]),
                        ("scales", scales[:2]), ("scales", scales.double()), ("out", out.half()), ("out", out[:, :40]), ("out", out.t().contiguous().t()),
                        ("out", out[:1].expand(12, 48)), ("slices", (32,)), ("slices", (48, 0)), ("slices", (50, -2)), ("slices", (20, 16)), ("slices", None),
                        ("plan", K_().adapter_plan(ids, 4)), ("plan", K_().adapter_plan(ids[:11].contiguous(), 3))):
        with pytest.raises(K_().KernelError):
            K_().adapter_product(**dict(good, **{name: value}))
    with pytest.raises(K_().KernelError):
        K_().adapter_product(x.float(), down.float(), up.float(), scales, plan, out.bfloat16(), (32, 16))
    wide = make(9, 4, 16, (8,), 513, 1, "float32", "float32")
    with pytest.raises(K_().KernelError):
        run(*wide[:5], wide[5], (8,))
    for bad in (ids.long(), ids.cpu()):
        with pytest.raises(K_().KernelError):
            K_().adapter_plan(bad, 3)
    with pytest.raises(K_().KernelError):
        K_().adapter_plan(ids, 0)
    with pytest.raises(K_().KernelError):
        K_().adapter_plan(ids, 8193)
    for used in (0, 4):
        with pytest.raises(K_().KernelError):
            K_().adapter_plan(ids, 3, used=used)


@pytest.mark.parametrize("T", [100, 700, 3000])
def test_few_of_many_adapters(T):
    x, down, up, scales, out, ids = make(11, T, 128, (72,), 8, 900, "bfloat16", "float32")
    ids = torch.where(ids >= 0, ids % 5 * 179, ids).contiguous()
    got = out.clone()
    K_().adapter_product(x, down, up, scales, K_().adapter_plan(ids, 900, used=5), got)
    compare(x, down, up, scales, out, ids, (72,), got)


def test_the_rows_that_need_no_plan_are_the_librarys():
    from geneinfer_b200.ops import kernels
    from geneinfer_b200.ops.library import lib
    assert lib().gi_adapter_direct_rows(kernels.ADAPTER_DIRECT_ADAPTERS) == kernels.ADAPTER_DIRECT_ROWS
    assert lib().gi_adapter_direct_rows(kernels.ADAPTER_DIRECT_ADAPTERS + 1) == 0


def test_the_limits_are_the_librarys():
    from geneinfer_b200.ops import kernels
    from geneinfer_b200.ops.library import lib
    assert lib().gi_adapter_ranks_most() == kernels.ADAPTER_RANKS_MOST and lib().gi_adapter_adapters_most() == kernels.ADAPTER_ADAPTERS_MOST


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("T", [3, 40, 500, 2500])
def test_the_values_between_the_products_keep_all_their_bits(dtype, out_dtype, T):
    """(1 + 2^-9 + 2^-18) - (1 + 2^-9): every product and sum is exact in 32 bits, and so is the answer in either type."""
    K, N = 64, 40
    x = torch.zeros(T, K, dtype=dt(dtype), device=DEV)
    x[:, 0], x[:, 1], x[:, 2] = 1.0, 2.0 ** -9, 2.0 ** -18
    down = torch.zeros(1, 4, K, dtype=dt(dtype), device=DEV)
    down[:, 0, :3], down[:, 1, :2] = 1.0, 1.0
    up = torch.zeros(1, N, 4, dtype=dt(dtype), device=DEV)
    up[:, :, 0], up[:, :, 1] = 1.0, -1.0
    out = torch.zeros(T, N, dtype=dt(out_dtype), device=DEV)
    got = run(x, down, up, torch.ones(1, device=DEV), out, torch.zeros(T, dtype=torch.int32, device=DEV), (N,))
    assert bool((got == 2.0 ** -18).all())


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("T", [9, 200, 500, 3000])
@pytest.mark.parametrize("rank", [4, 12, 24, 40, 80])
def test_infinite_values_of_the_second_matrix(dtype, out_dtype, T, rank):
    """An infinity times a number that is not zero is infinite, whatever the values between the products are held as; two of opposite signs are no number. Row t's
    values between the products are all 1 (three bits of a sum) or all 1 + 2^-9 + 2^-18 (no part of it is like another)."""
    K, N, A = 64, 72, 2
    x = torch.zeros(T, K)
    x[:, 0] = 1.0
    x[1::2, 1], x[1::2, 2] = 2.0 ** -9, 2.0 ** -18
    x[2::3] *= -1
    down = torch.zeros(A, rank, K)
    down[:, :, :3] = 1.0
    up = torch.full((A, N, rank), 2.0 ** -6)
    up[0, 5, 1], up[0, 17, rank - 1], up[0, 40, 0] = math.inf, -math.inf, math.inf
    up[0, 40, rank - 2] = -math.inf
    up[0, 71] = math.inf
    up[0, 60, 3] = math.nan
    x, down, up = (v.to(dt(dtype)).to(DEV) for v in (x, down, up))
    scales = torch.ones(A, device=DEV)
    out = torch.zeros(T, N, dtype=dt(out_dtype), device=DEV)
    ids = torch.arange(T, dtype=torch.int32, device=DEV) % 3 - 1
    got = run(x, down, up, scales, out, ids, (N,)).float()
    want, _ = exact(x, down, up, scales, out, ids, (N,))
    want = want.float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(torch.isinf(got), torch.isinf(want))
    some = torch.isinf(want)
    assert torch.equal(got[some], want[some])
    rest = torch.isfinite(want)
    assert bool(((got - want)[rest].abs() <= 2.0 ** -8 * want[rest].abs()).all())


@pytest.mark.parametrize("dtype,out_dtype", TYPES)
@pytest.mark.parametrize("T", [9, 500])
def test_sums_between_the_products_near_the_largest_value(dtype, out_dtype, T):
    """3.3996e38 is finite in 32 bits and rounds to an infinity in bfloat16."""
    K, N = 64, 40
    x = torch.zeros(T, K, dtype=dt(dtype), device=DEV)
    x[:, 0], x[:, 1], x[:, 2] = 2.0 ** 127, 2.0 ** 126, 2.0 ** 119
    down = torch.zeros(1, 4, K, dtype=dt(dtype), device=DEV)
    down[:, :, 0], down[:, :, 1], down[:, :, 2] = 1.0, 1.984375, 1.5
    up = torch.full((1, N, 4), 2.0 ** -70, dtype=dt(dtype), device=DEV)
    ids = torch.zeros(T, dtype=torch.int32, device=DEV)
    out = torch.zeros(T, N, dtype=dt(out_dtype), device=DEV)
    assert 3.39e38 < 2.0 ** 127 + 2.0 ** 126 * 1.984375 + 2.0 ** 119 * 1.5 < float(torch.finfo(torch.float32).max)
    compare(x, down, up, torch.ones(1, device=DEV), out, ids, (N,), run(x, down, up, torch.ones(1, device=DEV), out, ids, (N,)))


@pytest.mark.parametrize("T", [9, 500])
def test_infinite_values_between_the_products(T):
    """Infinite inputs times a second matrix of numbers, zeros and infinities: the formula's infinities and its places without a number."""
    K, N = 64, 40
    g = torch.Generator().manual_seed(T)
    x = torch.randn(T, K, generator=g)
    x[::2, 7] = math.inf
    x[1::4, 7] = -math.inf
    down = torch.zeros(1, 4, K)
    down[0, :, 7] = torch.tensor([1.0, -1.0, 0.5, 0.0])          # (the last is zero times infinity: no number)
    down[0, 3, 8] = 1.0
    up = torch.randn(1, N, 4, generator=g)
    up[0, :, 3] = 0.0
    up[0, ::3, 1] = 0.0
    up[0, 4, 2] = math.inf
    x, down, up = (v.bfloat16().to(DEV) for v in (x, down, up))
    ids = torch.zeros(T, dtype=torch.int32, device=DEV)
    out = torch.zeros(T, N, device=DEV)
    got = run(x, down, up, torch.ones(1, device=DEV), out, ids, (N,))
    want = exact(x, down, up, torch.ones(1, device=DEV), out, ids, (N,))[0].float()
    finite = torch.isfinite(x).all(1)
    assert torch.isnan(got[~finite]).all() and torch.isnan(want[~finite]).all()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    # without the row of zeros times infinity: infinities of either sign, and cancelling ones
    down[0, 3] = 0.25
    up[0, :, 3] = 0.0078125
    got = run(x, down, up, torch.ones(1, device=DEV), out, ids, (N,))
    want = exact(x, down, up, torch.ones(1, device=DEV), out, ids, (N,))[0].float()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[torch.isinf(want)], want[torch.isinf(want)])
    assert bool(torch.isinf(want).any()) and bool(torch.isnan(want).any())
