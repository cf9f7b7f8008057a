"""Weights and rows in 8-bit integers without a GPU: layouts, plans, scratch sizes, and what is refused before a kernel runs."""
import pytest
import torch

import kidarax_configs
import nipadra_configs
import tiny_configs as tc
from geneinfer_b200.ops import kernels as k


def _unlaid(w, K):
    """[parts, channels, K] from the tiles: the definition of the layout, read backwards."""
    parts = 2 if w.gated else 1
    blocks = (w.width + 127) // 128
    t = w.tiles.view(-1, parts, blocks, 128, 8, 16)
    out = torch.zeros(parts, t.shape[0] * 128, blocks * 128, dtype=torch.int8)
    for tile in range(t.shape[0]):
        for part in range(parts):
            for b in range(blocks):
                for piece in range(8):
                    for r in range(128):
                        out[part, tile * 128 + r, b * 128 + piece * 16:b * 128 + piece * 16 + 16] = t[tile, part, b, r, piece ^ (r % 8)]
    return out


@pytest.mark.parametrize("N,K,gated", [(1, 1, False), (130, 200, False), (256, 128, False), (6, 33, True), (300, 129, True)])
def test_the_layout_of_a_weight(N, K, gated):
    g = torch.Generator().manual_seed(N + K)
    q = torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8)
    w = k.int8_weight(q, torch.ones(N), gated=gated)
    parts = 2 if gated else 1
    assert (w.channels, w.width, w.gated) == (N // parts, k.int8_width(K), gated) and w.width % 16 == 0 and 0 <= w.width - K < 16
    back = _unlaid(w, K)
    assert torch.equal(back[:, :N // parts, :K], q.view(parts, N // parts, K))
    assert not back[:, N // parts:].any() and not back[:, :, K:].any()


def test_plans_fit_the_kernels():
    """Every plan names a tile that exists, ranges of K that are not empty, and few rows' CTAs that fit on the GPU at once."""
    w = k.int8_weight(torch.zeros(1, 1, dtype=torch.int8), torch.ones(1))
    for channels in (1, 128, 300, 2048, 6144, 16384, 128256):
        for width in (16, 128, 2048, 14336, k.INT8_WIDTH_MOST):
            for gated in (False, True):
                w.channels, w.width, w.gated, w.works = channels, width, gated, {}
                few_ended = False
                for T in list(range(0, 70)) + [96, 128, 200, 256, 300, 512, 1000, 4096, 100000]:
                    plan = k._int8_plan_of(T, w)
                    if plan[0] == "few":
                        _, bq, splits, stages = plan
                        assert bq in (8, 32, 64, 128) and 1 <= splits <= (1 if bq == 128 else 8) and stages == 0 and not few_ended
                        assert splits == 1 or splits * ((channels + 127) // 128) * (2 if gated else 1) * ((T + bq - 1) // bq) <= 264
                        assert splits <= (width + 127) // 128
                        assert not gated or 2 * channels * T <= k.int8_gated_work(T, w)
                    else:
                        few_ended = True
                        assert T > 64 and 1 <= plan[1] <= (T + 255) // 256
                        assert not gated or (channels + 7) // 8 * 8 * T <= 2 * k.int8_gated_work(T, w)
                    assert not gated or k.int8_gated_work(T, w) <= k.int8_gated_work(T + 1, w)


def test_weights_that_do_not_fit_are_refused():
    q, s = torch.zeros(4, 8, dtype=torch.int8), torch.ones(4)
    for bad in ((q.float(), s), (q, s[:3]), (q, s.double()), (q[0], s), (q[:, :0], s), (torch.zeros(1, k.INT8_WIDTH_MOST + 1, dtype=torch.int8), s[:1])):
        with pytest.raises(k.KernelError):
            k.int8_weight(*bad)
    with pytest.raises(k.KernelError, match="two parts"):
        k.int8_weight(q[:3], s[:3], gated=True)


def test_calls_that_do_not_fit_are_refused():
    """Shapes first, so that a wrong call is told what is wrong with it on any machine; then that there is no CPU path."""
    x, w, s = torch.zeros(3, 20), torch.ones(20), torch.zeros(3)
    q = torch.zeros(3, 32, dtype=torch.int8)
    for call in (lambda: k.quantize_rows(x, q[:, :16], s), lambda: k.quantize_rows(x, q[:2], s), lambda: k.quantize_rows(x, q, s[:2]),
                 lambda: k.quantize_rows(x[0], q, s), lambda: k.quantize_rows(x[:, :0], q, s),
                 lambda: k.rmsnorm_int8(x, w[:19], q, s, 1e-5), lambda: k.rmsnorm_int8(x, w, q, s, 1e-5, add=x[:2]),
                 lambda: k.rmsnorm_int8(x.bfloat16(), w, q, s, 1e-5), lambda: k.rmsnorm_int8(x, w, q, s, 1e-5, add=x),
                 lambda: k.gated_act_int8(x[:, :19], q, s), lambda: k.gated_act_int8(torch.zeros(3, 40), q, s, "tanh"),
                 lambda: k.gated_act_int8(torch.zeros(3, 40), q, s, bias=torch.zeros(20)),
                 lambda: k.quantize_rows(x, q, s), lambda: k.quantize_rows(x.double(), q, s)):
        with pytest.raises(k.KernelError):
            call()
    plain, pair = k.int8_weight(torch.zeros(8, 20, dtype=torch.int8), torch.ones(8)), k.int8_weight(torch.zeros(8, 20, dtype=torch.int8), torch.ones(8), gated=True)
    out, wide = torch.zeros(3, 8), torch.zeros(100)
    for call in (lambda: k.int8_product(q[:, :16], s, plain, out), lambda: k.int8_product(q, s[:2], plain, out), lambda: k.int8_product(q, s, pair, out),
                 lambda: k.int8_product(q, s, plain, out[:, :7]), lambda: k.int8_product(q, s, plain, out.bfloat16(), accumulate=True),
                 lambda: k.int8_gated(q, s, plain, q[:, :16], s, wide), lambda: k.int8_gated(q, s, pair, q, s, wide),
                 lambda: k.int8_gated(q, s, pair, q[:, :16].contiguous(), s, wide, "tanh"), lambda: k.int8_gated(q, s, pair, q[:, :16].contiguous(), s, wide[:4]),
                 lambda: k.int8_gated(q, s, pair, q[:, :16].contiguous(), s, wide, bias=torch.zeros(4))):
        with pytest.raises(k.KernelError):
            call()


def test_models_without_such_a_form_are_refused():
    from geneinfer_b200 import Engine, SpeculativeEngine
    from geneinfer_b200.config import parse_config
    from geneinfer_b200.parts import DecoderModel
    with pytest.raises(ValueError, match="adapters"):
        Engine("nowhere", adapter_slots=1, weights="int8")
    with pytest.raises(ValueError, match="adapters"):
        SpeculativeEngine("nowhere", "nowhere", adapter_slots=1, weights="int8")
    for config in (nipadra_configs.NIP_P, kidarax_configs.KID_A):
        with pytest.raises(ValueError, match="8 bits"):
            DecoderModel(parse_config(config)[1].model_spec(), {}, torch.bfloat16, torch.device("cpu"), weights="int8")
    llama = parse_config(tc.TINY_A)[1].model_spec()
    with pytest.raises(ValueError, match="int4"):
        DecoderModel(llama, {}, torch.bfloat16, torch.device("cpu"), weights="int4")


def test_command_line():
    from geneinfer_b200.cli.generate_main import UsageError, parse
    base = ["--model", "m", "--prompt-ids", "1 2"]
    assert parse(base + ["--weights", "int8"])["weights"] == "int8"
    assert parse(base + ["--weights", "int8", "--dtype", "bf16"])["weights"] == "int8"
    assert parse(base + ["--weights", "int8", "--dtype", "fp32"])["weights"] == "f32"
    assert parse(base + ["--dtype", "bf16"])["weights"] == "native"
    for bad in (["--weights", "int4"], ["--weights", "int8", "--adapter", "a"]):
        with pytest.raises(UsageError):
            parse(base + bad)


def test_an_addition_that_overlaps_the_stream_is_refused():
    """The stream is written while the addition is read, by other blocks: any shared value is a race. Between rows that lie apart nothing is shared."""
    D = 20
    flat, w = torch.zeros(40 * D), torch.ones(D)

    def call(x, add):
        T = x.shape[0]
        return lambda: k.rmsnorm_int8(x, w, torch.zeros(T, 32, dtype=torch.int8), torch.zeros(T), 1e-5, add=add)

    rows = flat.view(-1, D)
    apart = flat.view(-1, 4 * D)[:, :D]
    for x, add in ((rows[1:], rows[:-1]), (rows[:-1], rows[1:]), (rows[:5], rows[:5]), (rows[:5], rows[4:9]), (flat[:3 * D].view(3, D), flat[1:3 * D + 1].view(3, D)),
                   (apart[:2], rows[3:5]), (apart[:2], rows[4:6]), (apart[1:3], rows[3:5]), (apart[:1], rows[:1]), (rows[1:3], flat.view(torch.bfloat16)[2 * D:4 * D].view(2, D))):
        with pytest.raises(k.KernelError, match="overlap"):
            call(x, add)()
    for x, add in ((rows[:5], rows[5:10]), (rows[5:10], rows[:5]), (apart[:2], rows[1:3]), (apart[:2], rows[2:4]), (apart[:1], rows[1:2]), (apart[8:], rows[38:40][:2]),
                   (rows[2:3], flat.view(torch.bfloat16)[:D].view(1, D))):
        with pytest.raises(k.KernelError, match="no CPU path"):      # taken, up to there
            call(x, add)()


def test_plans_that_do_not_exist_are_refused():
    """By an error code of the library, before anything is divided by a tile's height or launched (no GPU needed)."""
    a, scales, out = torch.zeros(16, 16, dtype=torch.int8), torch.ones(16), torch.zeros(16, 4)
    w = k.int8_weight(torch.zeros(4, 16, dtype=torch.int8), torch.ones(4))
    room = torch.zeros(w.tiles.numel() + 128, dtype=torch.int8)
    tiles = room.data_ptr() + -room.data_ptr() % 128
    status = torch.zeros(1, dtype=torch.int32)

    def few(bq, splits, ldo=4, gated=0):
        return k.lib().gi_int8_product_few(a.data_ptr(), scales.data_ptr(), 16, 16, tiles, scales.data_ptr(), 4, gated, out.data_ptr(), k.F32, ldo, 0, bq, splits, 0, 0,
                                           status.data_ptr(), 0)

    def many(group, ldo=4):
        return k.lib().gi_int8_product_many(a.data_ptr(), scales.data_ptr(), 16, 16, tiles, scales.data_ptr(), 4, 0, 0, 0.0, 0, out.data_ptr(), k.F32, ldo, 0, group,
                                            status.data_ptr(), 0)

    for code, message in ((lambda: few(0, 1), "tiles of 0 rows"), (lambda: few(-8, 1), "tiles of -8 rows"), (lambda: few(16, 1), "tiles of 16 rows"), (lambda: few(8, 0), "ranges of K"),
                          (lambda: few(8, 9), "ranges of K"), (lambda: few(128, 2), "ranges of K"), (lambda: few(8, 1, ldo=3), "overlap"), (lambda: few(8, 1, ldo=7, gated=1), "overlap"),
                          (lambda: many(0), "groups of 0"), (lambda: many(1, ldo=0), "overlap")):
        with pytest.raises(k.KernelError, match=message):
            k.check(code(), "int8_product")


def test_command_line_weights_and_type_in_either_order():
    """``--weights int8`` and ``--dtype`` say two things, and neither is lost to the other's place."""
    from geneinfer_b200.cli.generate_main import UsageError, parse
    base = ["--model", "m", "--prompt-ids", "1 2"]
    int8, fp32, bf16, f32, native = ["--weights", "int8"], ["--dtype", "fp32"], ["--dtype", "bf16"], ["--weights", "f32"], ["--weights", "native"]
    for flags, want in (([], (False, "bfloat16")), (int8, (True, "bfloat16")), (int8 + fp32, (True, "float32")), (fp32 + int8, (True, "float32")),
                        (int8 + bf16, (True, "bfloat16")), (bf16 + int8, (True, "bfloat16")), (fp32 + int8 + bf16, (True, "bfloat16")), (fp32, (False, "float32")),
                        (f32, (False, "float32")), (f32 + int8, (True, "bfloat16")), (int8 + f32, (False, "float32")), (fp32 + native, (False, "bfloat16")),
                        (f32 + bf16, (False, "bfloat16")), (native + fp32, (False, "float32")), (int8 + fp32 + native, (False, "bfloat16"))):
        o = parse(base + flags)
        assert (o["int8"], o["dtype"]) == want, flags
    for flags in (int8 + fp32, fp32 + int8):
        with pytest.raises(UsageError, match="--adapter"):
            parse(base + flags + ["--adapter", "a"])


def test_a_bound_below_zero_is_refused():
    """Such a bound makes something of the zeros behind a row (min(0, limit)), which would go into its integers and its scale. No GPU needed."""
    x, q, s = torch.zeros(2, 40), torch.zeros(2, 32, dtype=torch.int8), torch.zeros(2)
    room = torch.zeros(64 + 16, dtype=torch.int8)
    at = room.data_ptr() + -room.data_ptr() % 16

    def rows(limit, activation):
        return k.lib().gi_rows_int8(2, x.data_ptr(), k.F32, 40, 0, 0, 0, 0.0, k.ACTIVATIONS[activation], limit, at, 32, s.data_ptr(), 2, 20, 0, 0)

    with pytest.raises(k.KernelError, match="bound of -1"):
        k.check(rows(-1.0, "capped_swish"), "gated_act_int8")
    tiles = torch.zeros(2 * 16384 + 128, dtype=torch.int8)
    a = torch.zeros(2 * 16 + 16, dtype=torch.int8)
    code = k.lib().gi_int8_product_many(a.data_ptr() + -a.data_ptr() % 16, s.data_ptr(), 2, 16, tiles.data_ptr() + -tiles.data_ptr() % 128, s.data_ptr(), 20, 1,
                                        k.ACTIVATIONS["capped_swish"], -1.0, 0, x.data_ptr(), k.BF16, 24, 0, 1, s.data_ptr(), 0)
    with pytest.raises(k.KernelError, match="bound of -1"):
        k.check(code, "int8_gated")


def test_tiles_put_together_by_hand_have_to_be_the_weights():
    """The kernels take sizes from the weight: tiles or scales that are fewer would be read behind their end."""
    w = k.int8_weight(torch.zeros(300, 200, dtype=torch.int8), torch.ones(300))
    pair = k.int8_weight(torch.zeros(300, 200, dtype=torch.int8), torch.ones(300), gated=True)
    assert k.Int8Weight(w.tiles, w.scales, 300, 208, False).constant is False and w.constant and pair.constant
    k.Int8Weight(pair.tiles, pair.scales, 150, 208, True)
    for tiles, scales, channels, width, gated in ((w.tiles[:-1], w.scales, 300, 208, False), (w.tiles, w.scales, 300, 257 + 15, False), (w.tiles, w.scales, 385, 208, False),
                                                  (w.tiles, w.scales, 300, 208, True), (w.tiles, w.scales[:299], 300, 208, False), (w.tiles, w.scales.double(), 300, 208, False),
                                                  (w.tiles.float(), w.scales, 300, 208, False), (w.tiles, w.scales, 300, 200, False), (w.tiles, w.scales, 0, 208, False),
                                                  (w.tiles.view(2, -1).T, w.scales, 300, 208, False), (pair.tiles, pair.scales[:150], 150, 208, True)):
        with pytest.raises(k.KernelError, match="Int8Weight"):
            k.Int8Weight(tiles, scales, channels, width, gated)
