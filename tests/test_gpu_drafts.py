"""Verification of drafted tokens and token probabilities against plain 64-bit computations of their formulas.

A kept or drawn token is a decision about real numbers, so it is checked as one: the drawn token's interval of the running sum, in
64 bits, must hold the target within the error that the 32-bit probabilities may have, and a draft may be kept or refused either way only
where both sides of its comparison agree within that error. The bound of a probability's relative error: the argument (l - m) / T is
rounded twice (2^-24 each, of its own size), exp and the product with the reciprocal add at most three units in the last place:
2^-23 (|argument| + 4).
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def K():
    from geneinfer_b200.ops import kernels
    return kernels


def dt(name):
    return torch.float32 if name == "float32" else torch.bfloat16


def distribution(row, t):
    """(p, bound of |error|) of a row in 64 bits; None where it has none."""
    z = row.double()
    m = z.max()
    if bool(torch.isnan(z).any()) or not math.isfinite(float(m)):
        return None
    a = (z - m) / t
    p = torch.exp(a)
    p = p / p.sum()
    bound = torch.where(p > 0, p * 2.0 ** -23 * (a.abs().clamp(max=1e4) + 4), 0.0) + 2.0 ** -126
    return p, bound


def argmax_of(row):
    z = row.double()
    z = torch.where(torch.isnan(z), torch.full_like(z, -math.inf), z)
    some = (z == z.max()).nonzero()[:, 0]
    keep = some[~torch.isnan(row[some])]
    return int(keep[0]) if keep.numel() else 0


def check_verification(logits, row_start, drafted, counts, q, t, accept, draw, tokens, accepted):
    logits, tokens, accepted = logits.float().cpu(), tokens.cpu().tolist(), accepted.cpu().tolist()
    t, accept, draw = t.cpu().tolist(), accept.cpu(), draw.cpu().tolist()
    V = logits.shape[1]
    for r, (s, d) in enumerate(zip(row_start.tolist(), counts.tolist())):
        kept = accepted[r]
        assert 0 <= kept <= d, (r, kept, d)
        assert tokens[r][:kept] == drafted[r, :kept].tolist() and all(x == -1 for x in tokens[r][kept + 1:]), r
        got = tokens[r][kept]
        assert 0 <= got < V, (r, got)
        if not t[r] > 0:
            for j in range(min(kept + 1, d)):
                assert (int(drafted[r, j]) == argmax_of(logits[s + j])) == (j < kept), (r, j)
            assert got == argmax_of(logits[s + kept]), r
            continue
        for j in range(min(kept + 1, d)):
            x, dist = int(drafted[r, j]), distribution(logits[s + j], t[r])
            if dist is None:
                assert j == kept, f"request {r}: a draft was kept by a row without a distribution"
                continue
            p, bound = dist
            px, slack = (float(p[x]), float(bound[x])) if 0 <= x < V else (0.0, 0.0)
            qx = (float(q[r, j, x]) if 0 <= x < V else 0.0) if q is not None else 1.0
            left = float(accept[r, j]) * qx
            slack += left * 2.0 ** -23
            if j < kept:
                assert 0 <= x < V and left < px + slack, (r, j, left, px)
            else:
                assert not (0 <= x < V) or left >= px - slack, (r, j, left, px)
        dist = distribution(logits[s + kept], t[r])
        if dist is None:
            assert got == V - 1
            continue
        p, bound = dist
        w, slack = p, bound
        if kept < d:
            if q is not None:
                take = q[r, kept].double().cpu()
            else:
                take = torch.zeros(V, dtype=torch.float64)
                if 0 <= int(drafted[r, kept]) < V:
                    take[int(drafted[r, kept])] = 1.0
            rest = torch.where(p > take, p - take, 0.0)
            if float(rest.sum()) > float(bound.sum()):
                w, slack = rest, torch.where(p + bound > take, bound, 0.0) + rest * 2.0 ** -24
            else:               # what is left is within the rounding of p: either reading
                continue
        total, slack = float(w.sum()), float(slack.sum()) * 2
        cum = w.cumsum(0)
        before = float(cum[got - 1]) if got else 0.0
        v = draw[r]
        if v != v or v >= 1:
            assert float(w[got + 1:].sum()) <= slack, (r, got)      # the last token of some weight
        else:
            assert before - slack <= max(v, 0.0) * total <= float(cum[got]) + slack, (r, got, before, v * total, float(cum[got]))
        assert float(w[got]) + slack > 0


def inputs(seed, R, D, V, dtype, mixed=True, masked=False, probs=True, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    counts = torch.randint(0, D + 1, (R,), generator=g, dtype=torch.int32)
    if R:
        counts[0] = D
    order = torch.randperm(R, generator=g)                     # requests' rows lie in any order, with rows of nobody between
    row_start = torch.zeros(R, dtype=torch.int32)
    at = 1
    for r in order.tolist():
        row_start[r] = at
        at += int(counts[r]) + 2
    logits = (torch.randn(at, V, generator=g) * scale).to(dt(dtype))
    if masked:
        logits[torch.rand(at, V, generator=g) < 0.5] = -math.inf
        logits[torch.rand(at, V, generator=g) < 0.1] = torch.finfo(dt(dtype)).min
        logits[:, V // 2] = 1.0
    t = 0.5 + torch.rand(R, generator=g)
    if mixed:
        t[torch.rand(R, generator=g) < 0.3] = 0.0
    rows = (row_start[:, None] + torch.arange(D)[None, :]).clamp(max=at - 1).long()
    z = logits[rows].float() / t.clamp(min=0.3)[:, None, None] + 0.5 * torch.randn(R, D, V, generator=g)
    q = torch.softmax(z, -1) if D else torch.zeros(R, 0, V)
    drafted = torch.multinomial(q.reshape(-1, V), 1, generator=g).reshape(R, D).int() if D else torch.zeros(R, 0, dtype=torch.int32)
    greedy = (t == 0)[:, None] & (torch.rand(R, D, generator=g) < 0.8)
    best = torch.tensor([[argmax_of(logits[rows[r, j]].float()) for j in range(D)] for r in range(R)], dtype=torch.int32).reshape(R, D)
    drafted = torch.where(greedy, best, drafted)
    return logits, row_start, drafted, counts, q if probs else None, t, torch.rand(R, D, generator=g), torch.rand(R, generator=g)


def verify(logits, row_start, drafted, counts, q, t, accept, draw):
    R, D = drafted.shape
    tokens = torch.full((R, D + 1), 77, dtype=torch.int32, device=DEV)
    accepted = torch.full((R,), 77, dtype=torch.int32, device=DEV)
    work = torch.full((logits.shape[0], 4), float("nan"), device=DEV)
    d = [None if x is None else x if x.is_cuda else x.to(DEV) for x in (logits, row_start, drafted, counts, q, t, accept, draw)]
    K().verify_drafts(*d, tokens, accepted, work)
    return tokens, accepted


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("R,D,V,masked,probs", [(1, 0, 1, False, True), (1, 1, 1, False, False), (3, 2, 2, False, True), (9, 3, 7, False, True),
                                                (40, 4, 33, True, True), (40, 4, 33, False, False), (17, 5, 1001, True, False), (12, 2, 4099, False, True),
                                                (6, 8, 8190, False, True), (5, 3, 16387, True, True), (4, 4, 50257, True, False), (3, 3, 128256, False, True),
                                                (2, 2, 151669, True, True), (2, 2, 200003, False, True)])
def test_verification_follows_the_formulas(dtype, R, D, V, masked, probs):
    args = inputs(7 * V + D, R, D, V, dtype, masked=masked, probs=probs)
    tokens, accepted = verify(*args)
    check_verification(*args, tokens, accepted)


@pytest.mark.parametrize("dtype,R,D,V,masked,probs", [("float32", 110, 4, 70001, False, True), ("bfloat16", 130, 5, 66000, True, False),
                                                      ("float32", 400, 3, 6003, False, True)])
def test_more_rows_than_the_gpu_holds_at_a_time(dtype, R, D, V, masked, probs):
    """Rows behind a refusal may be left out, in clusters of two and in blocks of a row each: the answers are the same, in every run."""
    args = inputs(V, R, D, V, dtype, masked=masked, probs=probs)
    tokens, accepted = verify(*args)
    check_verification(*args, tokens, accepted)
    for _ in range(3):
        again = verify(*args)
        assert torch.equal(again[0], tokens) and torch.equal(again[1], accepted)


@pytest.mark.parametrize("dtype,V,masked,probs", [("float32", 12001, False, True), ("bfloat16", 16381, True, False), ("float32", 20003, True, True),
                                                  ("bfloat16", 20480, False, True)])
def test_many_rows_that_one_block_holds(dtype, V, masked, probs):
    args = inputs(V, 160, 3, V, dtype, masked=masked, probs=probs)
    tokens, accepted = verify(*args)
    check_verification(*args, tokens, accepted)


def test_every_count_of_kept_drafts_comes_up():
    args = inputs(3, 300, 4, 50, "float32")
    tokens, accepted = verify(*args)
    check_verification(*args, tokens, accepted)
    assert set(accepted.tolist()) == {0, 1, 2, 3, 4}


@pytest.mark.parametrize("probs", [True, False])
def test_rows_without_a_distribution_and_equal_logits(probs):
    logits, row_start, drafted, counts, q, t, accept, draw = inputs(5, 8, 3, 100, "float32", mixed=False, probs=probs)
    counts[:] = 3
    row_start = torch.arange(8, dtype=torch.int32) * 4
    logits = torch.randn(32, 100, generator=torch.Generator().manual_seed(1))
    accept[:] = 0.0                                  # every draft of some probability is kept
    logits[0] = -math.inf                            # request 0: nothing at all in its first row
    logits[5, 17] = math.nan                         # request 1: its second row
    logits[10, 3] = math.inf                         # request 2: its third
    logits[15] = -math.inf                           # request 3: the row behind its drafts
    logits[16:20] = 2.5                              # request 4: all equal
    t[5:] = 0.0                                      # 5 to 7 greedy
    logits[20:24] = 1.0                              # ties
    drafted[5] = torch.tensor([0, 0, 1])             # kept, kept, refused: token 0 is the lowest of equals
    logits[24] = math.nan
    drafted[6, 0] = 0                                # nothing but no numbers: token 0
    logits[28] = -math.inf
    logits[29, 40] = math.inf
    drafted[7] = torch.tensor([0, 40, 100])          # (the last one outside the vocabulary)
    args = (logits, row_start, drafted, counts, q, t, accept, draw)
    tokens, accepted = verify(*args)
    assert accepted[:4].tolist() == [0, 1, 2, 3] and accepted[5:].tolist() == [2, 3 if argmax_of(logits[25]) == int(drafted[6, 1]) else 1, 2]
    assert tokens[0, 0] == 99 and tokens[1, 1] == 99 and tokens[2, 2] == 99 and tokens[3, 3] == 99 and tokens[5, 2] == 0
    check_verification(*args, tokens, accepted)


def test_random_numbers_at_the_ends_and_beyond():
    logits, row_start, drafted, counts, q, t, accept, draw = inputs(6, 12, 2, 5000, "float32", mixed=False, masked=True)
    accept[:, 0] = 0.0
    accept[:, 1] = 2.0                               # never kept
    for r, v in enumerate((0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan, 0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -1.0, math.nan)):
        draw[r] = v
    counts[6:] = 1
    drafted[0, 0] = -1                               # outside the vocabulary: refused
    drafted[6, 0] = 5000
    args = (logits, row_start, drafted, counts, q, t, accept, draw)
    tokens, accepted = verify(*args)
    assert accepted[0] == 0 and accepted[6] == 0
    check_verification(*args, tokens, accepted)


def test_where_the_target_is_the_draft_the_draw_is_from_the_target():
    """p = q to the bit: nothing is left behind q, and a refused draft (u >= 1) is replaced by a draw from p."""
    g = torch.Generator().manual_seed(8)
    logits = torch.randn(40, 3000, generator=g)
    t = torch.ones(20)
    q = torch.empty(40, 3000, device=DEV)
    K().token_probabilities(logits.to(DEV), torch.ones(40, device=DEV), q)
    row_start = torch.arange(20, dtype=torch.int32) * 2
    q = q.view(20, 2, 3000)[:, :1]
    draw = torch.rand(20, generator=g)
    args = (logits, row_start, torch.zeros(20, 1, dtype=torch.int32), torch.ones(20, dtype=torch.int32), q, t, torch.full((20, 1), 1.0), draw)
    tokens, accepted = verify(*args)
    assert accepted.tolist() == [0] * 20
    free = (logits[::2].contiguous(), torch.arange(20, dtype=torch.int32), torch.zeros(20, 0, dtype=torch.int32), torch.zeros(20, dtype=torch.int32), None, t,
            torch.zeros(20, 0), draw)
    assert torch.equal(verify(*free)[0][:, 0], tokens[:, 0])


def test_a_draw_without_drafts_is_the_samplers():
    g = torch.Generator().manual_seed(9)
    logits = (torch.randn(30, 32003, generator=g) * 3).to(DEV)
    t, u = (0.5 + torch.rand(30, generator=g)).to(DEV), torch.rand(30, generator=g).to(DEV)
    want = torch.empty(30, dtype=torch.int32, device=DEV)
    K().sample(logits, torch.empty(30, 32003, device=DEV), t, torch.zeros(30, dtype=torch.int32, device=DEV), torch.ones(30, device=DEV), u, want)
    tokens, _ = verify(logits, torch.arange(30, dtype=torch.int32), torch.zeros(30, 0, dtype=torch.int32), torch.zeros(30, dtype=torch.int32), None, t,
                       torch.zeros(30, 0), u)
    assert torch.equal(tokens[:, 0], want)


def test_drafts_and_target_together_follow_the_target():
    """20,000 requests of one row pair: the token after the prompt is distributed as the target has it, whatever the drafter's
    distribution. Six standard deviations of a count."""
    n, V = 20000, 8
    g = torch.Generator().manual_seed(10)
    row, other = torch.randn(V, generator=g) * 1.5, torch.randn(V, generator=g) * 1.5
    q = torch.softmax(other, 0)
    drafted = torch.multinomial(q.expand(n, V), 1, generator=g).int()
    tokens, accepted = verify(row.expand(2 * n, V).contiguous(), torch.arange(n, dtype=torch.int32) * 2, drafted, torch.ones(n, dtype=torch.int32),
                              q.to(DEV).expand(n, 1, V), torch.ones(n), torch.rand(n, 1, generator=g), torch.rand(n, generator=g))
    p = torch.softmax(row.double(), 0)
    seen = torch.bincount(tokens[:, 0].cpu().long(), minlength=V).double()
    assert bool(((seen - n * p).abs() <= 6 * (n * p * (1 - p)).sqrt()).all())
    keep = float(torch.minimum(p, q.double()).sum())
    assert abs(float((accepted == 1).sum()) - n * keep) <= 6 * math.sqrt(n * keep * (1 - keep))


def test_strides_of_the_drafters_probabilities_offsets_streams_and_programs():
    logits, row_start, drafted, counts, q, t, accept, draw = inputs(11, 10, 3, 1003, "float32")
    want = verify(logits, row_start, drafted, counts, q, t, accept, draw)
    by_step = torch.empty(3, 12, 1010)                       # as a drafter fills it: a step at a time, padded rows
    by_step[:, 1:11, 2:1005] = q.transpose(0, 1)
    view = by_step.to(DEV).transpose(0, 1)[1:11, :, 2:1005]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    odd = torch.empty(logits.numel() + 3, device=DEV)[3:].view(logits.shape)     # rows off 16 bytes
    odd.copy_(logits)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = verify(odd, row_start, drafted, counts, view, t, accept, draw)
    side.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    d = [x.to(DEV) for x in (logits, row_start, drafted, counts, q, t, accept, draw)]
    tokens, accepted = torch.zeros_like(want[0]), torch.zeros_like(want[1])
    work = torch.empty(logits.shape[0], 4, device=DEV)
    with K().record() as rec:
        K().verify_drafts(*d, tokens, accepted, work)
    tokens.zero_()
    rec.program.run()
    assert torch.equal(tokens, want[0]) and len(rec.program) == 1 and rec.program.launches == 2


def test_requests_whose_rows_do_not_lie_in_the_logits():
    logits, row_start, drafted, counts, q, t, accept, draw = inputs(12, 4, 2, 64, "float32", mixed=False)
    row_start[1], row_start[2] = -1, logits.shape[0] - 1
    counts[2], counts[3] = 2, 9                               # (more than D drafts: D)
    row_start[3] = 1
    tokens, accepted = verify(logits, row_start, drafted, counts, q, t, accept, draw)
    assert accepted[1] == -1 and accepted[2] == -1 and (tokens[1:3] == -1).all()
    keep = [0, 3]
    counts[3] = 2
    check_verification(logits, row_start[keep], drafted[keep], counts[keep], q[keep], t[keep], accept[keep], draw[keep], tokens[keep], accepted[keep])


def test_verification_refuses_what_does_not_fit():
    logits, row_start, drafted, counts, q, t, accept, draw = (None if x is None else x.to(DEV) for x in inputs(13, 3, 2, 40, "float32"))
    tokens, accepted = torch.zeros(3, 3, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)
    work = torch.zeros(logits.shape[0], 4, device=DEV)
    good = dict(logits=logits, row_start=row_start, drafted=drafted, counts=counts, draft_probs=q, temperature=t, accept_uniform=accept,
                draw_uniform=draw, tokens=tokens, accepted=accepted, work=work)
    K().verify_drafts(**good)
    for name, value in (("logits", logits.half()), ("logits", logits.cpu()), ("logits", logits[:, ::2]), ("row_start", row_start.long()),
                        ("row_start", row_start[:2]), ("drafted", drafted[:, :1]), ("counts", counts[:1]), ("draft_probs", q[:, :, :39]),
                        ("draft_probs", q.double()), ("draft_probs", q.cpu()), ("draft_probs", q.transpose(1, 2).contiguous().transpose(1, 2)),
                        ("temperature", t.double()), ("accept_uniform", accept[:, :1]), ("draw_uniform", draw[:2]), ("tokens", tokens[:, :2]),
                        ("accepted", accepted.long()), ("work", work[:2]), ("work", torch.zeros(4 * logits.shape[0] + 1, device=DEV)[1:])):
        with pytest.raises(K().KernelError):
            K().verify_drafts(**dict(good, **{name: value}))
    empty = {k: v[:0] if k not in ("logits", "work") else v for k, v in good.items()}
    K().verify_drafts(**empty)                                # no requests: nothing to do
    torch.cuda.synchronize()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,V", [(1, 1), (2, 3), (5, 130), (33, 1001), (3, 4100), (4, 8193), (3, 32003), (9, 50257), (2, 128256), (3, 151669), (2, 163840), (2, 200003)])
def test_token_probabilities(dtype, rows, V):
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(rows, V, generator=g) * 4).to(dt(dtype))
    logits[torch.rand(rows, V, generator=g) < 0.2] = -math.inf
    logits[:, V // 3] = 2.0
    t = 0.3 + torch.rand(rows, generator=g)
    t[rows // 2] = 0.0 if rows > 1 else t[0]
    out = torch.full((rows, V), float("nan"), device=DEV)
    K().token_probabilities(logits.to(DEV), t.to(DEV), out)
    out = out.cpu()
    for r in range(rows):
        if t[r] > 0:
            p, bound = distribution(logits[r].float(), float(t[r]))
            assert bool(((out[r].double() - p).abs() <= bound).all()), r
        else:
            want = torch.zeros(V)
            want[argmax_of(logits[r].float())] = 1.0
            assert torch.equal(out[r], want)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("rows,V", [(310, 5113), (620, 8191), (600, 12001), (640, 16380), (601, 20475), (310, 20481), (150, 32003), (320, 40959),
                                    (160, 50257), (170, 81917), (76, 128256), (77, 163837), (40, 200003)])
def test_token_probabilities_of_many_rows(dtype, rows, V):
    """Blocks of a row, clusters of two to eight, each size of block: rows against the formula, all of them against calls of a few rows (whose sum
    may round the other way: two 32-bit roundings of a value)."""
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(rows, V, generator=g) * 4).to(dt(dtype)).to(DEV)
    logits[:, V // 2:V // 2 + 9] = -math.inf
    logits[rows // 2] = -math.inf
    t = (0.3 + torch.rand(rows, generator=g)).to(DEV)
    t[rows - 1] = 0.0
    out = torch.full((rows, V), float("nan"), device=DEV)
    K().token_probabilities(logits, t, out)
    for r in (0, 1, rows - 2):
        p, bound = distribution(logits[r].float().cpu(), float(t[r]))
        assert bool(((out[r].double().cpu() - p).abs() <= bound).all()), r
    assert torch.isnan(out[rows // 2]).all()
    few = torch.empty_like(out)
    for r in range(0, rows, 5):
        K().token_probabilities(logits[r:r + 5], t[r:r + 5], few[r:r + 5])
    torch.testing.assert_close(out, few, rtol=2.0 ** -21, atol=2.0 ** -126, equal_nan=True)


def test_token_probabilities_of_rows_without_any_and_of_extreme_temperatures():
    logits = torch.randn(7, 77, generator=torch.Generator().manual_seed(3))
    logits[0] = -math.inf
    logits[1, 5] = math.nan
    logits[2, 76] = math.inf
    logits[3, :] = -3e38
    logits[3, 9] = 3e38
    t = torch.tensor([1.0, 1.0, 1.0, 1.0, 1e-30, 1e30, -1.0])
    out = torch.zeros(7, 77, device=DEV)
    K().token_probabilities(logits.to(DEV), t.to(DEV), out)
    out = out.cpu()
    assert torch.isnan(out[:3]).all()
    for r in (3, 4, 6):
        want = torch.zeros(77)
        want[int(logits[r].argmax())] = 1.0
        assert torch.equal(out[r], want), r
    assert bool(((out[5] - 1 / 77).abs() <= 2.0 ** -23 * 4 / 77).all())


def test_token_probabilities_refuses_what_does_not_fit():
    x, t = torch.zeros(2, 8, device=DEV), torch.ones(2, device=DEV)
    for logits, temp, out in ((x.half(), t, x), (x, t[:1], x), (x, t, x[:1]), (x, t.double(), x), (x, t, x.bfloat16()), (x.cpu(), t, x)):
        with pytest.raises(K().KernelError):
            K().token_probabilities(logits, temp, out)
    K().token_probabilities(x[:0], t[:0], x[:0])


def test_the_quotient_by_the_temperature_is_the_divisions():
    """Two million quotients over 500 temperatures: to the bit what the general division and exp give."""
    g = torch.Generator(device=DEV).manual_seed(4)
    rows, V = 500, 4001
    t = torch.exp(torch.randn(rows, generator=g, device=DEV))
    logits = torch.randn(rows, V, generator=g, device=DEV) * torch.exp(torch.randn(rows, 1, generator=g, device=DEV))
    out = torch.empty(rows, V, device=DEV)
    K().token_probabilities(logits, t, out)
    e = torch.exp((logits - logits.amax(1, keepdim=True)) / t[:, None])
    assert torch.equal(out, e * (1.0 / e.double().sum(1, keepdim=True)).float())


@pytest.mark.parametrize("dtype,R,D,V", [("float32", 600, 3, 6003), ("bfloat16", 150, 4, 70001), ("float32", 40, 15, 128256)])
def test_requests_that_share_rows_end(dtype, R, D, V):
    """A shared row's results are either request's, but every call ends, with tokens of the vocabulary. Rows may be left out here: each cluster decides it for itself."""
    logits, row_start, drafted, counts, q, t, accept, draw = inputs(V, R, D, V, dtype, probs=False)
    counts[:] = D
    row_start = torch.arange(R, dtype=torch.int32) % 3
    logits = logits[:D + 4].contiguous()
    for _ in range(3):
        tokens, accepted = verify(logits, row_start, drafted, counts, None, t, accept, draw)
        assert bool(((tokens >= -1) & (tokens < V)).all()) and bool(((accepted >= 0) & (accepted <= D)).all())


@pytest.mark.parametrize("R,V", [(1, 7), (3, 1000), (400, 33), (5, 50257), (700, 5001), (2, 151669), (100, 70001)])
def test_an_infinite_temperature_is_the_even_distribution(R, V):
    """exp((l - m) / inf) = 1 for every finite logit, as the sampler has it; -infinity over infinity is no number, and then neither is any."""
    g = torch.Generator().manual_seed(V)
    logits = (torch.randn(R, V, generator=g) * 3).to(DEV)
    t = torch.full((R,), math.inf, device=DEV)
    out = torch.empty(R, V, device=DEV)
    K().token_probabilities(logits, t, out)
    assert torch.equal(out, torch.full_like(out, float(torch.tensor(1.0 / V))))
    # drafts: a third of the mass is what a draft of probability 1 / V is kept from; the draw's place is that of the running sum
    start = torch.arange(R, dtype=torch.int32, device=DEV)
    none = torch.zeros(R, 0, dtype=torch.int32, device=DEV)
    draw = ((torch.arange(R) + 0.5) / R).to(DEV)
    tokens, accepted = verify(logits, start, none, torch.zeros_like(start), None, t, torch.zeros(R, 0, device=DEV), draw)
    want = (draw.double() * V).floor().int()
    assert bool(((tokens[:, 0] - want).abs() <= 1).all()) and not accepted.any()
    scratch, ids = torch.empty_like(logits), torch.zeros(R, dtype=torch.int32, device=DEV)
    K().sample(logits, scratch, t, torch.zeros_like(ids), torch.ones(R, device=DEV), draw, ids)
    assert torch.equal(ids, tokens[:, 0])
    if R > 1 and V > 1:
        logits[1, V // 2] = -math.inf
        K().token_probabilities(logits, t, out)
        assert torch.isnan(out[1]).all() and torch.equal(out[0], torch.full_like(out[0], float(torch.tensor(1.0 / V))))
        assert int(verify(logits, start, none, torch.zeros_like(start), None, t, torch.zeros(R, 0, device=DEV), draw)[0][1, 0]) == V - 1
