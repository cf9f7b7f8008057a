"""Timed cases of the operators that a server with drafted tokens and per-request adapters runs beside the model.

Four operators of one serving loop: the step's tables built on the device from the requests' lengths, low-rank adapters of
many requests added to a shared projection, the drafter's probabilities, and the verification of its drafts. Every one has a plain
form here, of elementary torch operations. What is a token id or a page number at the end is decided by sums in 64 bits (as this
repository's sampler has them): it must not depend on the order of a summation. Everything else is computed in 32 bits.
"""
import math

import torch

own = False          # False: the plain forms; True: this repository's kernels

DEV = "cuda:0"
VOCAB = 128256       # of the benchmark's shapes


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    verify = {"op": "verify", "dtype": "float32", "probs": True, "masked": False, "mixed": False}
    tables = {"op": "tables", "page": 16}
    adapt = {"op": "adapter", "dtype": "bfloat16", "out": "float32", "order": "rows", "without": 0.0}
    return [
        # one user, four drafted tokens a round: latency
        dict(verify, name="verify_one_user", requests=1, drafts=4, vocab=VOCAB),
        # drafts looked up in the prompt (no probabilities), a few requests, a masked vocabulary of an odd size in 16 bits
        dict(verify, name="verify_lookup", requests=16, drafts=7, vocab=50257, dtype="bfloat16", probs=False, masked=True),
        # a full batch with a draft model, ragged drafts, greedy requests among the sampled ones
        dict(verify, name="verify_batch", requests=128, drafts=6, vocab=VOCAB, mixed=True),
        # the drafter's rows of one drafted token of a small batch
        {"op": "probabilities", "name": "probabilities_few", "rows": 8, "vocab": VOCAB, "dtype": "float32", "mixed": False},
        # every row of a large batch, an odd vocabulary, greedy rows among them
        {"op": "probabilities", "name": "probabilities_many", "rows": 512, "vocab": 151669, "dtype": "float32", "mixed": True},
        # a small server's round: a row for the last token and one for each of four drafts
        dict(tables, name="tables_small", requests=16, new=5, context=8192),
        # a large server's step: portions of prompts beside single tokens
        dict(tables, name="tables_large", requests=1024, new=128, context=8192),
        # eight requests, a token and an adapter each, at the attention's output projection of the 1B shape
        dict(adapt, name="adapter_decode", rows=8, K=2048, slices="2048", rank=16, adapters=8),
        # a round of drafts: 51 requests of five rows on 24 adapters, gate and up of the 1B shape, some requests without an adapter
        dict(adapt, name="adapter_drafts", rows=255, K=2048, slices="8192,8192", rank=32, adapters=24, order="requests", without=0.2),
        # the true 32-bit path: a portion of a prompt for each of three requests, an odd rank
        dict(adapt, name="adapter_float32", rows=700, K=2048, slices="2048", rank=12, adapters=3, dtype="float32", order="prompts"),
        # a prompt step into [q; k; v] of the 8B shape: four prompts, four adapters
        dict(adapt, name="adapter_prompts", rows=2048, K=4096, slices="4096,1024,1024", rank=16, adapters=4, order="prompts"),
        # the down projection of the 8B shape for a large step, a high rank
        dict(adapt, name="adapter_large", rows=8192, K=14336, slices="4096", rank=64, adapters=8, out="bfloat16", order="prompts"),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["verify", "verify", "probabilities", "tables", "adapter", "adapter", "adapter"])
    if op == "verify":
        vocab, drafts = _log(rng, 1000, 152000), rng.randint(1, 8)
        return {"op": op, "requests": _log(rng, 1, max(1, min(256, 110_000_000 // (vocab * (drafts + 1))))), "drafts": drafts, "vocab": vocab,
                "dtype": rng.choice(["float32", "float32", "bfloat16"]), "probs": rng.random() < 0.7,
                "masked": rng.random() < 0.3, "mixed": rng.random() < 0.5}
    if op == "probabilities":
        vocab = _log(rng, 1000, 152000)
        return {"op": op, "rows": _log(rng, 1, max(1, min(1024, 77_000_000 // vocab))), "vocab": vocab,
                "dtype": rng.choice(["float32", "float32", "bfloat16"]), "mixed": rng.random() < 0.5}
    if op == "tables":
        return {"op": op, "requests": _log(rng, 1, 1024), "new": _log(rng, 1, 128), "context": _log(rng, 64, 8192), "page": rng.choice([8, 16, 32, 64])}
    K, widths = rng.choice([(2048, "2048"), (2048, "8192,8192"), (8192, "2048"), (4096, "4096,1024,1024"), (4096, "4096"),
                            (14336, "4096"), (2056, "1000,520")])
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    most = min(8192, 350_000_000 // (2 * K + 8 * sum(int(v) for v in widths.split(","))))
    return {"op": op, "dtype": dtype, "out": "float32" if dtype == "float32" else rng.choice(["float32", "bfloat16"]),
            "rows": _log(rng, 1, most if dtype == "bfloat16" else min(most, 2048)), "K": K, "slices": widths,
            "rank": rng.choice([4, 8, 12, 16, 24, 32, 64]), "adapters": _log(rng, 1, 16),
            "order": rng.choice(["rows", "requests", "prompts"]), "without": rng.choice([0.0, 0.3])}


# ---------------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    return {"verify": _prepare_verify, "probabilities": _prepare_probabilities, "tables": _prepare_tables, "adapter": _prepare_adapter}[case["op"]](case, g)


def _dtype(name):
    return {"float32": torch.float32, "bfloat16": torch.bfloat16}[name]


def _rand(g, *shape):
    return torch.rand(*shape, generator=g, device=DEV)


def _logits(g, rows, vocab):
    """Logits as a language model has them: a broad bulk and a few dozen likely tokens a row."""
    x = torch.randn(rows, vocab, generator=g, device=DEV) * 2.0
    if rows:
        likely = torch.randint(0, vocab, (rows, 40), generator=g, device=DEV)
        x.scatter_add_(1, likely, torch.randn(rows, 40, generator=g, device=DEV).abs() * 4.0 + 4.0)
    return x


def _temperatures(g, n, mixed):
    t = 0.6 + 0.6 * _rand(g, n)
    return torch.where(_rand(g, n) < 0.3, torch.zeros_like(t), t) if mixed else t


def _prepare_verify(case, g):
    R, D, V = case["requests"], case["drafts"], case["vocab"]
    counts = torch.full((R,), D, dtype=torch.int32, device=DEV)
    if R > 1:                                       # a drafter stops early where it is unsure
        counts = torch.where(_rand(g, R) < 0.4, torch.randint(0, D + 1, (R,), generator=g, device=DEV, dtype=torch.int32), counts)
    ends = (counts + 1).cumsum(0)
    N = int(ends[-1])
    row_start = (ends - counts - 1).to(torch.int32)
    logits = _logits(g, N, V)
    if case["masked"]:
        logits[logits < 1.0] = -math.inf
    temperature = _temperatures(g, R, case["mixed"])
    # the drafter sees almost the same distribution: most of its tokens are accepted
    place = torch.arange(D, device=DEV)
    rows = (row_start[:, None] + torch.minimum(place[None, :], counts[:, None].clamp(min=1) - 1)).long()
    probs = torch.empty(R, D, V, device=DEV) if case["probs"] else None
    drafted = torch.empty(R, D, dtype=torch.int32, device=DEV)
    for j in range(D):
        z = (logits[rows[:, j]] + 0.7 * torch.randn(R, V, generator=g, device=DEV)) / temperature.clamp(min=0.3)[:, None]
        if probs is not None:
            probs[:, j] = torch.softmax(z, dim=1)
        drafted[:, j] = (z - torch.log(-torch.log(_rand(g, R, V).clamp(1e-9, 1 - 1e-6)))).argmax(1).to(torch.int32)
    return {"op": "verify", "logits": logits.to(_dtype(case["dtype"])), "row_start": row_start, "counts": counts, "drafted": drafted,
            "probs": probs, "temperature": temperature, "accept": _rand(g, R, D), "draw": _rand(g, R),
            "tokens": torch.empty(R, D + 1, dtype=torch.int32, device=DEV), "accepted": torch.empty(R, dtype=torch.int32, device=DEV),
            "work": torch.empty(N, 4, device=DEV)}


def _prepare_probabilities(case, g):
    rows, V = case["rows"], case["vocab"]
    return {"op": "probabilities", "logits": _logits(g, rows, V).to(_dtype(case["dtype"])), "temperature": _temperatures(g, rows, case["mixed"]),
            "out": torch.empty(rows, V, device=DEV)}


def _prepare_tables(case, g):
    R, most, page = case["requests"], case["new"], case["page"]
    def whole(low, high):
        return torch.randint(low, high, (R,), generator=g, device=DEV, dtype=torch.int32)
    lengths = whole(0, case["context"] + 1)
    counts = torch.where(_rand(g, R) < 0.5, whole(0, most + 1), torch.full_like(lengths, min(most, 5)))
    kept = (counts * _rand(g, R)).to(torch.int32)                       # what stays of them after the verification
    held = (lengths + page - 1) // page
    stride = (case["context"] + most + page - 1) // page
    pool = R * (stride + 1)
    order = torch.randperm(pool, generator=g, device=DEV).to(torch.int32)
    place = torch.arange(stride, device=DEV)[None, :]
    first = (held.cumsum(0) - held)[:, None]
    tables = torch.where(place < held[:, None], order[(first + place).clamp(max=pool - 1)], -1).to(torch.int32)
    free = torch.full((pool,), -1, dtype=torch.int32, device=DEV)
    n_free = pool - int(held.sum())
    free[:n_free] = order[pool - n_free:]      # (the first ones are held)
    def ints(*shape):
        return torch.empty(*shape, dtype=torch.int32, device=DEV)
    return {"op": "tables", "lengths": lengths, "counts": counts, "after": lengths + kept, "tables": tables.contiguous(), "held": held, "free": free,
            "n_free": torch.tensor([n_free], dtype=torch.int32, device=DEV), "page": page, "row_start": ints(R + 1), "row_req": ints(R * most),
            "positions": ints(R * most), "slots": ints(R * most), "status": ints(1)}


def _prepare_adapter(case, g):
    T, K, r, A = case["rows"], case["K"], case["rank"], case["adapters"]
    widths = [int(v) for v in case["slices"].split(",")]
    S, N, dtype = len(widths), sum(widths), _dtype(case["dtype"])
    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)
    if case["order"] == "rows":                     # single tokens: a request a row
        row_adapter = torch.randint(0, A, (T,), generator=g, device=DEV)
        if T == A:
            row_adapter = torch.randperm(A, generator=g, device=DEV)
    else:                                           # five rows a request, or a prompt for every adapter
        run = 5 if case["order"] == "requests" else -(-T // A)
        row_adapter = torch.randint(0, A, (-(-T // run),), generator=g, device=DEV)
        if case["order"] == "prompts":
            row_adapter = torch.randperm(A, generator=g, device=DEV)[:row_adapter.numel()]
        row_adapter = torch.where(_rand(g, row_adapter.numel()) < case["without"], -1, row_adapter).repeat_interleave(run)[:T]
    return {"op": "adapter", "x": normal(T, K).to(dtype), "down": (normal(A, S * r, K) / math.sqrt(K)).to(dtype), "up": (normal(A, N, r) / math.sqrt(r)).to(dtype),
            "scales": 0.5 + _rand(g, A), "row_adapter": row_adapter.to(torch.int32).contiguous(), "widths": widths,
            "out": normal(T, N).to(_dtype(case["out"]))}


# ---------------------------------------------------------------------------------------------------- one pass
def run(state):
    if own:
        return _own(state)
    return {"verify": _plain_verify, "probabilities": _plain_probabilities, "tables": _plain_tables, "adapter": _plain_adapter}[state["op"]](state)


def _own(s):
    from geneinfer_b200.ops import kernels
    if s["op"] == "verify":
        kernels.verify_drafts(s["logits"], s["row_start"], s["drafted"], s["counts"], s["probs"], s["temperature"], s["accept"], s["draw"],
                              s["tokens"], s["accepted"], s["work"])
        return {"tokens": s["tokens"], "accepted": s["accepted"]}
    if s["op"] == "probabilities":
        kernels.token_probabilities(s["logits"], s["temperature"], s["out"])
        return {"probabilities": s["out"]}
    if s["op"] == "tables":                          # a round: places for the new tokens, then back to what was kept of them
        kernels.step_tables(s["lengths"], s["counts"], s["tables"], s["held"], s["free"], s["n_free"], s["page"], s["row_start"], s["row_req"],
                            s["positions"], s["slots"], s["status"])
        kernels.trim_tables(s["after"], s["tables"], s["held"], s["free"], s["n_free"], s["page"], s["status"])
        return _tables_out(s)
    plan = kernels.adapter_plan(s["row_adapter"], s["down"].shape[0])
    kernels.adapter_product(s["x"], s["down"], s["up"], s["scales"], plan, s["out"], s["widths"])
    return {"out": s["out"]}


def _softmax(z, temperature):
    """exp((z - max) / T) over its sum, which is taken in 64 bits."""
    e = torch.exp((z - z.amax(1, keepdim=True)) / temperature[:, None])
    return e * (1.0 / e.double().sum(1, keepdim=True)).float()


def _one_hot(index, vocab):
    return (torch.arange(vocab, device=index.device)[None, :] == index[:, None]).float()


def _plain_probabilities(s):
    z, t = s["logits"].float(), s["temperature"]
    p = _softmax(z, torch.where(t > 0, t, 1.0))
    return {"probabilities": torch.where(t[:, None] > 0, p, _one_hot(z.argmax(1), z.shape[1]))}


def _plain_verify(s):
    z, start, counts, drafted, t = s["logits"].float(), s["row_start"].long(), s["counts"].long(), s["drafted"].long(), s["temperature"]
    R, D = drafted.shape
    N, V = z.shape
    sampled = t > 0
    safe = torch.where(sampled, t, 1.0)
    place = torch.arange(D, device=z.device)[None, :]
    rows = (start[:, None] + place).clamp(max=N - 1)
    row_req = torch.searchsorted(start, torch.arange(N, device=z.device), right=True) - 1
    p = _softmax(z, safe[row_req])
    best = z.argmax(1)
    # how many drafts every request keeps
    q_at = s["probs"].gather(2, drafted[:, :, None])[:, :, 0] if s["probs"] is not None else torch.ones_like(s["accept"])
    good = torch.where(sampled[:, None], s["accept"] * q_at < p[rows, drafted], drafted == best[rows])
    accepted = (good & (place < counts[:, None])).long().cumprod(1).sum(1)
    stop = start + accepted
    # the token behind them
    w = p[stop]
    refused = (accepted < counts) & sampled
    if D:
        at = accepted.clamp(max=D - 1)
        own_token = drafted.gather(1, at[:, None])[:, 0]
        q = s["probs"][torch.arange(R, device=z.device), at] if s["probs"] is not None else _one_hot(own_token, V)
        rest = torch.where(w > q, w - q, 0.0)
        w = torch.where(refused[:, None] & (rest.amax(1, keepdim=True) > 0), rest, w)
    cum = w.double().cumsum(1)
    over = (cum > s["draw"].double()[:, None] * cum[:, -1:]) & (w > 0)
    token = torch.where(sampled, over.byte().argmax(1), best[stop])
    wide = torch.arange(D + 1, device=z.device)[None, :]
    tokens = torch.where(wide < accepted[:, None], torch.cat([drafted, drafted.new_zeros(R, 1)], 1), -1)
    tokens = torch.where(wide == accepted[:, None], token[:, None], tokens)
    return {"tokens": tokens.int(), "accepted": accepted.int()}


def _settle(lengths, s):
    """Pages back to the stack and from it until every request holds what ``lengths`` positions need."""
    tables, held, free, n, page = s["tables"], s["held"], s["free"], s["n_free"], s["page"]
    need = (lengths + page - 1) // page
    place = torch.arange(tables.shape[1], device=tables.device)[None, :]
    back = (held - need).clamp(min=0)
    take = (need - held).clamp(min=0)
    giving = (place >= need[:, None]) & (place < held[:, None])
    taking = (place >= held[:, None]) & (place < need[:, None])
    total_back = back.sum()
    # given back from the last request's last page on: the place on the stack counts what lies behind
    behind = (total_back - back.cumsum(0))[:, None] + (held[:, None] - 1 - place)
    pool = free.numel()
    stack = torch.cat([free, free.new_zeros(1)])
    stack = stack.scatter(0, torch.where(giving, n + behind, pool).clamp(max=pool).flatten().long(), tables.flatten())
    order = (take.cumsum(0) - take)[:, None] + (place - held[:, None])
    page_of = stack[(n + total_back - 1 - order).clamp(0, pool).long()]
    tables.copy_(torch.where(taking, page_of, torch.where(giving, -1, tables)))
    free.copy_(stack[:pool])
    n.copy_(n + total_back - take.sum())
    held.copy_(need)


def _plain_tables(s):
    lengths, counts, page = s["lengths"], s["counts"], s["page"]
    _settle(lengths + counts, s)
    ends = counts.cumsum(0)
    row = torch.arange(s["row_req"].numel(), device=ends.device)
    req = torch.searchsorted(ends, row, right=True).clamp(max=ends.numel() - 1)
    some = row < ends[-1]
    positions = lengths[req] + row - (ends - counts)[req]
    at = torch.where(some, positions // page, 0).clamp(max=s["tables"].shape[1] - 1)
    s["row_start"].copy_(torch.cat([ends.new_zeros(1), ends]))
    s["row_req"].copy_(torch.where(some, req, -1))
    s["positions"].copy_(torch.where(some, positions, 0))
    s["slots"].copy_(torch.where(some, s["tables"][req, at] * page + positions % page, -1))
    _settle(s["after"], s)
    s["status"].zero_()
    return _tables_out(s)


def _tables_out(s):
    return {k: s[k] for k in ("row_start", "row_req", "positions", "slots", "tables", "held", "free", "n_free", "status")}


def _plain_adapter(s):
    x, down, up, out = s["x"].float(), s["down"].float(), s["up"].float(), s["out"]
    A, N, r = up.shape
    T, K = x.shape
    S = down.shape[1] // r
    h = (x @ down.reshape(A * S * r, K).T).reshape(T, A, S, r)
    own_adapter = torch.arange(A, device=x.device)[None, :] == s["row_adapter"][:, None]
    h = torch.where(own_adapter[:, :, None, None], h * s["scales"][None, :, None, None], 0.0)
    parts = [h[:, :, i].reshape(T, A * r) @ u.transpose(1, 2).reshape(A * r, -1) for i, u in enumerate(up.split(s["widths"], dim=1))]
    out.copy_(out.float() + torch.cat(parts, 1))
    return {"out": out}


# ---------------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = {"float32": 4, "bfloat16": 2}
    if case["op"] == "verify":
        R, D, V = case["requests"], case["drafts"], case["vocab"]
        rows = R * (1 + (D if R == 1 else 0.8 * D))                     # four in ten requests bring half of the drafts
        return {"bytes": rows * V * size[case["dtype"]] + (R * V * 4 if case["probs"] else 0) + R * (8 * D + 20), "flops": 10 * rows * V}
    if case["op"] == "probabilities":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * (size[case["dtype"]] + 4), "flops": 5 * n}
    if case["op"] == "tables":
        R, rows = case["requests"], case["requests"] * case["new"]
        return {"bytes": 12 * rows + 24 * R + 8 * rows / case["page"], "flops": 10 * rows}
    T, K, r = case["rows"], case["K"], case["rank"]
    widths = [int(v) for v in case["slices"].split(",")]
    S, N = len(widths), sum(widths)
    share = 1.0 - case["without"]
    used = min(case["adapters"], T)
    b = size[case["dtype"]]
    return {"bytes": share * T * (K * b + 2 * N * size[case["out"]]) + used * r * (S * K + N) * b + 4 * T, "flops": share * 2.0 * T * r * (S * K + N)}


# ---------------------------------------------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    """Token ids and tables are whole numbers: they have to be equal, and no 64-bit value says more."""
    if case["op"] not in ("probabilities", "adapter"):
        return None
    s = prepare(case, seed)
    if case["op"] == "probabilities":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEV)
        for i, t in enumerate(s["temperature"].tolist()):
            z = s["logits"][i].double()
            if t > 0:
                e = torch.exp((z - z.max()) / t)
                out[i] = e / e.sum()
            else:
                out[i, int((z == z.max()).nonzero()[0])] = 1.0
        return {"probabilities": out}
    out = s["out"].double()
    r = s["up"].shape[2]
    for a in range(s["up"].shape[0]):
        rows = (s["row_adapter"] == a).nonzero()[:, 0]
        h = s["x"][rows].double() @ s["down"][a].double().T * s["scales"][a].double()
        at = 0
        for i, n in enumerate(s["widths"]):
            out[rows, at:at + n] += h[:, i * r:(i + 1) * r] @ s["up"][a, at:at + n].double().T
            at += n
    return {"out": out}
