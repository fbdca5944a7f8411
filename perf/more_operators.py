"""Timing cases of the operators that complete a serving step: the page plan of a batch (block tables and
slots from request lengths), low-rank adapters beside a shared projection, the gated activation that ends in
8 bits with scales, and the sampling of the next tokens from their logits.

``listed()`` and ``draw()`` give the cases, ``prepare()`` what a serving program holds before the call,
``run()`` one pass (the plain torch form, or the package's operator where ``own`` is true), ``work()`` the
bytes and operations that no implementation can do without, and ``exact()`` the result in 64 bits.
"""

from __future__ import annotations

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
MIN_FP32_SCALE = 2.0 ** -149
LEAST_WEIGHT = 2.0 ** -126  # a token whose weight is below this part of the largest has none


# ------------------------------------------------------------------------------------------------ cases
def listed() -> list[dict]:
    return [
        # One decode step of 64 sequences, most of whose last pages have room: latency.
        dict(name="plan-step-64", op="plan", mode="step", batch=64, tokens=64, ctx=8192, page=64),
        # The prompts of a dozen requests beside running ones that get a token each, ragged, small pages.
        dict(name="plan-prompts-33001", op="plan", mode="prompts", batch=157, tokens=33001, ctx=4001, page=16),
        # A batch of 2048 requests is finished; its pages go back and a batch of prompts takes them.
        dict(name="plan-turnover-131072", op="plan", mode="turnover", batch=2048, tokens=131072, ctx=512, page=32),
        # One token of one request beside a fused projection: latency.
        dict(name="adapt-1x4096x6144", op="adapt", tokens=1, k=4096, n=6144, rank=16, adapters=8, mix="each", x="bf16",
             y="fp32", out="bf16"),
        # A decode step of 64 requests, nearly each with an adapter of its own.
        dict(name="adapt-64x4096x4096", op="adapt", tokens=64, k=4096, n=4096, rank=32, adapters=64, mix="each",
             x="bf16", y="fp32", out="bf16"),
        # A prefill batch of ragged prompts; the adapter reads the norm's 8-bit operand, as the projection does.
        dict(name="adapt-8192x4096x12288", op="adapt", tokens=8192, k=4096, n=12288, rank=16, adapters=6, mix="runs",
             x="fp8_row", y="fp32", out="bf16"),
        # A pruned layer whose widths no vector size divides, fp16 throughout.
        dict(name="adapt-777x2045x1030", op="adapt", tokens=777, k=2045, n=1030, rank=12, adapters=5, mix="runs",
             x="fp16", y="fp16", out="fp16"),
        # A prefill batch's gate and up halves of one fp32 projection into MXFP8: bandwidth.
        dict(name="gated-8192x12288", op="gated", rows=8192, k=12288, dtype="fp32", scheme="mxfp8_e4m3", act="silu"),
        # An odd width, 16-bit halves, one scale a row.
        dict(name="gated-333x1537", op="gated", rows=333, k=1537, dtype="bf16", scheme="fp8_row", act="gelu_tanh"),
        # The next token of one request over a large vocabulary: latency.
        dict(name="sample-1x131072", op="sample", rows=1, vocab=131072, dtype="bf16", mix="k_p"),
        # A large batch, nucleus sampling over an odd vocabulary in fp32: bandwidth.
        dict(name="sample-256x150001", op="sample", rows=256, vocab=150001, dtype="fp32", mix="p"),
        # Requests with settings of their own: greedy ones, top-k, top-p, min-p, banned tokens.
        dict(name="sample-64x32000", op="sample", rows=64, vocab=32000, dtype="fp16", mix="all"),
    ]


def _log(rng: random.Random, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng: random.Random) -> dict:
    op = rng.choice(("plan", "adapt", "adapt", "gated", "sample", "sample"))
    if op == "plan":
        batch, page = _log(rng, 1, 2048), rng.choice((8, 16, 32, 64, 128, 256))
        mode = rng.choice(("step", "prompts", "turnover"))
        tokens = batch if mode == "step" else _log(rng, batch + 1, 131072)
        return dict(op=op, mode=mode, batch=batch, tokens=tokens, ctx=_log(rng, 16, 16384 if batch < 300 else 2048),
                    page=page)
    if op == "adapt":
        k, n, rank = _log(rng, 64, 8192), _log(rng, 64, 16384), rng.choice((4, 8, 16, 16, 24, 32, 64))
        if rng.random() < 0.7:
            k, n, rank = max(64, k // 64 * 64), max(64, n // 64 * 64), max(8, rank)
        x = rng.choice(("bf16", "fp16", "fp8_row", "int8_row"))
        out = rng.choice(("bf16", "fp32")) if x.endswith("row") else x
        return dict(op=op, tokens=_log(rng, 1, max(1, min(8192, (1 << 26) // max(k, n)))), k=k, n=n, rank=rank,
                    adapters=_log(rng, 1, 48), mix=rng.choice(("each", "runs", "one")), x=x,
                    y=rng.choice(("fp32", out)), out=out)
    if op == "gated":
        k = _log(rng, 64, 16384)
        if rng.random() < 0.6:
            k = max(64, k // 64 * 64)
        return dict(op=op, rows=_log(rng, 1, max(1, min(8192, (1 << 26) // k))), k=k,
                    dtype=rng.choice(("bf16", "fp16", "fp32")),
                    scheme=rng.choice(("fp8_row", "int8_row", "mxfp8_e4m3", "fp8_group128")),
                    act=rng.choice(("silu", "gelu", "gelu_tanh", "relu")))
    vocab = _log(rng, 1000, 200000)
    return dict(op=op, rows=_log(rng, 1, max(1, min(256, (1 << 25) // vocab))), vocab=vocab,
                dtype=rng.choice(("bf16", "fp16", "fp32")), mix=rng.choice(("none", "k", "p", "k_p", "min_p", "all")))


# ------------------------------------------------------------------------------------------------ inputs
def _heavy(shape, g, scale: float = 1.0):
    """Normal values with one channel in 64 eight times larger, as activations have."""
    x = torch.randn(shape, generator=g, device="cuda") * scale
    hot = torch.randperm(shape[-1], generator=g, device="cuda")[: max(1, shape[-1] // 64)]
    x[..., hot] *= 8
    return x


def _lengths(case: dict) -> tuple[list[int], list[int], int]:
    """Every sequence's tokens in the cache and new ones, and the pages of a table row: the sizes are the
    case's, the same for every seed."""
    b, tokens, ctx, page = case["batch"], case["tokens"], case["ctx"], case["page"]
    rng = random.Random(1000003 * b + 1009 * tokens + ctx)
    if case["mode"] == "step":  # a few rows of the batch are idle
        have = [rng.randint(1, ctx) for _ in range(b)]
        new = [0 if i and rng.random() < 0.05 else 1 for i in range(b)]
    elif case["mode"] == "prompts":  # prompts, running requests, idle rows
        kind = [rng.choice((0, 1, 1, 1, 2)) for _ in range(b)]
        kind[0] = 2
        prompts = kind.count(2)
        rest = tokens - kind.count(1)
        cuts = sorted(rng.randint(0, rest) for _ in range(prompts - 1))
        sizes = [hi - lo for lo, hi in zip([0] + cuts, cuts + [rest])]
        have = [rng.randint(1, ctx) if t == 1 else 0 for t in kind]
        new = [1 if t == 1 else sizes.pop() if t == 2 else 0 for t in kind]
    else:
        cuts = sorted(rng.randint(0, tokens) for _ in range(b - 1))
        new = [hi - lo for lo, hi in zip([0] + cuts, cuts + [tokens])]
        have = [0] * b
    most = max(h + n for h, n in zip(have, new)) + ctx // 4
    return have, new, -(-most // page) + 1


def _prepare_plan(case, g):
    have, new, width = _lengths(case)
    page = case["page"]
    used, after = [-(-h // page) for h in have], [-(-(h + n) // page) for h, n in zip(have, new)]
    spare = 5 + sum(after) // 16
    pages = sum(after) + spare
    free = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    held = after if case["mode"] == "turnover" else used  # what the rows hold before the call
    h = torch.tensor(held, device="cuda")
    col = torch.arange(width, device="cuda")
    first = h.cumsum(0) - h
    table = torch.where(col < h[:, None], free[(first[:, None] + col).clamp(max=pages - 1)], -1)
    as32 = dict(dtype=torch.int32, device="cuda")
    return dict(table=table.to(torch.int32), free=free, taken=torch.tensor([sum(held)], **as32),
                lens=torch.tensor(have, **as32), new=torch.tensor(new, **as32),
                ended=torch.ones(case["batch"], dtype=torch.bool, device="cuda"))


def _index(case, g):
    """The adapter of each token: a request's tokens follow one another, some requests have none."""
    t, a = case["tokens"], case["adapters"]
    if case["mix"] == "each":
        who = torch.randperm(max(t, a), generator=g, device="cuda")[:t] % a
        return torch.where(torch.rand(t, generator=g, device="cuda") < 0.05, -1, who).to(torch.int32)
    if case["mix"] == "one":
        return torch.full((t,), a // 2, dtype=torch.int32, device="cuda")
    starts = torch.rand(t, generator=g, device="cuda") < 12 / max(t, 24)
    owner = torch.randint(-1, a, (t + 1,), generator=g, device="cuda")
    return owner[starts.cumsum(0)].to(torch.int32)


def _prepare_adapt(case, g):
    t, k, n, r, a = (case[i] for i in ("tokens", "k", "n", "rank", "adapters"))
    x = _heavy((t, k), g)
    st = {}
    if case["x"].endswith("row"):
        top = 448.0 if case["x"] == "fp8_row" else 127.0
        s = _row_scale(x.abs().amax(-1, keepdim=True), top)
        st["x"] = (x / s).to(torch.float8_e4m3fn) if top == 448.0 else (x / s).round().clamp(-127, 127).to(torch.int8)
        st["xs"] = s
        weights = torch.bfloat16
    else:
        weights = DTYPES[case["x"]]
        st["x"], st["xs"] = x.to(weights), None
    st["a"] = (torch.randn((a, r, k), generator=g, device="cuda") * k ** -0.5).to(weights)
    st["b"] = (torch.randn((a, n, r), generator=g, device="cuda") * 0.1).to(weights)
    st["gain"] = 0.5 + torch.rand(a, generator=g, device="cuda")
    st["y"] = torch.randn((t, n), generator=g, device="cuda").to(DTYPES[case["y"]])
    st["index"] = _index(case, g)
    return st


def _prepare_gated(case, g):
    both = _heavy((case["rows"], 2 * case["k"]), g, 1.5).to(DTYPES[case["dtype"]])
    return dict(gate=both[:, :case["k"]], up=both[:, case["k"]:])


def _prepare_sample(case, g):
    rows, vocab, mix = case["rows"], case["vocab"], case["mix"]
    logits = torch.randn((rows, vocab), generator=g, device="cuda") * 2.5
    hot = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")  # what the context makes likely
    logits.scatter_add_(1, hot, 4 + 5 * torch.rand((rows, 24), generator=g, device="cuda"))

    def choose(*of):
        return torch.tensor(of, device="cuda")[torch.randint(0, len(of), (rows,), generator=g, device="cuda")]

    st = dict(temperature=choose(0.7, 0.8, 1.0, 1.2), top_k=None, top_p=None, min_p=None)
    if mix in ("k", "k_p"):
        st["top_k"] = choose(20, 50, 100).to(torch.int32)
    if mix in ("p", "k_p"):
        st["top_p"] = choose(0.8, 0.9, 0.95)
    if mix == "min_p":
        st["min_p"] = choose(0.02, 0.05, 0.1)
    if mix == "all":
        st["temperature"] = choose(0.0, 0.6, 1.0, 1.5)
        st["top_k"] = choose(0, 1, 40, 5000).to(torch.int32)
        st["top_p"] = choose(1.0, 0.5, 0.9, 0.99)
        st["min_p"] = choose(0.0, 0.0, 0.03)
        logits[torch.rand((rows, vocab), generator=g, device="cuda") < 0.1] = float("-inf")  # banned by a grammar
    st["logits"] = logits.to(DTYPES[case["dtype"]])
    st["uniform"] = torch.rand(rows, generator=g, device="cuda")
    return st


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = {"plan": _prepare_plan, "adapt": _prepare_adapt, "gated": _prepare_gated, "sample": _prepare_sample}
    return {"case": case, **make[case["op"]](case, g)}


# ------------------------------------------------------------------------------------------------ one pass
def run(st: dict):
    op = st["case"]["op"]
    if own:
        return {"plan": _own_plan, "adapt": _own_adapt, "gated": _own_gated, "sample": _own_sample}[op](st)
    return {"plan": _run_plan, "adapt": _run_adapt, "gated": _run_gated, "sample": _run_sample}[op](st)


def _own_plan(st):
    from tricast_b200 import plan_pages, release_pages

    case, taken = st["case"], st["taken"]
    if case["mode"] == "turnover":
        taken = release_pages(st["table"], st["ended"], st["free"], taken)
    plan = plan_pages(st["lens"], st["new"], st["table"], st["free"], taken, page_size=case["page"],
                      tokens=case["tokens"])
    return [st["table"], plan.seq_lens, plan.cu_q, plan.slots, plan.sequence, plan.positions, plan.taken, plan.missing]


def _own_adapt(st):
    from tricast_b200 import QTensor, get_scheme, low_rank_add

    case, x = st["case"], st["x"]
    if st["xs"] is not None:
        x = QTensor(x, st["xs"], None, None, get_scheme(case["x"]), tuple(x.shape))
    return low_rank_add(st["y"], x, st["a"], st["b"], st["index"], gain=st["gain"], dtype=DTYPES[case["out"]])


def _own_gated(st):
    from tricast_b200 import gated_quantize

    q = gated_quantize(st["gate"], st["up"], st["case"]["scheme"], activation=st["case"]["act"])
    return [_value(q.values), _value(q.scale)]


def _own_sample(st):
    from tricast_b200 import sample_tokens

    return list(sample_tokens(st["logits"], st["uniform"], temperature=st["temperature"], top_k=st["top_k"],
                              top_p=st["top_p"], min_p=st["min_p"], return_logprobs=True))


def _run_plan(st):
    case, table, free, lens = st["case"], st["table"], st["free"], st["lens"].long()
    page, tokens, taken = case["page"], case["tokens"], st["taken"].long()
    batch, width = table.shape
    if case["mode"] == "turnover":
        back = (table >= 0) & st["ended"][:, None]
        rank = back.flatten().long().cumsum(0) - 1
        taken = taken - back.sum()
        at = torch.where(back.flatten(), taken + rank, free.numel())
        free.copy_(torch.cat((free, free[:1])).scatter_(0, at, table.flatten())[:-1])
        table.copy_(torch.where(st["ended"][:, None], -1, table))
    new = st["new"].long().clamp(min=0)
    start = (new.cumsum(0) - new).clamp(max=tokens)
    new = torch.minimum(new, tokens - start)
    used = (lens + page - 1) // page
    wanted = (lens + new + page - 1) // page - used
    need = torch.minimum(wanted, (width - used).clamp(min=0))
    first = taken + need.cumsum(0) - need
    col = torch.arange(width, device=table.device)
    at = first[:, None] + col - used[:, None]
    fresh = (col >= used[:, None]) & (col < (used + need)[:, None])
    picked = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(fresh, picked, table))
    cu = torch.cat((start, (start[-1:] + new[-1:])))
    t = torch.arange(tokens, device=table.device)
    seq = torch.searchsorted(cu[1:].contiguous(), t, right=True)
    real = seq < batch
    s = seq.clamp(max=batch - 1)
    pos = lens[s] + t - cu[s]
    held = torch.where(pos // page < width, table[s, (pos // page).clamp(max=width - 1)].long(), -1)
    slots = torch.where(real & (held >= 0), held * page + pos % page, -1)
    total = taken + need.sum()
    after = total.clamp(max=free.numel())
    missing = total - after + (wanted - need).sum()
    return [table, (lens + new).to(torch.int32), cu.to(torch.int32), slots, torch.where(real, seq, -1).to(torch.int32),
            torch.where(real, pos, -1).to(torch.int32), after.to(torch.int32), missing.to(torch.int32)]


def _run_adapt(st):
    """Every adapter's down projection in one product, of which each token keeps its own."""
    case, index = st["case"], st["index"].long()
    a, r, _ = st["a"].shape
    x = st["x"].float()
    h = (x @ st["a"].float().flatten(0, 1).T).unflatten(1, (a, r))
    if st["xs"] is not None:
        h = h * st["xs"][:, :, None]
    mine = index[:, None] == torch.arange(a, device=index.device)
    h = torch.where(mine[:, :, None], h * st["gain"][:, None], 0.0)
    up = st["b"].float().permute(0, 2, 1).flatten(0, 1)
    return (st["y"].float() + h.flatten(1) @ up).to(DTYPES[case["out"]])


def _act(v, name: str):
    if name == "silu":
        return v / (1 + torch.exp(-v))
    if name == "relu":
        return v.clamp(min=0)
    if name == "gelu":
        return 0.5 * v * (1 + torch.erf(v * math.sqrt(0.5)))
    return 0.5 * v * (1 + torch.tanh(math.sqrt(2 / math.pi) * (v + 0.044715 * v * v * v)))


def _row_scale(amax, top: float):
    s = amax / torch.full_like(amax, top)  # by a tensor: torch multiplies by a scalar's reciprocal instead
    s = torch.where(s == 0, MIN_FP32_SCALE, s)
    return torch.where(amax == 0, 1.0, s)


def _pow2_scale(amax, top: int):
    """2**(floor(log2 amax) - top), clamped to E8M0; an all-zero group counts as amax 2**-126."""
    _, e = torch.frexp(torch.where(amax == 0, 2.0 ** -126, amax))
    return torch.ldexp(torch.ones_like(amax), (e - 1 - top).clamp(-127, 127))


def _value(t):
    """What codes and E8M0 scales stand for."""
    return t.float() if t.dtype in (torch.int8, torch.float8_e8m0fnu) else t


def _run_gated(st):
    case = st["case"]
    y = _act(st["gate"].float(), case["act"]) * st["up"].float()
    k, scheme = y.shape[1], case["scheme"]
    n = {"mxfp8_e4m3": 32, "fp8_group128": 128}.get(scheme, k)
    g = torch.nn.functional.pad(y, (0, -k % n)).unflatten(-1, (-1, n))
    amax = g.abs().amax(-1)
    s = _pow2_scale(amax, 8) if n == 32 else _row_scale(amax, 127.0 if scheme == "int8_row" else 448.0)
    v = (g / s[..., None]).flatten(-2)[:, :k]
    if scheme == "int8_row":
        return [v.round().clamp(-127, 127), s]
    return [v.clamp(-448.0, 448.0).to(torch.float8_e4m3fn), s]


def _run_sample(st):
    z = st["logits"].double()
    rows, vocab = z.shape
    u = st["uniform"].double()[:, None]
    heat = st["temperature"].double()[:, None]
    z, order = torch.sort(z, dim=1, descending=True, stable=True)
    w = torch.exp((z - z[:, :1]) / torch.where(heat > 0, heat, 1.0))
    w = torch.where(w < LEAST_WEIGHT, 0.0, w)
    rank = torch.arange(vocab, device=z.device)
    keep = w > 0
    if st["top_k"] is not None:
        k = st["top_k"].long()[:, None]
        keep &= (rank < k) | (k <= 0)
    if st["top_p"] is not None:
        p = st["top_p"].double()[:, None]
        mass = torch.where(keep, w, 0.0)
        upto = mass.cumsum(1)
        keep &= (upto - mass < p * upto[:, -1:]) | (rank == 0) | (p >= 1)
    if st["min_p"] is not None:
        keep &= w >= st["min_p"].double()[:, None]
    keep &= (heat > 0) | (rank == 0)
    mass = torch.zeros_like(w).scatter_(1, order, torch.where(keep, w, 0.0))
    upto = mass.cumsum(1)
    total = upto[:, -1:]
    token = (upto <= u * total).sum(1, keepdim=True)
    last = torch.where(mass > 0, rank, 0).amax(1, keepdim=True)
    token = torch.minimum(token, last)
    return [token.squeeze(1), torch.log(mass.gather(1, token) / total).squeeze(1).float()]


# ------------------------------------------------------------------------------------------------ work
def work(case: dict) -> dict:
    if case["op"] == "plan":
        have, new, width = _lengths(case)
        page = case["page"]
        fresh = sum(-(-(h + n) // page) - -(-h // page) for h, n in zip(have, new))
        moved = 16 * case["tokens"] + 8 * fresh + 16 * case["batch"]
        return {"bytes": moved + (8 * fresh if case["mode"] == "turnover" else 0), "flops": 4 * case["tokens"]}
    if case["op"] == "adapt":
        t, k, n, r = (case[i] for i in ("tokens", "k", "n", "rank"))
        held = min(t, 1 if case["mix"] == "one" else case["adapters"]) * r * (k + n) * 2
        x = t * (k + 4) if case["x"].endswith("row") else t * k * 2
        return {"bytes": x + held + t * n * (DTYPES[case["y"]].itemsize + DTYPES[case["out"]].itemsize) + 4 * t,
                "flops": 2 * t * r * (k + n)}
    if case["op"] == "gated":
        n = case["rows"] * case["k"]
        scales = {"mxfp8_e4m3": case["rows"] * -(-case["k"] // 32),
                  "fp8_group128": 4 * case["rows"] * -(-case["k"] // 128)}.get(case["scheme"], 4 * case["rows"])
        return {"bytes": n * (2 * DTYPES[case["dtype"]].itemsize + 1) + scales, "flops": 12 * n}
    n = case["rows"] * case["vocab"]
    return {"bytes": n * DTYPES[case["dtype"]].itemsize + 32 * case["rows"], "flops": 12 * n}


# ------------------------------------------------------------------------------------------------ 64 bits
def exact(case: dict, seed: int):
    if case["op"] == "plan":
        return None  # whole numbers
    st = prepare(case, seed)
    return {"adapt": _exact_adapt, "gated": _exact_gated, "sample": _exact_sample}[case["op"]](case, st)


def _exact_adapt(case, st):
    """One adapter after the other, over the tokens that it has."""
    out = st["y"].double()
    x = st["x"].double()
    if st["xs"] is not None:
        x = x * st["xs"].double()
    for i in range(case["adapters"]):
        mine = (st["index"] == i).nonzero().squeeze(1)
        if mine.numel():
            down = torch.einsum("tk,rk->tr", x[mine], st["a"][i].double())
            out[mine] += st["gain"][i].double() * torch.einsum("tr,nr->tn", down, st["b"][i].double())
    return out


def _grid64(v):
    """Nearest E4M3 value, ties to even, saturating, in fp64."""
    _, e = torch.frexp(v)
    step = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return ((v / step).round() * step).clamp(-448.0, 448.0)


def _exact_gated(case, st):
    """The activations from their definitions: the logistic function, the normal distribution, a tanh of exponentials."""
    codes, scales = [], []
    for lo in range(0, case["rows"], 1024):
        g, up = st["gate"][lo:lo + 1024].double(), st["up"][lo:lo + 1024].double()
        if case["act"] == "silu":
            a = g * torch.special.expit(g)
        elif case["act"] == "gelu":
            a = g * torch.special.ndtr(g)
        elif case["act"] == "relu":
            a = torch.maximum(g, torch.zeros_like(g))
        else:
            a = g * torch.special.expit(2 * math.sqrt(2 / math.pi) * (g + 0.044715 * g ** 3))
        y = a * up
        width = {"mxfp8_e4m3": 32, "fp8_group128": 128}.get(case["scheme"], case["k"])
        parts = y.split(width, dim=1)
        top = torch.stack([p.abs().amax(1) for p in parts], 1)
        if case["scheme"] == "mxfp8_e4m3":
            m, _ = torch.frexp(top)  # top / 2m: the largest power of two that is not above it
            s = top / (2 * m) / 2.0 ** 8
        else:
            s = top / (127.0 if case["scheme"] == "int8_row" else 448.0)
        v = torch.cat([p / s[:, i:i + 1] for i, p in enumerate(parts)], 1)
        codes.append(v.round().clamp(-127, 127) if case["scheme"] == "int8_row" else _grid64(v))
        scales.append(s)
    return [torch.cat(codes), torch.cat(scales)]


def _exact_sample(case, st):
    """One row after the other: the log-probability of the token that its random number falls on."""
    got = []
    for i in range(case["rows"]):
        z = st["logits"][i].double()
        heat = float(st["temperature"][i])
        if heat == 0:
            got.append(0.0)
            continue
        p = (z / heat - (z / heat).max()).exp()
        p[p < LEAST_WEIGHT] = 0.0
        by = torch.argsort(z, descending=True, stable=True)
        by = by[p[by] > 0]
        if st["top_k"] is not None and int(st["top_k"][i]) > 0:
            by = by[:int(st["top_k"][i])]
        if st["top_p"] is not None and float(st["top_p"][i]) < 1:
            short = p[by].cumsum(0) < float(st["top_p"][i]) * p[by].sum()
            by = by[:int(short.sum()) + 1]
        if st["min_p"] is not None:
            by = by[p[by] >= float(st["min_p"][i])]
        ids = by.sort().values
        upto = p[ids].cumsum(0)
        j = min(int(torch.searchsorted(upto, float(st["uniform"][i]) * upto[-1:], right=True)), ids.numel() - 1)
        got.append(math.log(float(p[ids[j]] / upto[-1])))
    return [None, torch.tensor(got, dtype=torch.float64, device="cuda")]
