"""Cases for three operators of a serving step, their plain forms and their exact values.

  attention  decode attention for streams that share a long prefix (a voice prompt, a system prompt): one new token per
             stream over a paged bf16 cache, the first pages of a group's tables being the same pages
  linear     projections with 8-bit integer weights: activations quantised per token row, weights per output channel
  sample     temperature, top-k, top-p, min-p and the draw, from given uniform numbers

`own` chooses between the plain form (elementary torch operations) and the calls a user makes of the library.
"""
import functools
import importlib
import math

import torch

own = False

HEAD = 128          # head dimension and page size of the library's paged cache
PAGE = 64
EPSILON = 1.0e-6


def listed():
    return [
        # four requests of one voice right after their prompts: the smallest batch that shares anything
        {"name": "attention few streams", "op": "attention", "batch": 4, "groups": 1, "shared": 16, "suffix": 40, "kv_heads": 8, "idle": False},
        # a full batch behind one voice prompt, ragged replies
        {"name": "attention one voice", "op": "attention", "batch": 64, "groups": 1, "shared": 32, "suffix": 1024, "kv_heads": 8, "idle": False},
        # several voices at once, prefixes of different lengths, some slots idle
        {"name": "attention five voices", "op": "attention", "batch": 83, "groups": 5, "shared": 67, "suffix": 517, "kv_heads": 8, "idle": True},
        # a document-sized prefix
        {"name": "attention long prefix", "op": "attention", "batch": 32, "groups": 1, "shared": 512, "suffix": 1024, "kv_heads": 8, "idle": False},
        # one token through one projection: latency
        {"name": "linear one token", "op": "linear", "kind": "linear", "rows": 1, "inner": 2048, "outer": 2048, "norm": True, "bias": True, "residual": False},
        # a decode batch through the down projection with its residual
        {"name": "linear decode down", "op": "linear", "kind": "linear", "rows": 32, "inner": 6144, "outer": 2048, "norm": False, "bias": False, "residual": True},
        # a decode batch through the normalised gated feed-forward input
        {"name": "linear decode gated", "op": "linear", "kind": "gated", "rows": 61, "inner": 2048, "outer": 6144, "norm": True, "bias": False, "residual": False},
        # packed prompts through one projection
        {"name": "linear prompt rows", "op": "linear", "kind": "linear", "rows": 9923, "inner": 2048, "outer": 6144, "norm": False, "bias": True, "residual": False},
        # one stream's next code
        {"name": "sample one code", "op": "sample", "batch": 1, "vocab": 2048, "dtype": "bfloat16", "mix": "top_k", "spread": 3.0},
        # a batch of codes, every row with parameters of its own
        {"name": "sample code batch", "op": "sample", "batch": 64, "vocab": 2048, "dtype": "float32", "mix": "all", "spread": 2.0},
        # a text-sized vocabulary
        {"name": "sample words", "op": "sample", "batch": 32, "vocab": 131072, "dtype": "float32", "mix": "all", "spread": 2.5},
        # an odd vocabulary in bf16, where many scores are equal
        {"name": "sample odd words", "op": "sample", "batch": 96, "vocab": 100003, "dtype": "bfloat16", "mix": "nucleus", "spread": 2.0},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["attention", "linear", "sample"])
    if op == "attention":
        batch = _spread(rng, 1, 128)
        shared = _spread(rng, 1, 512)
        suffix = _spread(rng, 1, 1024)
        while batch * (shared * PAGE + suffix) > 32 * (512 * PAGE + 1024):
            shared = max(1, shared // 2)
        return {"op": op, "batch": batch, "groups": min(batch, _spread(rng, 1, 8)), "shared": shared, "suffix": suffix,
                "kv_heads": rng.choice([2, 4, 8, 8]), "idle": rng.random() < 0.5}
    if op == "linear":
        rows = _spread(rng, 1, 9923)
        inner, outer = 16 * _spread(rng, 16, 384), 8 * _spread(rng, 16, 768)
        while rows * inner * outer > 9923 * 2048 * 6144:
            rows = max(1, rows // 2)
        kind = rng.choice(["linear", "linear", "gated"])
        if kind == "gated" and 2 * rows * inner * outer > 9923 * 2048 * 6144:
            rows = max(1, rows // 2)
        plain = kind == "linear"
        return {"op": op, "kind": kind, "rows": rows, "inner": inner, "outer": outer, "norm": rng.random() < 0.5,
                "bias": plain and rng.random() < 0.5, "residual": plain and rng.random() < 0.5}
    vocab, batch = _spread(rng, 40, 200000), _spread(rng, 1, 128)
    while vocab * batch > 96 * 100003:
        batch = max(1, batch // 2)
    return {"op": op, "batch": batch, "vocab": vocab, "dtype": rng.choice(["bfloat16", "float32"]),
            "mix": rng.choice(["all", "top_k", "nucleus", "open"]), "spread": round(rng.uniform(1.0, 4.0), 2)}


@functools.lru_cache(maxsize=None)
def _package():
    return importlib.import_module("qingming-qwen3-tts_b200")


@functools.lru_cache(maxsize=None)
def _engine():
    """The handle that a program keeps for the calls that need no cache of their own."""
    return _package().TalkerAttention(layers=1, num_pages=1, max_positions=64)


# ---- inputs

def _layout(case, seed):
    """Whole numbers on the host: streams of each group, shared pages of each group, keys of each stream, page table."""
    gen = torch.Generator().manual_seed(seed)
    batch, groups = case["batch"], case["groups"]
    cuts = torch.randperm(batch - 1, generator=gen)[: groups - 1].sort().values + 1 if groups > 1 else torch.zeros(0, dtype=torch.int64)
    starts = torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([batch])])
    shared = torch.randint(max(1, case["shared"] // 4), case["shared"] + 1, (groups,), generator=gen)
    shared[int(torch.randint(0, groups, (1,), generator=gen))] = case["shared"]
    of = torch.bucketize(torch.arange(batch), starts[1:], right=True)
    lens = shared[of] * PAGE + torch.randint(1, case["suffix"] + 1, (batch,), generator=gen)
    if case["idle"]:
        idle = torch.rand(batch, generator=gen) < 0.1
        idle[0] = False
        lens[idle] = 0
    own_pages = (case["suffix"] + PAGE - 1) // PAGE
    max_pages = int(shared.max()) + own_pages
    first = torch.cat([torch.zeros(1, dtype=torch.int64), shared.cumsum(0)])
    pages = int(first[-1]) + batch * own_pages
    names = torch.randperm(pages, generator=gen)
    column = torch.arange(max_pages)[None, :]
    behind = column - shared[of][:, None]
    table = torch.where(behind < 0, first[of][:, None] + column,
                        first[-1] + torch.arange(batch)[:, None] * own_pages + behind.clamp(0, own_pages - 1))
    return starts, shared, lens, names[table], pages


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.bfloat16, scale=1.0):
        return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)

    if case["op"] == "attention":
        starts, shared, lens, table, pages = _layout(case, seed)
        heads = case["kv_heads"]
        q, k, v = normal(case["batch"], 2 * heads, HEAD), normal(pages, heads, PAGE, HEAD), normal(pages, heads, PAGE, HEAD)
        state = {"op": "attention", "q": q, "starts": starts.int().cuda(), "shared": shared.int().cuda(), "lens": lens.int().cuda(),
                 "table": table.int().cuda(), "max_shared": int(shared.max()), "k": k, "v": v}
        if own:      # the user's cache is the library's page pool
            state["engine"] = _package().TalkerAttention(layers=1, num_pages=pages, q_heads=2 * heads, kv_heads=heads, max_positions=64)
            key, value = state["engine"].pool_view(0)
            key.copy_(k)
            value.copy_(v)
            del state["k"], state["v"]
        return state
    if case["op"] == "linear":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        # activations have a few channels far larger than the rest
        x = (torch.randn((rows, inner), generator=gen, device="cuda") *
             torch.exp(0.5 * torch.randn((inner,), generator=gen, device="cuda"))).to(torch.bfloat16)
        state = {"op": "linear", "kind": case["kind"], "x": x, "norm": None, "bias": None, "residual": None}
        names = ("w",) if case["kind"] == "linear" else ("gate", "up")
        for name in names:       # weights quantised beforehand, one scale for each output channel
            state[name] = torch.randint(-127, 128, (outer, inner), generator=gen, device="cuda", dtype=torch.int8)
            state[name + "_scale"] = torch.rand((outer,), generator=gen, device="cuda") * (2.0 / (127 * math.sqrt(inner))) + 1e-6
        if case["norm"]:
            state["norm"] = normal(inner, scale=0.2) + 1
        if case["bias"]:
            state["bias"] = normal(outer, scale=0.5)
        if case["residual"]:
            state["residual"] = normal(rows, outer)
        return state
    batch, mix = case["batch"], case["mix"]
    logits = normal(batch, case["vocab"], dtype=getattr(torch, case["dtype"]), scale=case["spread"])

    def rand(low, high):
        return torch.rand((batch,), generator=gen, device="cuda") * (high - low) + low

    def some(share):
        return torch.rand((batch,), generator=gen, device="cuda") < share

    temperature = rand(0.6, 1.2)
    top_k = torch.randint(1, 101, (batch,), generator=gen, device="cuda", dtype=torch.int32)
    top_p, min_p = rand(0.7, 1.0), rand(0.0, 0.1)
    if mix == "top_k":
        top_p, min_p = torch.ones_like(top_p), torch.zeros_like(min_p)
    elif mix == "nucleus":
        top_k, min_p = torch.zeros_like(top_k), torch.zeros_like(min_p)
    elif mix == "open":
        top_k, top_p, min_p = torch.zeros_like(top_k), torch.ones_like(top_p), torch.zeros_like(min_p)
    else:       # requests of every kind in one batch, greedy ones among them
        temperature = torch.where(some(0.1), torch.zeros_like(temperature), temperature)
        top_k = torch.where(some(0.4), torch.zeros_like(top_k), top_k)
        top_p = torch.where(some(0.4), torch.ones_like(top_p), top_p)
        min_p = torch.where(some(0.5), torch.zeros_like(min_p), min_p)
    return {"op": "sample", "logits": logits, "temperature": temperature, "top_k": top_k, "top_p": top_p, "min_p": min_p,
            "uniform": torch.rand((batch,), generator=gen, device="cuda")}


# ---- one pass

def _plain_attention(s):
    batch, q_heads, _ = s["q"].shape
    keys = s["k"].shape[1]
    length = s["table"].shape[1] * PAGE
    k = s["k"][s["table"].long()].float().transpose(1, 2).reshape(batch, keys, length, HEAD)
    v = s["v"][s["table"].long()].float().transpose(1, 2).reshape(batch, keys, length, HEAD)
    q = s["q"].float().reshape(batch, keys, 2, HEAD)
    score = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(HEAD))
    seen = (torch.arange(length, device="cuda")[None, :] < s["lens"][:, None])[:, None, None, :]
    score = torch.where(seen, score, torch.full_like(score, -torch.inf))
    top = score.amax(3, keepdim=True)
    weight = torch.where(seen, torch.exp(score - torch.where(torch.isfinite(top), top, torch.zeros_like(top))), torch.zeros_like(score))
    total = weight.sum(3, keepdim=True)
    out = torch.matmul(weight, v) / torch.where(total > 0, total, torch.ones_like(total))
    return out.reshape(batch, q_heads, HEAD).to(torch.bfloat16)


def _plain_linear(s):
    x = s["x"].float()
    if s["norm"] is not None:
        x = x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPSILON) * s["norm"].float()
    scale = x.abs().amax(1, keepdim=True) / 127
    level = torch.round(x / torch.where(scale > 0, scale, torch.ones_like(scale))).clamp(-127, 127)

    def product(name):
        return torch.matmul(level, s[name].float().t()) * scale * s[name + "_scale"]

    if s["kind"] == "gated":
        gate = product("gate")
        return (gate / (1 + torch.exp(-gate)) * product("up")).to(torch.bfloat16)
    out = product("w")
    if s["bias"] is not None:
        out = out + s["bias"].float()
    if s["residual"] is not None:
        out = out + s["residual"].float()
    return out.to(torch.bfloat16)


def _plain_sample(s):
    # In 64 bits: sums over a whole vocabulary meet borders (top-p's and the draw's) that 32 bits blur.
    score = s["logits"].double()
    vocab = score.shape[1]
    greedy = s["temperature"] <= 0
    heat = torch.where(greedy, torch.ones_like(s["temperature"]), s["temperature"]).double()[:, None]
    weight = torch.exp((score - score.amax(1, keepdim=True)) / heat)
    order = torch.sort(score, dim=1, descending=True, stable=True).indices
    ranked = weight.gather(1, order)
    rank = torch.arange(vocab, device="cuda")[None, :]
    limit = torch.where(s["top_k"] > 0, s["top_k"], torch.full_like(s["top_k"], vocab)).long()[:, None]
    limit = torch.where(greedy[:, None], torch.ones_like(limit), limit)
    ranked = torch.where(rank < limit, ranked, torch.zeros_like(ranked))
    mass = ranked.cumsum(1)
    share = torch.where(s["top_p"] < 1, s["top_p"].double(), torch.full_like(s["top_p"], torch.inf, dtype=torch.float64))[:, None]
    keep = (rank < limit) & ((mass - ranked < share * mass[:, -1:]) | (rank == 0)) & (ranked >= s["min_p"].double()[:, None] * ranked[:, :1])
    left = torch.zeros_like(weight).scatter(1, order, torch.where(keep, ranked, torch.zeros_like(ranked)))
    sums = left.cumsum(1)
    token = (sums <= s["uniform"].double()[:, None] * sums[:, -1:]).sum(1)
    return token.to(torch.int32), (left.gather(1, token[:, None])[:, 0] / sums[:, -1]).float()


def run(state):
    if state["op"] == "attention":
        if own:
            return state["engine"].launch_attention_shared(0, state["q"], state["lens"], state["table"], state["starts"],
                                                           state["shared"], state["max_shared"])
        return _plain_attention(state)
    if state["op"] == "linear":
        if own:
            engine = _engine()
            level, scale = engine.quantize_rows_int8(state["x"], state["norm"])
            if state["kind"] == "gated":
                return engine.gate_up_swiglu_int8(level, scale, state["gate"], state["gate_scale"], state["up"], state["up_scale"])
            return engine.linear_int8(level, scale, state["w"], state["w_scale"], state["bias"], state["residual"])
        return _plain_linear(state)
    if own:
        return _engine().sample_filtered(state["logits"], state["uniform"], state["temperature"], state["top_k"], state["top_p"],
                                         state["min_p"])
    return _plain_sample(state)


def work(case):
    if case["op"] == "attention":
        starts, shared, lens, _, _ = _layout(case, 0)
        heads, batch = case["kv_heads"], case["batch"]
        of = torch.bucketize(torch.arange(batch), starts[1:], right=True)
        rest = (lens - shared[of] * PAGE).clamp(min=0)
        tokens = int(shared.sum()) * PAGE + int(rest.sum())
        return {"bytes": tokens * heads * HEAD * 4 + 2 * batch * 2 * heads * HEAD * 2, "flops": 4 * int(lens.sum()) * 2 * heads * HEAD}
    if case["op"] == "linear":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        both = 2 if case["kind"] == "gated" else 1
        moved = rows * inner * 2 + both * outer * (inner + 4) + rows * outer * (4 if case["residual"] else 2)
        moved += (inner * 2 if case["norm"] else 0) + (outer * 2 if case["bias"] else 0)
        return {"bytes": moved, "flops": 2 * both * rows * inner * outer}
    values = case["batch"] * case["vocab"]
    return {"bytes": values * (2 if case["dtype"] == "bfloat16" else 4) + case["batch"] * 28, "flops": 4 * values}


# ---- the definitions in 64 bits

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["op"] == "attention":
        out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
        for b, n in enumerate(s["lens"].tolist()):
            if n == 0:
                continue
            at = torch.arange(n, device="cuda")
            page, slot = s["table"][b].long()[at // PAGE], at % PAGE
            for h in range(case["kv_heads"]):
                k, v = s["k"][page, h, slot].double(), s["v"][page, h, slot].double()
                p = torch.softmax(s["q"][b, 2 * h:2 * h + 2].double() @ k.t() / math.sqrt(HEAD), 1)
                out[b, 2 * h:2 * h + 2] = p @ v
        return out
    if case["op"] == "linear":
        x = s["x"].double()
        if s["norm"] is not None:
            x = x / torch.sqrt(x.pow(2).mean(1, keepdim=True) + EPSILON) * s["norm"].double()
        step = x.abs().max(1, keepdim=True).values / 127
        x = torch.where(step > 0, torch.round(x / step), torch.zeros_like(x)) * step
        if case["kind"] == "gated":
            gate = x @ (s["gate"].double() * s["gate_scale"].double()[:, None]).t()
            up = x @ (s["up"].double() * s["up_scale"].double()[:, None]).t()
            return gate * torch.sigmoid(gate) * up
        out = x @ (s["w"].double() * s["w_scale"].double()[:, None]).t()
        if s["bias"] is not None:
            out = out + s["bias"].double()
        if s["residual"] is not None:
            out = out + s["residual"].double()
        return out
    tokens, chances = [], []
    for b in range(case["batch"]):
        z, heat = s["logits"][b].double(), float(s["temperature"][b])
        if heat <= 0:
            tokens.append(int(torch.nonzero(z == z.max())[0, 0]))
            chances.append(1.0)
            continue
        p = torch.softmax(z / heat, 0)
        best = torch.argsort(z, descending=True, stable=True)
        k, share, low = int(s["top_k"][b]), float(s["top_p"][b]), float(s["min_p"][b])
        if k > 0:
            best = best[:k]
        if share < 1:
            ahead = torch.cat([torch.zeros(1, dtype=torch.float64, device="cuda"), p[best].cumsum(0)])
            best = best[: max(1, int((ahead[:-1] < share * ahead[-1]).sum()))]
        best = best[p[best] >= low * p[best[0]]]
        kept = best.sort().values
        c = p[kept].cumsum(0)
        at = min(int(torch.searchsorted(c, c[-1] * float(s["uniform"][b]), right=True)), len(kept) - 1)
        tokens.append(int(kept[at]))
        chances.append(float(p[kept[at]] / c[-1]))
    return torch.tensor(tokens, dtype=torch.int32), torch.tensor(chances, dtype=torch.float64)
