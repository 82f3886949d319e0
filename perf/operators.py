"""The cases by which the embedding and routing operators are measured, and the operators in plain torch.

Four kinds of pass, each as a program makes it:

* ``lookup``    out[t] = scale * table[tokens[t] - first_id], zero rows for ids outside the table's range;
* ``gradient``  the tokens grouped by id, then grad_table[v] = scale * sum of the grad rows of v's tokens (plus what is there);
* ``dispatch``  tokens per expert, and the (token, choice) pairs in expert order;
* ``balance``   the balance loss of a router with its per-expert counts, and the gradient of the router's logits.
"""
import math

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2}
_IDS = {"i32": torch.int32, "i64": torch.int64}


def listed():
    return [
        # one token for each of 16 running sequences: the latency of a serving step
        dict(name="lookup step", kind="lookup", tokens=16, rows=131072, dim=4096, type="bf16", ids="i64", pitch=4096, first=0, shards=1),
        # a prompt on one of two vocabulary shards (half of the ids lie in the other), odd width, padded table rows
        dict(name="lookup shard odd", kind="lookup", tokens=4099, rows=50021, dim=1001, type="f16", ids="i32", pitch=1024, first=50021, shards=2),
        # a training batch in full precision
        dict(name="lookup batch", kind="lookup", tokens=65536, rows=131072, dim=2048, type="f32", ids="i64", pitch=2048, first=0, shards=1),
        # a short micro-batch added to a full-precision gradient buffer
        dict(name="gradient micro", kind="gradient", tokens=509, rows=32768, dim=1024, type="bf16", out="f32", ids="i64", hot=0.0, add=True),
        # one sequence of 8192, gradient in the table's type: most rows of the table stay without a token
        dict(name="gradient sequence", kind="gradient", tokens=8192, rows=131072, dim=4096, type="bf16", out="bf16", ids="i64", hot=0.0, add=False),
        # half of the tokens are one placeholder id, odd width
        dict(name="gradient hot odd", kind="gradient", tokens=20011, rows=50021, dim=1001, type="f16", out="f32", ids="i32", hot=0.5, add=False),
        # a training batch of 131072 tokens
        dict(name="gradient batch", kind="gradient", tokens=131072, rows=131072, dim=4096, type="bf16", out="f32", ids="i64", hot=0.0, add=False),
        # a serving step of 64 tokens, 8 experts each
        dict(name="dispatch step", kind="dispatch", tokens=64, experts=256, choices=8, ids="i64", masked=0.0),
        # a training batch, 8 experts each, padded tokens masked
        dict(name="dispatch batch", kind="dispatch", tokens=65536, experts=256, choices=8, ids="i64", masked=0.1),
        # a short micro-batch with padded tokens
        dict(name="balance micro", kind="balance", tokens=128, experts=64, choices=6, type="bf16", ids="i64", masked=0.25),
        # an ordinary batch, router logits in full precision
        dict(name="balance sequence", kind="balance", tokens=16384, experts=128, choices=8, type="f32", ids="i64", masked=0.0),
        # a large batch, odd length
        dict(name="balance batch", kind="balance", tokens=262139, experts=256, choices=8, type="bf16", ids="i64", masked=0.1),
    ]


def _log(rng, low, high):
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    kind = rng.choice(["lookup", "gradient", "gradient", "dispatch", "balance", "balance"])
    if kind == "lookup":
        dim, shards = _log(rng, 64, 8192), rng.choice([1, 1, 2, 4])
        rows = _log(rng, 1000, min(131072, 536870912 // dim))
        return dict(kind=kind, tokens=_log(rng, 1, min(65536, 134217728 // dim)), rows=rows, dim=dim, type=rng.choice(["f32", "f16", "bf16", "bf16"]),
                    ids=rng.choice(["i32", "i64"]), pitch=dim + rng.choice([0, 0, 8, 24]), first=rows * rng.randrange(shards), shards=shards)
    if kind == "gradient":
        dim, in_type = _log(rng, 64, 8192), rng.choice(["f32", "f16", "bf16", "bf16"])
        return dict(kind=kind, tokens=_log(rng, 1, min(131072, 268435456 // dim)), rows=_log(rng, 1000, min(131072, 268435456 // dim)), dim=dim,
                    type=in_type, out=rng.choice(["f32", in_type]), ids=rng.choice(["i32", "i64"]), hot=rng.choice([0.0, 0.0, 0.3]), add=rng.random() < 0.5)
    experts = _log(rng, 4, 512)
    case = dict(kind=kind, tokens=_log(rng, 1, 262139 if kind == "balance" else 65536), experts=experts, choices=rng.randint(1, min(8, experts)),
                ids=rng.choice(["i32", "i64"]), masked=rng.choice([0.0, 0.1, 0.5]))
    if kind == "balance":
        case["type"] = rng.choice(["f32", "f16", "bf16"])
        case["tokens"] = min(case["tokens"], 67107584 // experts)
    return case


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _zipf(n, ids, g):
    """Token ids whose frequency falls as one over their rank."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    return (torch.exp(u * math.log(ids + 1.0)) - 1.0).to(torch.int64).clamp_(0, ids - 1)


def _normal(rows, cols, type, g):
    out = torch.empty(rows, cols, dtype=_TYPES[type], device="cuda")
    return out.normal_(generator=g)


def prepare(case, seed):
    g = _generator(seed)
    if case["kind"] == "lookup":
        table = _normal(case["rows"], case["pitch"], case["type"], g)[:, :case["dim"]]
        tokens = _zipf(case["tokens"], case["rows"], g)
        if case["shards"] > 1:  # the other shards' ids, spread over all of the vocabulary
            every = torch.randint(case["rows"] * case["shards"], (case["tokens"],), generator=g, device="cuda")
            tokens = torch.where(torch.rand(case["tokens"], generator=g, device="cuda") < 0.5, tokens + case["first"], every)
        return dict(case, table=table, tokens=tokens.to(_IDS[case["ids"]]), scale=math.sqrt(case["dim"]))
    if case["kind"] == "gradient":
        tokens = _zipf(case["tokens"], case["rows"], g)
        if case["hot"]:
            hot = torch.rand(case["tokens"], generator=g, device="cuda") < case["hot"]
            tokens = torch.where(hot, torch.full_like(tokens, case["rows"] // 3), tokens)
        state = dict(case, tokens=tokens.to(_IDS[case["ids"]]), grad=_normal(case["tokens"], case["dim"], case["type"], g).mul_(1 / 64), scale=math.sqrt(case["dim"]))
        if case["add"]:
            state["sum"] = _normal(case["rows"], case["dim"], case["out"], g)
        return state
    # routers prefer some experts: a bias of each expert on top of what the token asks for
    bias = torch.randn(case["experts"], generator=g, device="cuda")
    logits = torch.randn(case["tokens"], case["experts"], generator=g, device="cuda").mul_(1.5).add_(bias)
    type = case.get("type", "f32")
    logits = logits.to(_TYPES[type])
    experts = torch.topk(logits.float(), case["choices"], dim=1).indices.to(_IDS[case["ids"]])
    mask = torch.rand(case["tokens"], generator=g, device="cuda") >= case["masked"] if case["masked"] else None
    if case["kind"] == "dispatch":
        if mask is not None:  # a padded token goes to no expert
            experts = torch.where(mask[:, None], experts, torch.full_like(experts, -1))
        return dict(case, chosen=experts)
    return dict(case, logits=logits, chosen=experts, mask=mask, coefficient=0.01, loss_grad=torch.full((), 0.5, device="cuda"))


def _run_own(s):
    if s["kind"] == "lookup":
        from loops_amd import embedding
        return embedding.lookup(s["table"], s["tokens"], scale=s["scale"], first_id=s["first"])
    if s["kind"] == "gradient":
        from loops_amd import embedding
        groups = embedding.group_tokens(s["tokens"], s["rows"])
        if s["add"]:
            return embedding.gradient(groups, s["grad"], scale=s["scale"], out=s["sum"], accumulate=True)
        return embedding.gradient(groups, s["grad"], scale=s["scale"], dtype=_TYPES[s["out"]])
    if s["kind"] == "dispatch":
        from loops_amd import embedding, routing
        counts = routing.expert_counts(s["chosen"], s["experts"])
        groups = embedding.group_tokens(s["chosen"], s["experts"])
        return dict(counts=counts, ids=groups.ids, positions=groups.positions)
    from loops_amd import routing
    forward = routing.balance_loss(s["logits"], s["chosen"], coefficient=s["coefficient"], mask=s["mask"])
    grad = routing.balance_loss_backward(s["logits"], forward, mask=s["mask"], grad_loss=s["loss_grad"])
    return dict(loss=forward.loss, counts=forward.counts, probability=forward.probability, grad=grad)


def _plain_counts(ids, inside, rows):
    return torch.zeros(rows + 1, dtype=torch.int32, device="cuda").index_add_(0, torch.where(inside, ids, rows), torch.ones_like(ids, dtype=torch.int32))[:rows]


def run(s):
    if own:
        return _run_own(s)
    if s["kind"] == "lookup":
        ids = s["tokens"].long() - s["first"]
        inside = (ids >= 0) & (ids < s["rows"])
        out = s["table"][torch.where(inside, ids, 0)].float() * s["scale"]
        return torch.where(inside[:, None], out, 0.0).to(s["table"].dtype)
    if s["kind"] == "gradient":
        into = s["sum"].float() if s["add"] else torch.zeros(s["rows"], s["dim"], device="cuda")
        into.index_add_(0, s["tokens"].long(), s["grad"].float() * s["scale"])
        if s["add"]:
            return s["sum"].copy_(into)
        return into.to(_TYPES[s["out"]])
    ids = s["chosen"].reshape(-1).long()
    if s["kind"] == "dispatch":
        inside = (ids >= 0) & (ids < s["experts"])
        keys, order = torch.sort(torch.where(inside, ids, s["experts"]), stable=True)
        return dict(counts=_plain_counts(ids, inside, s["experts"]), ids=keys.int(), positions=order.int())
    x = s["logits"].float()
    p = torch.exp(x - x.amax(1, keepdim=True))
    p = p / p.sum(1, keepdim=True)
    keep = torch.ones(x.shape[0], dtype=torch.bool, device="cuda") if s["mask"] is None else s["mask"]
    p = torch.where(keep[:, None], p, 0.0)
    inside = keep.repeat_interleave(s["choices"]) & (ids >= 0) & (ids < s["experts"])
    counts = _plain_counts(ids, inside, s["experts"])
    n = keep.sum().clamp(min=1)
    share, probability = counts / (n * s["choices"]), p.sum(0) / n
    loss = s["coefficient"] * s["experts"] * (share * probability).sum()
    grad = p * (share - (p * share).sum(1, keepdim=True)) * (s["loss_grad"] * s["coefficient"] * s["experts"] / n)
    return dict(loss=loss, counts=counts, probability=probability, grad=grad.to(s["logits"].dtype))


def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "lookup":
        wide = torch.zeros(s["tokens"].shape[0], s["dim"], dtype=torch.float64, device="cuda")
        at = torch.nonzero((s["tokens"] >= s["first"]) & (s["tokens"] < s["first"] + s["rows"]))[:, 0]
        wide[at] = torch.index_select(s["table"], 0, s["tokens"][at].long() - s["first"]).double().mul_(s["scale"])
        return wide
    if s["kind"] == "gradient":
        # differences of the running sums over the tokens in id order, a block of columns at a time
        tokens, order = torch.sort(s["tokens"].long(), stable=True)
        ends = torch.searchsorted(tokens, torch.arange(s["rows"], device="cuda"), right=True)
        starts = torch.searchsorted(tokens, torch.arange(s["rows"], device="cuda"))
        out = torch.empty(s["rows"], s["dim"], dtype=torch.float64, device="cuda")
        step = max(1, 33554432 // case["tokens"])
        for c in range(0, s["dim"], step):
            part = s["grad"][:, c:c + step].double()[order]
            sums = torch.cat([torch.zeros(1, part.shape[1], dtype=torch.float64, device="cuda"), part.cumsum(0)])
            out[:, c:c + step] = (sums[ends] - sums[starts]) * s["scale"]
        out[starts == ends] = 0.0
        return out + s["sum"].double() if s["add"] else out
    if s["kind"] == "dispatch":
        ids = s["chosen"].reshape(-1).cpu().numpy().astype(np.int64)
        keys = np.where((ids >= 0) & (ids < s["experts"]), ids, s["experts"])
        order = np.argsort(keys, kind="stable")
        return dict(counts=np.bincount(keys, minlength=s["experts"] + 1)[:s["experts"]].astype(np.int32), ids=keys[order].astype(np.int32), positions=order.astype(np.int32))
    k, experts = s["choices"], s["experts"]
    keep = torch.arange(case["tokens"], device="cuda") if s["mask"] is None else torch.nonzero(s["mask"])[:, 0]
    n = max(1, keep.numel())
    log_p = torch.log_softmax(s["logits"][keep].double(), 1)
    p = log_p.exp()
    share = torch.bincount(s["chosen"][keep].reshape(-1).long(), minlength=experts).double() / (n * k)
    probability = p.sum(0) / n
    along = float(s["loss_grad"]) * s["coefficient"] * experts / n * share  # d loss / d p, the same for every token
    grad = torch.zeros(s["logits"].shape, dtype=torch.float64, device="cuda")
    grad[keep] = p * along - p * (p @ along)[:, None]
    return dict(loss=s["coefficient"] * experts * (share @ probability), counts=None, probability=probability, grad=grad)


def work(case):
    if case["kind"] == "lookup":
        t, size = case["tokens"], _BYTES[case["type"]]
        # frequent ids repeat: the distinct rows that n tokens of a Zipf-like vocabulary need
        mine = t if case["shards"] == 1 else t * (0.5 + 0.5 / case["shards"])
        row = case["dim"] * size
        return {"bytes": _distinct(mine, case["rows"]) * row + t * row + t * (4 if case["ids"] == "i32" else 8), "flops": mine * case["dim"]}
    if case["kind"] == "gradient":
        t, d, out = case["tokens"], case["dim"], _BYTES[case["out"]]
        ids = 4 if case["ids"] == "i32" else 8
        written = 2 * _distinct(t * (1 - case["hot"]), case["rows"]) if case["add"] else case["rows"]
        return {"bytes": t * (ids + d * _BYTES[case["type"]]) + written * d * out, "flops": t * d}
    n, ids = case["tokens"] * case["choices"], 4 if case["ids"] == "i32" else 8
    if case["kind"] == "dispatch":
        return {"bytes": n * (ids + 8) + 4 * case["experts"], "flops": n}
    cells = case["tokens"] * case["experts"]
    # the gradient needs the counts of all tokens first, so the logits are read in both directions
    return {"bytes": 3 * cells * _BYTES[case["type"]] + n * ids + (2 * case["tokens"] if case["masked"] else 0) + 8 * case["experts"], "flops": 13 * cells}


def _distinct(tokens, ids):
    """About how many distinct ids `tokens` draws of _zipf have: rank r is drawn with probability log(1 + 1 / r) / log(ids + 1)."""
    found, low = 0.0, 1.0
    while low <= ids:  # ranks in runs of an eighth of their size
        high = min(ids + 1.0, max(low + 1.0, low * 1.125))
        share = math.log(high / low) / math.log(ids + 1.0) / (high - low)
        found += (high - low) * (1.0 - (1.0 - share) ** tokens)
        low = high
    return found
