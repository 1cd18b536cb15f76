"""The operators of a mixture-of-experts serving step, as measurable cases.

Every case is one call of an operator that a serving loop of such a model makes beside its attention:

* ``route``: each token's experts and their weights, from the router's logits: softmax or sigmoid scores, a bias that
  only the choice sees, groups of experts of which the best few stay, renormalised weights;
* ``experts``: the feed-forward block of each token's experts on packed weights, weighted and summed per token;
* ``logprobs``: log probabilities of given tokens, with their rank, the distribution's entropy and the likeliest tokens.

Packed weights are [experts, rows, K] codes as one little-endian bit stream (fp4_e2m1, int4 and uint4 two codes a byte,
the lower nibble first; the 6-bit formats four codes in three bytes), with one scale per block of K: a power of two per 32
for the float formats, stored as the exponent plus 127, and a 16- or 32-bit number per 32, 64 or 128 for integers.
Gate and up rows of an expert alternate: rows 2 i and 2 i + 1.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BITS = {"fp4_e2m1": 4, "fp6_e2m3": 6, "fp6_e3m2": 6, "int4": 4, "uint4": 4}
# float formats: exponent bits, mantissa bits, exponent bias
FLOATS = {"fp4_e2m1": (2, 1, 1), "fp6_e2m3": (2, 3, 1), "fp6_e3m2": (3, 2, 3)}


def listed():
    return [
        # one decode step of eight sequences: the smallest call
        dict(name="route_decode", kind="route", dtype="float32", tokens=8, experts=64, top_k=6, score="softmax", bias=False,
             groups=1, top_groups=1, renormalize=True, scale=1.0),
        # a long prompt's choice among many experts: sigmoid scores, a balancing bias, half of the groups
        dict(name="route_prompt_groups", kind="route", dtype="float32", tokens=8192, experts=256, top_k=8, score="sigmoid",
             bias=True, groups=8, top_groups=4, renormalize=True, scale=2.5),
        # a prompt of an odd length, few experts, 16-bit logits full of ties
        dict(name="route_bf16_prompt", kind="route", dtype="bfloat16", tokens=4001, experts=8, top_k=2, score="softmax",
             bias=False, groups=1, top_groups=1, renormalize=True, scale=1.0),
        # one token through two of eight large experts: the weights' bytes bound it
        dict(name="experts_one", kind="experts", fmt="fp4_e2m1", group=32, scales="e8m0", tokens=1, padded=0, experts=8,
             top_k=2, hidden=4096, ffn=14336, skew=0.5),
        # one token of each of eight sequences through many small experts, most of them alone
        dict(name="experts_fine_b8", kind="experts", fmt="fp4_e2m1", group=32, scales="e8m0", tokens=8, padded=0, experts=64,
             top_k=6, hidden=2048, ffn=1408, skew=0.5),
        # a decode batch of odd size on integer weights, some of its places empty
        dict(name="experts_int4_b45", kind="experts", fmt="int4", group=128, scales="float16", tokens=45, padded=3,
             experts=16, top_k=4, hidden=4096, ffn=2048, skew=0.7),
        # a chunk of a prompt of odd length through 6-bit experts
        dict(name="experts_fp6_chunk", kind="experts", fmt="fp6_e2m3", group=32, scales="e8m0", tokens=509, padded=0,
             experts=32, top_k=4, hidden=2048, ffn=1408, skew=0.7),
        # a long prompt through many small experts
        dict(name="experts_fine_prompt", kind="experts", fmt="fp4_e2m1", group=32, scales="e8m0", tokens=2048, padded=0,
             experts=64, top_k=6, hidden=2048, ffn=1408, skew=0.5),
        # eight prompts of 512 tokens through large experts: the products bound it
        dict(name="experts_prompt", kind="experts", fmt="fp4_e2m1", group=32, scales="e8m0", tokens=4096, padded=0,
             experts=8, top_k=2, hidden=4096, ffn=14336, skew=0.3),
        # the tokens just drawn for eight sequences, with twenty alternatives each
        dict(name="logprobs_step", kind="logprobs", dtype="float32", rows=8, vocab=32000, top=20),
        # one sequence over a large vocabulary
        dict(name="logprobs_one_131072", kind="logprobs", dtype="float32", rows=1, vocab=131072, top=5),
        # scoring eight prompts: every position's logits
        dict(name="logprobs_prompts", kind="logprobs", dtype="bfloat16", rows=4000, vocab=32000, top=5),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    kind = rng.choice(["route", "route", "experts", "experts", "experts", "experts", "logprobs", "logprobs"])
    if kind == "route":
        groups = rng.choice([1, 1, 1, 2, 4, 8])
        experts = groups * rng.randint(2, 32) if groups > 1 else _log_int(rng, 4, 256)
        top_groups = rng.randint(1, groups)
        return dict(kind=kind, dtype=rng.choice(["float32", "float32", "bfloat16", "float16"]),
                    tokens=_log_int(rng, 1, 8192), experts=experts,
                    top_k=rng.randint(1, min(8, experts // groups * top_groups)),
                    score=rng.choice(["softmax", "sigmoid"]), bias=rng.choice([False, True]), groups=groups,
                    top_groups=top_groups, renormalize=rng.choice([False, True, True]), scale=rng.choice([1.0, 2.5]))
    if kind == "logprobs":
        vocab = _log_int(rng, 500, 131072)
        return dict(kind=kind, dtype=rng.choice(["float32", "bfloat16", "float16"]),
                    rows=_log_int(rng, 1, min(4000, 60000000 // vocab)), vocab=vocab, top=rng.choice([0, 1, 5, 20, 50]))
    fmt = rng.choice(["fp4_e2m1", "fp4_e2m1", "fp4_e2m1", "fp6_e2m3", "fp6_e3m2", "int4", "int4", "uint4"])
    hidden, ffn = 128 * rng.randint(4, 32), 128 * _log_int(rng, 4, 112)
    experts = min(_log_int(rng, 4, 64), 1400000000 // (3 * hidden * ffn))  # codes of the largest listed
    top_k = rng.randint(1, min(8, experts))
    tokens = _log_int(rng, 1, min(4096, 2800000000000 // (6 * hidden * ffn * top_k)))  # operations of the largest listed
    integer = fmt not in FLOATS
    return dict(kind=kind, fmt=fmt, group=rng.choice([32, 64, 128]) if integer else 32,
                scales=rng.choice(["float16", "bfloat16", "float32"]) if integer else "e8m0", tokens=tokens,
                padded=rng.choice([0, 0, tokens // 5]), experts=experts, top_k=top_k, hidden=hidden, ffn=ffn,
                skew=rng.choice([0.0, 0.5, 1.0]))


# ------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, device=DEVICE, generator=g)


def _weight(g, case, rows, k):
    """Codes, and scales that make values of about 0.02."""
    e = case["experts"]
    data = torch.randint(0, 256, (e * rows * k * BITS[case["fmt"]] // 8,), dtype=torch.uint8, device=DEVICE, generator=g)
    shape = (e, rows, k // case["group"])
    if case["scales"] == "e8m0":
        mid = {"fp4_e2m1": 120, "fp6_e2m3": 119, "fp6_e3m2": 118}[case["fmt"]]  # of 2.9, 3.9 and 10 on average
        scales = torch.randint(mid - 1, mid + 2, shape, dtype=torch.uint8, device=DEVICE, generator=g)
    else:
        scales = (torch.rand(shape, device=DEVICE, generator=g) * 0.003 + 0.002).to(DTYPES[case["scales"]])
    return data, scales


def _inputs(case, seed):
    """What the operator takes, as plain tensors."""
    g, kind = _generator(seed), case["kind"]
    if kind == "route":
        logits = (_randn(g, case["tokens"], case["experts"]) * 1.5).to(DTYPES[case["dtype"]])
        return dict(logits=logits, bias=_randn(g, case["experts"]) * 0.1 if case["bias"] else None)
    if kind == "logprobs":
        logits = (_randn(g, case["rows"], case["vocab"]) * 3).to(DTYPES[case["dtype"]])
        # a drawn token is mostly a likely one: the largest of a few at random
        some = torch.randint(0, case["vocab"], (case["rows"], 64), device=DEVICE, generator=g)
        best = logits.gather(1, some).float().argmax(1, keepdim=True)
        return dict(logits=logits, tokens=some.gather(1, best)[:, 0].to(torch.int32))
    t, e, k = case["tokens"], case["experts"], case["top_k"]
    x = _randn(g, t, case["hidden"]).to(_x_dtype(case))
    score = _randn(g, t, e) + case["skew"] * _randn(g, e)  # some experts are more popular
    top = torch.sort(score, dim=-1, descending=True)
    weights = torch.softmax(top.values[:, :k], -1).contiguous()
    ids = top.indices[:, :k].to(torch.int32).contiguous()
    ids[t - case["padded"]:] = -1  # places of the batch that hold no token
    gate_up = _weight(g, case, 2 * case["ffn"], case["hidden"])
    down = _weight(g, case, case["hidden"], case["ffn"])
    return dict(x=x, ids=ids, weights=weights, gate_up=gate_up, down=down)


def _x_dtype(case):
    """The activations' type on weights of this format."""
    return torch.bfloat16 if case["fmt"] in FLOATS else torch.float16


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if own:
        path = str(Path(__file__).resolve().parent.parent / "tinygrad-dx12_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        if case["kind"] == "logprobs":
            from tinygrad_mi355x.sampling import log_probs

            state["call"] = log_probs
        elif case["kind"] == "route":
            from tinygrad_mi355x.experts import route

            state["call"] = route
        else:
            from tinygrad_mi355x.codegen.decomp.mi355x import PackedTensor
            from tinygrad_mi355x.experts import PackedExperts

            e, d, f = case["experts"], case["hidden"], case["ffn"]
            packed = []
            for (data, scales), shape in ((state["gate_up"], (e, 2 * f, d)), (state["down"], (e, d, f))):
                scales = scales.view(torch.float8_e8m0fnu) if case["scales"] == "e8m0" else scales
                packed.append(PackedTensor(data, case["fmt"], shape, scales, case["group"]))
            state["call"] = PackedExperts(*packed).apply
    return state


# ------------------------------------------------------------------------------------ one pass
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        if kind == "route":
            got = state["call"](state["logits"], case["top_k"], score=case["score"], bias=state["bias"],
                                groups=case["groups"], top_groups=case["top_groups"], renormalize=case["renormalize"],
                                scale=case["scale"])
            return dict(ids=got.ids, weights=got.weights)
        if kind == "experts":
            return state["call"](state["x"], state["ids"], state["weights"])
        got = state["call"](state["logits"], state["tokens"], top=case["top"])
        return dict(logprobs=got.logprobs, ranks=got.ranks, entropy=got.entropy, top_ids=got.top_ids,
                    top_logprobs=got.top_logprobs)
    return {"route": _plain_route, "experts": _plain_experts, "logprobs": _plain_logprobs}[kind](state)


# ------------------------------------------------------------------------------- plain forms
def _plain_route(state):
    """Scores in 64 bits: a choice next to a border is decided by their last places."""
    case, x = state["case"], state["logits"].double()
    if case["score"] == "softmax":
        p = torch.exp(x - x.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
    else:
        p = 1 / (1 + torch.exp(-x))
    choice = p if state["bias"] is None else p + state["bias"].double()
    rank = x if state["bias"] is None else choice  # without a bias the logits' own order
    n = case["groups"]
    if case["top_groups"] < n:  # a group counts by the sum of its two best
        best = torch.sort(choice.unflatten(-1, (n, -1)), dim=-1, descending=True).values[..., :2].sum(-1)
        out = torch.sort(best, dim=-1, descending=True, stable=True).indices[:, case["top_groups"]:]
        left = torch.zeros_like(best, dtype=torch.bool).scatter_(1, out, True)
        rank = rank.masked_fill(left.repeat_interleave(case["experts"] // n, 1), -math.inf)
    ids = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]]  # ties: the lower index first
    weights = p.gather(1, ids)
    if case["renormalize"]:
        weights = weights / weights.sum(-1, keepdim=True)
    return dict(ids=ids.to(torch.int32), weights=(weights * case["scale"]).float())


def _plain_values(data, scales, case, rows, k):
    """Packed weights of some experts, [n, rows, k] in 32 bits; data [n, bytes], scales [n, rows, blocks]."""
    fmt = case["fmt"]
    if BITS[fmt] == 4:
        code = torch.stack((data & 15, data >> 4), -1).flatten(1)
    else:
        a, b, c = (t.to(torch.int16) for t in data.unflatten(1, (-1, 3)).unbind(-1))
        code = torch.stack((a & 63, (a >> 6) | ((b & 15) << 2), (b >> 4) | ((c & 3) << 4), c >> 2), -1).flatten(1)
    if fmt in FLOATS:
        eb, mb, bias = FLOATS[fmt]
        table = torch.arange(1 << (eb + mb + 1), dtype=torch.int32, device=data.device)
        exp, frac = (table >> mb) & ((1 << eb) - 1), table & ((1 << mb) - 1)
        mag = torch.ldexp((frac + ((exp > 0) << mb)).float(), exp.clamp(min=1) - bias - mb)
        values = torch.where(table >> (eb + mb) > 0, -mag, mag)
    else:
        values = torch.arange(16, dtype=torch.float32, device=data.device)
        values = torch.where(values < 8, values, values - 16) if fmt == "int4" else values
    blocks = values[code.int()].unflatten(1, (rows, k // case["group"], case["group"]))
    one = torch.ones((), device=data.device)
    scale = torch.ldexp(one, scales.int() - 127) if fmt in FLOATS else scales.float()
    return (blocks * scale[..., None]).flatten(2)


def _plain_experts(state):
    """The tokens of each expert that any token names, padded to the longest list, in one batched product."""
    case, x, ids = state["case"], state["x"], state["ids"].long()
    e, d, f, k = case["experts"], case["hidden"], case["ffn"], case["top_k"]
    used, slot, count = torch.unique(ids.flatten(), return_inverse=True, return_counts=True)
    order = torch.argsort(slot, stable=True)
    place = torch.empty_like(slot)
    place[order] = torch.arange(slot.numel(), device=DEVICE) - (count.cumsum(0) - count)[slot[order]]
    rows = torch.zeros((used.numel(), int(count.max()), d), device=DEVICE)
    rows[slot, place] = x.float().repeat_interleave(k, 0)
    used = used.clamp(min=0)

    def product(packed, n, m, columns):  # [experts, tokens, n] from [experts, m, tokens]
        data, scales = packed
        w = _plain_values(data.view(e, -1)[used], scales[used], case, n, m)
        return torch.matmul(w, columns.contiguous()).transpose(1, 2)

    both = product(state["gate_up"], 2 * f, d, rows.transpose(1, 2))
    gate, up = both[..., 0::2], both[..., 1::2]
    hidden = gate / (1 + torch.exp(-gate)) * up
    out = product(state["down"], d, f, hidden.transpose(1, 2))[slot, place].view(-1, k, d)
    weights = state["weights"].masked_fill(ids < 0, 0.0)
    return (out * weights[..., None]).sum(1).to(x.dtype)


def _plain_logprobs(state):
    """Sums over the vocabulary in 64 bits."""
    case, x = state["case"], state["logits"].float()
    tok = state["tokens"].long()[:, None]
    top = x.amax(-1, keepdim=True)
    d = x - top
    w = torch.exp(d)
    total = w.double().sum(-1, keepdim=True)
    log_total = total.log()
    at = x.gather(1, tok)
    index = torch.arange(case["vocab"], device=DEVICE)
    ranks = ((x > at) | ((x == at) & (index < tok))).sum(-1)
    best = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lower index first
    return dict(logprobs=((at - top) - log_total)[:, 0].float(), ranks=ranks.to(torch.int32),
                entropy=(log_total - (w * d).double().sum(-1, keepdim=True) / total)[:, 0].float(),
                top_ids=best.indices[:, :case["top"]].to(torch.int32),
                top_logprobs=((best.values[:, :case["top"]] - top) - log_total).float())


# --------------------------------------------------------------------------------- what it takes
def _expected(experts, tokens, top_k):
    """Experts that some token names, on average, each with the same chance."""
    return experts * (1 - (1 - top_k / experts) ** tokens)


def work(case):
    kind = case["kind"]
    if kind == "route":
        n = case["tokens"] * case["experts"]
        return dict(bytes=n * DTYPES[case["dtype"]].itemsize + case["tokens"] * case["top_k"] * 8, flops=4 * n)
    if kind == "logprobs":
        n = case["rows"] * case["vocab"]
        return dict(bytes=n * DTYPES[case["dtype"]].itemsize + case["rows"] * (16 + 8 * case["top"]), flops=4 * n)
    d, f, t = case["hidden"], case["ffn"], case["tokens"] - case["padded"]
    scale = 1 if case["scales"] == "e8m0" else DTYPES[case["scales"]].itemsize
    weight = 3 * d * f * (BITS[case["fmt"]] / 8 + scale / case["group"])
    return dict(bytes=_expected(case["experts"], t, case["top_k"]) * weight + t * (4 * d + 8 * case["top_k"]),
                flops=6 * d * f * t * case["top_k"])


# ------------------------------------------------------------------------------ 64-bit results
def _value(fmt, code):
    """The value of a code, from the formats' definition."""
    if fmt == "uint4":
        return float(code)
    if fmt == "int4":
        return float(code if code < 8 else code - 16)
    eb, mb, bias = FLOATS[fmt]
    e, m = (code >> mb) % (1 << eb), code % (1 << mb)
    mag = (1 + m / (1 << mb)) * 2.0 ** (e - bias) if e else m / (1 << mb) * 2.0 ** (1 - bias)
    return -mag if code >> (eb + mb) else mag


def _matrix(packed, case, i, rows, k):
    """Expert i's weight in 64 bits."""
    data, scales = packed
    bits = BITS[case["fmt"]]
    n = rows * k * bits // 8
    stream = data[i * n:(i + 1) * n]
    if bits == 4:
        code = torch.stack((stream % 16, torch.div(stream, 16, rounding_mode="floor")), -1)
    else:
        three = stream.view(-1, 3).int()
        word = three[:, 0] + 256 * three[:, 1] + 65536 * three[:, 2]
        code = torch.stack([torch.div(word, 64 ** j, rounding_mode="floor") % 64 for j in range(4)], -1)
    table = torch.tensor([_value(case["fmt"], c) for c in range(1 << bits)], dtype=torch.float64, device=DEVICE)
    scale = scales[i].double()
    scale = torch.exp2(scale - 127) if case["scales"] == "e8m0" else scale
    return table[code.int()].view(rows, k) * scale.repeat_interleave(case["group"], -1)


def exact(case, seed):
    kind, inputs = case["kind"], _inputs(case, seed)
    if kind == "route":
        x = inputs["logits"].double()
        p = torch.softmax(x, -1) if case["score"] == "softmax" else torch.sigmoid(x)
        key = p if inputs["bias"] is None else p + inputs["bias"].double()
        per = case["experts"] // case["groups"]
        if case["top_groups"] < case["groups"]:
            held = key.view(len(key), case["groups"], per)
            keep = held.topk(min(2, per), -1).values.sum(-1).topk(case["top_groups"], -1).indices
            allowed = torch.zeros(held.shape[:2], device=DEVICE).scatter_(1, keep, 1.0).repeat_interleave(per, 1)
            key = torch.where(allowed > 0, key, torch.full_like(key, -1e9))
        # the chosen scores in descending order of the key; equal keys are equal scores but for the bias
        chosen = p.gather(1, torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :case["top_k"]])
        total = chosen.sum(-1, keepdim=True) if case["renormalize"] else torch.ones_like(chosen[:, :1])
        return dict(ids=None, weights=chosen * (case["scale"] / total))
    if kind == "logprobs":
        x = inputs["logits"].double()
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        return dict(logprobs=logp.gather(1, inputs["tokens"].long()[:, None])[:, 0], ranks=None,
                    entropy=-(logp.exp() * logp).sum(-1), top_ids=None, top_logprobs=logp.topk(case["top"], -1).values)
    x, ids, weights = inputs["x"].double(), inputs["ids"].long(), inputs["weights"].double()
    d, f = case["hidden"], case["ffn"]
    y = torch.zeros((case["tokens"], d), dtype=torch.float64, device=DEVICE)
    for i in range(case["experts"]):
        t, j = torch.nonzero(ids == i, as_tuple=True)
        if not len(t):
            continue
        both = x[t] @ _matrix(inputs["gate_up"], case, i, 2 * f, d).T
        gate, up = both[:, 0::2], both[:, 1::2]
        out = (gate * torch.sigmoid(gate) * up) @ _matrix(inputs["down"], case, i, d, f).T
        y.index_add_(0, t, out * weights[t, j, None])
    return y
