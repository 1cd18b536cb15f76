"""The operators of a decoder's serving step, as measurable cases.

Every case is one call of an operator that a serving loop makes between its matrix products:

* ``rotate``: rotary positions for query and key heads, read out of stacked q|k|v rows;
* ``append``: new keys (rotated) and values quantised into a paged cache as they are written, the
  queries rotated beside them, and what the cache now holds handed back for the prompt's attention;
* ``read``: a stretch of the cache read back in a floating type;
* ``attend``: grouped-query attention of new tokens over the quantised cache;
* ``shared``: the same for a batch whose sequences begin with one long common prefix;
* ``sample``: a token per row of logits, from temperature, top-k, top-p and min-p and given random numbers.

The cache holds pages of ``page`` positions.  Codes lie as [pages, kv_heads, page, head_dim] (fp8_e4m3
one a byte, fp4_e2m1 two a byte, the lower nibble first), with one power-of-two scale per 32 values of a
head, stored as the exponent plus 127 in [pages, kv_heads, head_dim / 32, page].  Row b of the page table
names the pages of sequence b.
"""

import math
import sys
from pathlib import Path

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bfloat16": torch.bfloat16, "float16": torch.float16, "float32": torch.float32}
BLOCK = 32  # values that share a scale
# per format: bits of a code, mantissa bits, exponent of the smallest normal, of the largest, largest value
FORMATS = {"fp8_e4m3": (8, 3, -6, 8, 448.0), "fp4_e2m1": (4, 1, 0, 2, 6.0)}
FP4_VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # one new token of each of eight sequences: 32 query and 8 key heads, the smallest call
        dict(name="rotate_decode", kind="rotate", dtype="float32", batch=8, tokens=1, heads=40, head_dim=128, rotary_dim=128,
             layout="half", scaling="none", base=10000.0, start=900),
        # a prompt continued far behind the trained length: adjacent pairs over half of each head, scaled frequencies
        dict(name="rotate_prompt_far", kind="rotate", dtype="bfloat16", batch=2, tokens=4096, heads=40, head_dim=128,
             rotary_dim=64, layout="interleaved", scaling="yarn", base=500000.0, start=120000),
        # the cache write of one decode step for eight sequences
        dict(name="append_decode", kind="append", dtype="float32", batch=8, tokens=1, heads=32, kv_heads=8, head_dim=128,
             page=64, k_format="fp8_e4m3", v_format="fp8_e4m3", start=1000),
        # the cache write of two prompts of odd length, 8-bit keys and 4-bit values
        dict(name="append_prompts", kind="append", dtype="bfloat16", batch=2, tokens=4001, heads=32, kv_heads=8,
             head_dim=128, page=64, k_format="fp8_e4m3", v_format="fp4_e2m1", start=0),
        # a conversation's cache decoded for a program that wants it in bf16
        dict(name="read_long", kind="read", dtype="bfloat16", batch=2, first=37, count=16001, kv_heads=8, head_dim=128,
             page=64, k_format="fp8_e4m3", v_format="fp4_e2m1"),
        # one sequence, one token, a short cache: what counts is latency
        dict(name="attend_one", kind="attend", dtype="float32", batch=1, tokens=1, heads=32, kv_heads=8, head_dim=128, page=64,
             k_format="fp8_e4m3", v_format="fp8_e4m3", length=1000, ragged=0.0, shared=0),
        # sixteen sequences of unequal length, the longest of 32k positions: the cache's bytes bound it
        dict(name="attend_ragged_32k", kind="attend", dtype="bfloat16", batch=16, tokens=1, heads=32, kv_heads=8, head_dim=128,
             page=64, k_format="fp8_e4m3", v_format="fp8_e4m3", length=32700, ragged=0.9, shared=0),
        # a chunk of a long prompt over what is cached of it, 4-bit cache
        dict(name="attend_chunk", kind="attend", dtype="bfloat16", batch=1, tokens=512, heads=32, kv_heads=8, head_dim=128,
             page=64, k_format="fp4_e2m1", v_format="fp4_e2m1", length=8500, ragged=0.0, shared=0),
        # eight sequences on one system prompt
        dict(name="shared_b8", kind="shared", dtype="float16", batch=8, tokens=1, heads=32, kv_heads=8, head_dim=128, page=64,
             k_format="fp8_e4m3", v_format="fp8_e4m3", length=2300, ragged=0.1, shared=2048),
        # many sequences on one long document
        dict(name="shared_b64_16k", kind="shared", dtype="bfloat16", batch=64, tokens=1, heads=32, kv_heads=8, head_dim=128,
             page=64, k_format="fp8_e4m3", v_format="fp8_e4m3", length=16900, ragged=0.03, shared=16384),
        # one sequence's next token, every filter on
        dict(name="sample_one", kind="sample", dtype="float32", rows=1, vocab=32000, temperature=0.8, top_k=50, top_p=0.9,
             min_p=0.02),
        # a large batch over a large vocabulary, nucleus sampling alone, 16-bit logits full of ties
        dict(name="sample_b64", kind="sample", dtype="bfloat16", rows=64, vocab=131072, temperature=1.0, top_k=0, top_p=0.95,
             min_p=0.0),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["rotate", "append", "append", "read", "attend", "attend", "attend", "shared", "shared", "sample",
                       "sample"])
    dtype = rng.choice(["bfloat16", "float16", "float32"])
    if kind == "sample":
        vocab = _log_int(rng, 500, 131072)
        return dict(kind=kind, dtype=dtype, rows=min(_log_int(rng, 1, 64), max(1, (1 << 22) // vocab)), vocab=vocab,
                    temperature=rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]), top_k=rng.choice([0, 0, 1, 20, 50, 400]),
                    top_p=rng.choice([1.0, 0.95, 0.9, 0.5]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]))
    head_dim = rng.choice([64, 128, 128])
    if kind == "rotate":
        batch = _log_int(rng, 1, 32)
        return dict(kind=kind, dtype=dtype, batch=batch, tokens=_log_int(rng, 1, max(1, 8192 // batch)),
                    heads=rng.randint(1, 40), head_dim=head_dim, rotary_dim=rng.choice([head_dim, head_dim // 2, 32]),
                    layout=rng.choice(["half", "interleaved"]), scaling=rng.choice(["none", "linear", "ntk", "yarn"]),
                    base=rng.choice([10000.0, 500000.0]), start=_log_int(rng, 1, 1000000) - 1)
    kv_heads, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 7, 8])
    cache = dict(dtype=dtype, kv_heads=kv_heads, head_dim=head_dim, page=rng.choice([16, 64, 128]),
                 k_format=rng.choice(["fp8_e4m3", "fp8_e4m3", "fp4_e2m1"]),
                 v_format=rng.choice(["fp8_e4m3", "fp4_e2m1"]))
    heads = min(kv_heads * group, 32)
    heads -= heads % kv_heads
    if kind == "append":
        batch = _log_int(rng, 1, 32)
        return dict(kind=kind, batch=batch, tokens=_log_int(rng, 1, max(1, 8000 // batch)), heads=heads,
                    start=rng.randint(0, 3000), **cache)
    if kind == "read":
        batch = _log_int(rng, 1, 16)
        return dict(kind=kind, batch=batch, first=rng.randint(0, 200), count=_log_int(rng, 1, 32000 // batch), **cache)
    if kind == "attend":
        batch = _log_int(rng, 1, 32)
        tokens = rng.choice([1, 1, 1, 2, 5, _log_int(rng, 2, 600)]) if batch <= 4 else rng.choice([1, 1, 3])
        most = min(33000, 200000 // batch, 4000000 // (batch * tokens))  # (token, position) pairs of the largest listed
        return dict(kind=kind, batch=batch, tokens=tokens, heads=heads, length=_log_int(rng, max(tokens, 16), most),
                    ragged=rng.choice([0.0, 0.5, 0.9]), shared=0, **cache)
    batch = _log_int(rng, 2, 64)
    shared = cache["page"] * _log_int(rng, 4, 16384 // cache["page"])
    return dict(kind=kind, batch=batch, tokens=rng.choice([1, 1, 2]) if batch <= 32 else 1, heads=heads, ragged=0.02,
                length=int(shared * 1.03) + _log_int(rng, 2, 500), shared=shared, **cache)


# ------------------------------------------------------------------------------------- inputs
def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(seed)
    return g


def _randn(g, *shape):
    return torch.randn(shape, device=DEVICE, generator=g)


def _scaling(case):
    """Arguments of the frequency scaling that a long-context model's configuration states."""
    return {"none": None, "linear": dict(kind="linear", factor=4.0), "ntk": dict(kind="ntk", factor=4.0),
            "yarn": dict(kind="yarn", factor=16.0, trained=8192)}[case.get("scaling", "none")]


def _pages_of(case, positions):
    return -(-positions // case["page"])


def _lengths(case):
    """Cached positions of each sequence, the new tokens among them: from the longest down to a share of it."""
    b = case["batch"]
    low = max(case["tokens"], case["shared"] + case["tokens"])
    return [max(low, round(case["length"] * (1 - case["ragged"] * ((5 * i) % b) / b))) for i in range(b)]


def _table(g, batch, per_row, shared_pages=0):
    """A page table whose pages lie in no order; the first shared_pages of every row are the same ones."""
    pages = shared_pages + batch * (per_row - shared_pages)
    order = torch.randperm(pages, device=DEVICE, generator=g).to(torch.int32)
    rows = order[shared_pages:].reshape(batch, per_row - shared_pages)
    return torch.cat((order[:shared_pages].expand(batch, -1), rows), 1).contiguous(), pages


def _exponent(x):
    """floor(log2 |x|), of any finite x but 0."""
    return torch.frexp(x)[1] - 1


def _quantised(x, fmt):
    """x [..., head_dim] rounded to the format: the codes' values, and each block's exponent."""
    _, mant, e_min, e_max, largest = FORMATS[fmt]
    blocks = x.unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1, keepdim=True)
    shared = torch.where(amax > 0, _exponent(amax) - e_max, torch.zeros_like(amax, dtype=torch.int32)).clamp(-127, 127)
    v = torch.ldexp(blocks, -shared)
    step = torch.where(v == 0, torch.full_like(shared, e_min), _exponent(v)).clamp(min=e_min) - mant
    v = torch.ldexp(torch.round(torch.ldexp(v, -step)), step).clamp(-largest, largest)
    return v.flatten(-2), shared.squeeze(-1)


def _bytes_of(v, fmt):
    """Codes' values [..., head_dim] as stored bytes."""
    if fmt == "fp8_e4m3":
        return v.to(torch.float8_e4m3fn).view(torch.uint8)
    levels = torch.tensor(FP4_VALUES, device=v.device)
    code = torch.searchsorted(levels, v.abs().contiguous()).to(torch.uint8) | ((v < 0).to(torch.uint8) << 3)
    return code[..., 0::2] | (code[..., 1::2] << 4)


def _stored(g, case, pages, spread):
    """A filled store: random values with some channels larger than others, quantised."""
    heads, hd = case["kv_heads"], case["head_dim"]
    data, scales = [], []
    for fmt in (case["k_format"], case["v_format"]):
        channel = torch.exp(spread * _randn(g, heads, 1, hd))
        d = torch.empty((pages, heads, case["page"], hd * FORMATS[fmt][0] // 8), dtype=torch.uint8, device=DEVICE)
        s = torch.empty((pages, heads, hd // BLOCK, case["page"]), dtype=torch.uint8, device=DEVICE)
        step = max(1, (1 << 26) // (heads * case["page"] * hd))
        for p in range(0, pages, step):
            n = min(step, pages - p)
            v, e = _quantised(_randn(g, n, heads, case["page"], hd) * channel, fmt)
            d[p:p + n] = _bytes_of(v, fmt)
            s[p:p + n] = (e + 127).to(torch.uint8).transpose(-1, -2)
        data.append(d)
        scales.append(s)
    return dict(k_data=data[0], k_scales=scales[0], v_data=data[1], v_scales=scales[1])


def _inputs(case, seed):
    """What the operator takes, as plain tensors."""
    g, kind, dt = _generator(seed), case["kind"], DTYPES[case["dtype"]]
    if kind == "sample":
        rows = case["rows"]
        logits = (_randn(g, rows, case["vocab"]) * 3).to(dt)
        u = torch.rand(rows, device=DEVICE, generator=g)
        # the parameters that requests of one batch set differ from row to row
        t = torch.full((rows,), case["temperature"], device=DEVICE) * torch.linspace(1.0, 1.25, rows, device=DEVICE)
        ks = torch.full((rows,), case["top_k"], dtype=torch.int32, device=DEVICE)
        ps = (torch.full((rows,), case["top_p"], device=DEVICE) if case["top_p"] >= 1 else
              case["top_p"] - 0.1 * torch.linspace(0, 1, rows, device=DEVICE))
        return dict(logits=logits, u=u, temperature=t, top_k=ks, top_p=ps,
                    min_p=torch.full((rows,), case["min_p"], device=DEVICE))
    b, t, hd = case["batch"], case.get("tokens", 1), case["head_dim"]
    if kind == "rotate":
        start = case["start"] + 7 * torch.arange(b, dtype=torch.int32, device=DEVICE)
        rows = _randn(g, b, t, case["heads"] + 8, hd).to(dt)  # the value heads of stacked q|k|v rows stay as they are
        return dict(x=rows[:, :, :case["heads"]], start=start)
    hk = case["kv_heads"]
    if kind == "append":
        start = case["start"] + 3 * torch.arange(b, dtype=torch.int32, device=DEVICE)
        table, pages = _table(g, b, _pages_of(case, case["start"] + 3 * (b - 1) + t))
        h = case["heads"]
        qkv = _randn(g, b, t, h + 2 * hk, hd).to(dt)
        return dict(q=qkv[:, :, :h], k=qkv[:, :, h:h + hk], v=qkv[:, :, h + hk:], table=table, start=start, pages=pages)
    if kind == "read":
        table, pages = _table(g, b, _pages_of(case, case["first"] + case["count"]))
        first = torch.full((b,), case["first"], dtype=torch.int32, device=DEVICE)
        return dict(table=table, first=first, pages=pages, **_stored(g, case, pages, 0.5))
    lengths = _lengths(case)
    table, pages = _table(g, b, _pages_of(case, max(lengths)), case["shared"] // case["page"])
    return dict(q=(_randn(g, b, t, case["heads"], hd) * 1.5).to(dt), table=table, pages=pages,
                lengths=torch.tensor(lengths, dtype=torch.int32, device=DEVICE), **_stored(g, case, pages, 0.5))


def prepare(case, seed):
    state = dict(case=case, **_inputs(case, seed))
    if case["kind"] in ("rotate", "append"):
        state["freq"], state["gain"] = _frequencies(case)
    if own:
        path = str(Path(__file__).resolve().parent.parent / "tinygrad-dx12_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        if case["kind"] == "sample":
            from tinygrad_mi355x.sampling import sample

            state["sample"] = sample
            return state
        if case["kind"] in ("rotate", "append"):
            from tinygrad_mi355x.rotary import Rotary

            state["rotary"] = Rotary(case["head_dim"], case.get("rotary_dim"), base=case.get("base", 10000.0),
                                     layout=case.get("layout", "half"), scaling=_scaling(case), device=DEVICE)
        if case["kind"] != "rotate":
            from tinygrad_mi355x.kv_cache import PackedKVCache

            cache = PackedKVCache(state["pages"], case["kv_heads"], case["head_dim"], page_size=case["page"],
                                  k_format=case["k_format"], v_format=case["v_format"], device=DEVICE)
            for name in ("k_data", "k_scales", "v_data", "v_scales"):
                if name in state:
                    getattr(cache, name).copy_(state[name])
            state["cache"] = cache
    elif case["kind"] == "append":  # the plain form's store, empty
        hk, hd = case["kv_heads"], case["head_dim"]
        for n, fmt in (("k", case["k_format"]), ("v", case["v_format"])):
            state[n + "_data"] = torch.zeros((state["pages"], hk, case["page"], hd * FORMATS[fmt][0] // 8),
                                             dtype=torch.uint8, device=DEVICE)
            state[n + "_scales"] = torch.zeros((state["pages"], hk, hd // BLOCK, case["page"]), dtype=torch.uint8,
                                               device=DEVICE)
    return state


# ------------------------------------------------------------------------------------ one pass
def run(state):
    case, kind = state["case"], state["case"]["kind"]
    if own:
        if kind == "sample":
            return state["sample"](state["logits"], state["u"], temperature=state["temperature"], top_k=state["top_k"],
                                   top_p=state["top_p"], min_p=state["min_p"])
        if kind == "rotate":
            return state["rotary"].rotate(state["x"], state["start"])
        cache = state["cache"]
        if kind == "append":
            done = cache.append(state["k"], state["v"], state["table"], state["start"], rotary=state["rotary"], q=state["q"],
                                seen=DTYPES[case["dtype"]])
            return dict(q=done.q, k=done.k, v=done.v)
        if kind == "read":
            k, v = cache.read(state["table"], state["first"], case["count"], DTYPES[case["dtype"]])
            return dict(k=k, v=v)
        return cache.attend(state["q"], state["table"], state["lengths"], shared=case["shared"])
    if kind == "sample":
        return _plain_sample(state)
    if kind == "rotate":
        return _plain_rotate(state["x"], state["start"], state["freq"], state["gain"], case["layout"]).to(state["x"].dtype)
    if kind == "append":
        return _plain_append(state)
    if kind == "read":
        pos = state["first"][:, None].long() + torch.arange(case["count"], device=DEVICE)
        return {n: _plain_read(state, n, pos).to(DTYPES[case["dtype"]]) for n in ("k", "v")}
    return _plain_attend(state)


# ------------------------------------------------------------------------------- plain forms
def _frequencies(case):
    """Radians per position of every rotated pair, in 64 bits, and the gain on the rotated values."""
    n = case.get("rotary_dim", case["head_dim"])
    base, gain, scaling = case.get("base", 10000.0), 1.0, _scaling(case)
    i = torch.arange(n // 2, dtype=torch.float64, device=DEVICE)
    if scaling and scaling["kind"] == "ntk":  # a larger base: the slowest pair slows by the factor, the fastest stays
        base = base * scaling["factor"] ** (n / (n - 2))
    freq = base ** (-2 * i / n)
    if scaling and scaling["kind"] == "linear":
        freq = freq / scaling["factor"]
    if scaling and scaling["kind"] == "yarn":
        # pairs that turn over 32 times in the trained length stay, under once are slowed, a ramp between
        at = [n * math.log(scaling["trained"] / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), n - 1)
        slowed = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        freq = freq * (1 - slowed) + freq / scaling["factor"] * slowed
        gain = 0.1 * math.log(scaling["factor"]) + 1.0
    return freq, gain


def _plain_rotate(x, start, freq, gain, layout):
    """x [B, T, H, D] with the leading 2 * len(freq) values of each head rotated: token t of sequence b is at
    position start[b] + t.  Angles and products in 64 bits, rounded once to 32."""
    pos = start[:, None].double() + torch.arange(x.shape[1], device=DEVICE)
    angle = (pos[..., None] * freq)[:, :, None]
    c, s = angle.cos() * gain, angle.sin() * gain
    n = 2 * freq.numel()
    head, rest = x[..., :n].double(), x[..., n:].float()
    if layout == "half":
        a, b = head[..., :n // 2], head[..., n // 2:]
        turned = torch.cat((a * c - b * s, b * c + a * s), -1)
    else:
        a, b = head[..., 0::2], head[..., 1::2]
        turned = torch.stack((a * c - b * s, b * c + a * s), -1).flatten(-2)
    return torch.cat((turned.float(), rest), -1)


def _plain_append(state):
    case, dt = state["case"], DTYPES[state["case"]["dtype"]]
    turn = (state["start"], state["freq"], state["gain"], "half")
    pos = state["start"][:, None].long() + torch.arange(case["tokens"], device=DEVICE)
    page, slot = state["table"].gather(1, pos // case["page"]).long(), pos % case["page"]
    out = dict(q=_plain_rotate(state["q"], *turn).to(dt))
    new = dict(k=_plain_rotate(state["k"], *turn), v=state["v"].float())
    for n, fmt in (("k", case["k_format"]), ("v", case["v_format"])):
        codes, shared = _quantised(new[n], fmt)
        state[n + "_data"][page, :, slot] = _bytes_of(codes, fmt)
        state[n + "_scales"][page, :, :, slot] = (shared + 127).to(torch.uint8)
        out[n] = torch.ldexp(codes, shared.repeat_interleave(BLOCK, -1)).to(dt)
    return out


def _plain_read(state, name, pos):
    """The values of positions pos [B, n] of every sequence, [B, n, kv_heads, head_dim] in 32 bits."""
    case = state["case"]
    page, slot = state["table"].gather(1, pos // case["page"]).long(), pos % case["page"]
    data, scales = state[name + "_data"][page, :, slot], state[name + "_scales"][page, :, :, slot]
    if case[name + "_format"] == "fp8_e4m3":
        v = data.view(torch.float8_e4m3fn).float()
    else:
        code = torch.stack((data & 15, data >> 4), -1).flatten(-2)
        v = torch.tensor(FP4_VALUES + [-x for x in FP4_VALUES], device=DEVICE)[code.int()]
    return torch.ldexp(v, scales.int().repeat_interleave(BLOCK, -1) - 127)


def _plain_attend(state):
    case, q, lengths = state["case"], state["q"], state["lengths"].long()
    b, t, h, hd = q.shape
    hk, shared = case["kv_heads"], case["shared"]
    g = h // hk
    rows = (q.float() / math.sqrt(hd)).reshape(b, t, hk, g, hd).permute(0, 2, 1, 3, 4).reshape(b, hk, t * g, hd)
    last = (lengths[:, None] - t + torch.arange(t, device=DEVICE)).repeat_interleave(g, 1)[:, None, :, None]
    capacity = state["table"].shape[1] * case["page"]
    pos = torch.arange(shared, capacity, device=DEVICE)
    k, v = (_plain_read(state, n, pos.expand(b, -1)).transpose(1, 2).contiguous() for n in ("k", "v"))
    scores = torch.matmul(rows, k.transpose(2, 3).contiguous()).masked_fill(pos > last, -math.inf)
    if shared:  # the common positions, read once: every sequence's rows of a head against them
        common = dict(case=case, table=state["table"][:1], **{n: state[n] for n in ("k_data", "k_scales", "v_data", "v_scales")})
        first = torch.arange(shared, device=DEVICE)[None]
        ck, cv = (_plain_read(common, n, first)[0].transpose(0, 1).contiguous() for n in ("k", "v"))
        flat = rows.transpose(0, 1).reshape(hk, b * t * g, hd)
        cs = torch.matmul(flat, ck.transpose(1, 2).contiguous()).reshape(hk, b, t * g, shared).transpose(0, 1)
        scores = torch.cat((cs.masked_fill(first[0] > last, -math.inf), scores), -1)
    top = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p[..., shared:].contiguous(), v)
    if shared:
        cp = p[..., :shared].transpose(0, 1).reshape(hk, b * t * g, shared)
        out = out + torch.matmul(cp, cv).reshape(hk, b, t * g, hd).transpose(0, 1)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.reshape(b, hk, t, g, hd).permute(0, 2, 1, 3, 4).reshape(b, t, h, hd).to(q.dtype)


def _plain_sample(state):
    """The weights in 64 bits: a cut or a draw that falls next to a border is decided by their last places."""
    x = state["logits"].double()
    rows, n = x.shape
    order = torch.sort(x, dim=-1, descending=True, stable=True)  # ties: the lower index first
    t = state["temperature"].double()[:, None]
    greedy = ~(t > 0)
    w = torch.exp((order.values - order.values[:, :1]) / torch.where(greedy, torch.ones_like(t), t))
    rank = torch.arange(n, device=DEVICE)
    k = state["top_k"].long()[:, None]
    w = torch.where((k <= 0) | (rank < k), w, torch.zeros_like(w))
    before = w.cumsum(-1) - w
    p = state["top_p"].double()[:, None]
    w = torch.where((p >= 1) | (before < p * w.sum(-1, keepdim=True)) | (rank == 0), w, torch.zeros_like(w))
    w = torch.where((w >= state["min_p"].double()[:, None]) & (~greedy | (rank == 0)), w, torch.zeros_like(w))
    weights = torch.zeros_like(w).scatter_(1, order.indices, w)  # back in the order of the vocabulary
    sums = weights.cumsum(-1)
    target = state["u"].double()[:, None] * sums[:, -1:]
    return ((sums > target) & (weights > 0)).to(torch.uint8).argmax(-1).to(torch.int32)


# --------------------------------------------------------------------------------- what it takes
def _row_bytes(case, name):
    """Stored bytes of one position of one head."""
    return case["head_dim"] * FORMATS[case[name + "_format"]][0] / 8 + case["head_dim"] / BLOCK


def work(case):
    kind, size = case["kind"], DTYPES[case["dtype"]].itemsize
    if kind == "sample":
        return dict(bytes=case["rows"] * (case["vocab"] * size + 24), flops=2 * case["rows"] * case["vocab"])
    b, t, hd = case["batch"], case.get("tokens", 1), case["head_dim"]
    if kind == "rotate":
        n = b * t * case["heads"]
        return dict(bytes=2 * n * hd * size + 4 * b, flops=3 * n * case["rotary_dim"])
    hk = case["kv_heads"]
    stored = _row_bytes(case, "k") + _row_bytes(case, "v")
    if kind == "append":
        q, kv = b * t * case["heads"] * hd, b * t * hk * hd
        return dict(bytes=2 * q * size + 4 * kv * size + b * t * hk * stored, flops=3 * (q + kv) + 6 * kv)
    if kind == "read":
        n = b * case["count"] * hk
        return dict(bytes=n * (stored + 2 * hd * size), flops=2 * n * hd)
    lengths = _lengths(case)
    cached = sum(lengths) - (b - 1) * case["shared"]  # the common positions are read once
    pairs = sum(n * t - t * (t - 1) // 2 for n in lengths)  # (token, position) pairs that meet
    return dict(bytes=cached * hk * stored + 2 * b * t * case["heads"] * hd * size, flops=4 * pairs * case["heads"] * hd)


# ------------------------------------------------------------------------------ 64-bit results
def _value_tables():
    """The value of every code, from the formats' definition."""
    e4m3 = []
    for c in range(256):
        e, f = (c >> 3) & 15, c & 7
        mag = math.nan if c & 127 == 127 else math.ldexp(8 + f, e - 10) if e else math.ldexp(f, -9)
        e4m3.append(-mag if c >> 7 else mag)
    e2m1 = []
    for c in range(16):
        e, f = (c >> 1) & 3, c & 1
        mag = math.ldexp(2 + f, e - 2) if e else 0.5 * f
        e2m1.append(-mag if c >> 3 else mag)
    return {"fp8_e4m3": e4m3, "fp4_e2m1": e2m1}


def _decoded(inputs, case, name):
    """The whole store in 64 bits, [pages, page, kv_heads, head_dim]."""
    fmt, data = case[name + "_format"], inputs[name + "_data"]
    if FORMATS[fmt][0] == 4:
        data = torch.stack((data & 15, data >> 4), -1).flatten(-2)
    values = torch.tensor(_value_tables()[fmt], dtype=torch.float64, device=DEVICE)[data.int()]
    scale = torch.exp2(inputs[name + "_scales"].double() - 127).transpose(-1, -2).repeat_interleave(BLOCK, -1)
    return (values * scale).transpose(1, 2)


def _turned(x, start, freq, gain, layout):
    """The rotation in 64 bits, as a product of complex numbers."""
    n = 2 * freq.numel()
    pos = (start[:, None] + torch.arange(x.shape[1], device=DEVICE)).double()
    unit = torch.polar(torch.full_like(pos, gain)[..., None].expand(*pos.shape, n // 2).contiguous(), pos[..., None] * freq)
    x = x.double()
    pairs = x[..., :n].unflatten(-1, (2, n // 2)).transpose(-1, -2) if layout == "half" else x[..., :n].unflatten(-1, (n // 2, 2))
    z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * unit[:, :, None])
    turned = z.transpose(-1, -2).flatten(-2) if layout == "half" else z.flatten(-2)
    return torch.cat((turned, x[..., n:]), -1)


def _nearest(x, fmt):
    """x in 64 bits as the cache holds it: the nearest value of the format times its block's scale."""
    levels = sorted({abs(v) for v in _value_tables()[fmt] if v == v})
    levels = torch.tensor(levels, dtype=torch.float64, device=DEVICE)
    blocks = x.unflatten(-1, (-1, BLOCK))
    amax = blocks.abs().amax(-1, keepdim=True)
    power = torch.where(amax > 0, torch.floor(torch.log2(amax.clamp(min=1e-300))) - FORMATS[fmt][3], torch.zeros_like(amax))
    scale = torch.exp2(power.clamp(-127, 127))
    a = blocks.abs() / scale
    upper = torch.searchsorted(levels, a.contiguous()).clamp(1, len(levels) - 1)
    low, high = levels[upper - 1], levels[upper]
    mid = (low + high) / 2
    up = (a > mid) | ((a == mid) & (upper % 2 == 0))  # levels ascend with their codes: an even one on a tie
    return (torch.where(up, high, low) * torch.sign(blocks) * scale).flatten(-2)


def exact(case, seed):
    kind, inputs = case["kind"], _inputs(case, seed)
    if kind == "sample":
        return None  # whole numbers
    if kind == "rotate":
        return _turned(inputs["x"], inputs["start"], *_frequencies(case), case["layout"])
    if kind == "append":
        turn = (inputs["start"], *_frequencies(case), "half")
        return dict(q=_turned(inputs["q"], *turn), k=_nearest(_turned(inputs["k"], *turn).float().double(), case["k_format"]),
                    v=_nearest(inputs["v"].double(), case["v_format"]))
    if kind == "read":
        got = {}
        for n in ("k", "v"):
            store = _decoded(inputs, case, n)
            rows = store[inputs["table"].long()].flatten(1, 2)
            got[n] = rows[:, case["first"]:case["first"] + case["count"]].contiguous()
            del store, rows
        return got
    q = inputs["q"].double()
    b, t, h, hd = q.shape
    hk = case["kv_heads"]
    out = torch.zeros_like(q)
    for i, n in enumerate(_lengths(case)):  # a sequence at a time, its prefix among its own positions
        own_pages = inputs["table"][i, :_pages_of(case, n)].long()
        part = {x: inputs[x][own_pages] for x in ("k_data", "k_scales", "v_data", "v_scales")}
        k, v = (_decoded(part, case, x).flatten(0, 1)[:n].transpose(0, 1).contiguous() for x in ("k", "v"))
        blocked = torch.arange(n, device=DEVICE)[None] > torch.arange(n - t, n, device=DEVICE)[:, None]
        for j in range(h):
            kh = j * hk // h
            s = (q[i, :, j] @ k[kh].T / math.sqrt(hd)).masked_fill(blocked, -math.inf)
            out[i, :, j] = torch.softmax(s, -1) @ v[kh]
    return out
