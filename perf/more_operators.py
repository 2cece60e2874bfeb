"""The operators of a serving step over a key/value cache held in 4 bits, as cases of known size, in their plain form and in 64 bits.

A case is one pass of one kind:

  rope       queries and keys turned by their positions: either layout of the pairs, a part of the head, frequencies scaled for long contexts;
  append     new rows of many sequences go into their pages (turned on the way, queries with them), and are read back as values;
  attention  the new rows of many sequences attend to what the cache holds of their sequence up to their own slot; with log-sum-exp;
  weights    what weight those rows gave each cached key, summed over the rows and the heads of a group, is added to a running sum;
  evict      every sequence and kv head keeps its first, its last and its heaviest rows, which move to the front of its pages.

The cache: pages of integers from -7 to 7, stored as n + 8 in 4 bits, two neighbouring dims in a byte (the even one low), [page][kv head][token][dim / 2]; for every 16 dims
of a row a scale in e4m3, [page][kv head][token][dim / 16]; for every kv head a 32-bit scale. A value is integer x scale x the head's scale. Row r of sequence i
lies in slot ctx[i] + r - row_start[i]; the page table says where a sequence's pages lie. A row's position may be another number than its slot.

Lengths follow from the case alone; the values, the order of the pages and the positions come from the seed."""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
BLOCK = 16


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    def rope(name, type, rows, heads, kv, dim, rot, layout, theta, scaling, factor, original, inverse=False):
        return {"name": name, "kind": "rope", "type": type, "rows": rows, "heads": heads, "kv": kv, "dim": dim, "rot": rot, "layout": layout,
                "theta": theta, "scaling": scaling, "factor": factor, "original": original, "inverse": inverse}

    def seqs(name, kind, type, heads, kv, dim, page, n, new_lo, new_hi, ctx_lo, ctx_hi, **more):
        return dict({"name": name, "kind": kind, "type": type, "heads": heads, "kv": kv, "dim": dim, "page": page, "seqs": n, "new_lo": new_lo,
                     "new_hi": new_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi}, **more)

    return [
        # one user's next token on the TinyLlama shape: latency
        rope("rope-one", "f32", 1, 32, 4, 64, 64, "half", 10000.0, "none", 1.0, 0),
        # prompts far behind the trained length, neighbouring pairs, three quarters of the head turned
        rope("rope-prompts", "bf16", 8192, 32, 8, 128, 96, "interleaved", 500000.0, "yarn", 16.0, 8192),
        # continuous batching on the 7B shape: 64 users' next tokens, whose caches have lost rows
        seqs("append-batch", "append", "f32", 32, 32, 128, 16, 64, 1, 1, 128, 4096, layout="half", rot=128, gone=5000),
        # prompts of unequal length arriving together, some behind a cached prefix that ends inside a page
        seqs("append-prompts", "append", "bf16", 32, 8, 128, 32, 5, 300, 2100, 0, 1300, layout="half", rot=128, gone=0),
        # one user's next token on the TinyLlama shape: latency
        seqs("attend-one", "attention", "f32", 32, 4, 64, 16, 1, 1, 1, 700, 700, window=0),
        # continuous batching, grouped heads: 64 users with 128 to 4096 tokens each
        seqs("attend-batch", "attention", "bf16", 32, 8, 128, 16, 64, 1, 1, 128, 4096, window=0),
        # drafts of four tokens checked behind two very long documents, grouped heads of the 70B shape
        seqs("attend-long", "attention", "f16", 64, 8, 128, 64, 2, 4, 4, 60001, 131000, window=0),
        # long prompts in chunks behind what earlier chunks have left
        seqs("attend-chunks", "attention", "bf16", 32, 8, 128, 32, 3, 700, 2048, 1000, 6100, window=0),
        # the same batch's step: what it looked at
        seqs("weights-batch", "weights", "bf16", 32, 8, 128, 16, 64, 1, 1, 128, 4096, window=0),
        # the last 64 rows of long prompts decide what is kept of them
        seqs("weights-window", "weights", "f16", 32, 8, 128, 32, 3, 64, 64, 3000, 16000, window=0),
        # the batch's contexts are cut to 1024 rows where they have grown past 1280
        seqs("evict-batch", "evict", "bf16", 32, 8, 128, 16, 64, 1, 1, 128, 4096, keep=1024, limit=1280, recent=128, first=4),
        # two very long documents are cut to 16384 rows
        seqs("evict-long", "evict", "bf16", 64, 8, 128, 64, 2, 4, 4, 60001, 131000, keep=16384, limit=16384, recent=512, first=16),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(("rope", "append", "attention", "attention", "weights", "evict"))
    heads, kv, dim = rng.choice(((32, 4, 64), (32, 32, 128), (32, 8, 128), (64, 8, 128), (8, 1, 128), (12, 4, 96)))
    case = {"kind": kind, "type": rng.choice(sorted(DTYPES)), "heads": heads, "kv": kv, "dim": dim}
    layout, rot = rng.choice(("half", "interleaved")), rng.choice((dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)))
    if kind == "rope":
        scaling = rng.choice(("none", "linear", "ntk", "yarn", "llama3"))
        case.update(rows=spread(1, min(8192, 25_000_000 // ((heads + kv) * dim))), layout=layout, rot=max(rot, 4), theta=rng.choice((10000.0, 500000.0)), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice((2.0, 8.0, 3.5)), original=rng.choice((2048, 8192)), inverse=rng.random() < 0.2)
        return case
    case["page"] = rng.choice((16, 16, 32, 64, 128))
    if kind == "append":
        seqs = spread(1, 64)
        new = 1 if rng.random() < 0.4 else spread(2, max(2, 4096 // seqs))
        ctx = spread(1, 8192)
        case.update(layout=layout, rot=rot, gone=rng.choice((0, 0, 100, 20000)))
    elif kind == "evict":
        seqs, new = spread(1, 64), 1
        ctx = spread(64, min(65536, 2 ** 27 // (kv * dim * seqs)))
        keep = max(2, int(ctx * rng.uniform(0.1, 0.9)))
        case.update(keep=keep, limit=rng.choice((keep, min(keep + keep // 8, ctx))), recent=int(keep * rng.uniform(0.0, 0.3)), first=int(keep * rng.uniform(0.0, 0.1)))
    elif rng.random() < 0.6:  # single tokens and drafts
        seqs = spread(1, 64)
        new = rng.choice((1, 1, 1, 2, 5))
        ctx = spread(16, min(65536, 2 ** 28 // (kv * dim * seqs)))
    else:
        seqs = spread(1, 6)
        new = spread(16, 2048 // seqs)
        ctx = spread(1, 4096)
    case.update(seqs=seqs, new_lo=max(1, int(new * rng.uniform(0.3, 1.0))), new_hi=new, ctx_lo=int(ctx * rng.uniform(0.0, 1.0)), ctx_hi=ctx)
    if kind in ("attention", "weights"):
        case["window"] = spread(16, 4096) if rng.random() < 0.2 else 0
    return case


def lengths(case):
    """(context, new rows) of each sequence, spread evenly over the logarithm and put in an order of the case's own."""
    def between(lo, hi, n):
        if n == 1:
            return [hi]
        a, b = math.log(max(lo, 1)), math.log(max(hi, 1))
        return [lo] + [int(round(math.exp(a + (b - a) * i / (n - 1)))) for i in range(1, n - 1)] + [hi]
    n, order = case["seqs"], random.Random(1000 * case["seqs"] + case["ctx_hi"])
    ctx, new = between(case["ctx_lo"], case["ctx_hi"], n), between(case["new_lo"], case["new_hi"], n)
    order.shuffle(ctx)
    order.shuffle(new)
    return list(zip(ctx, new))


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["kind"] == "rope":
        row = (case["heads"] + case["kv"]) * case["dim"]
        return {"bytes": case["rows"] * (2 * row * size + 8), "flops": case["rows"] * (case["heads"] + case["kv"]) * case["rot"] * 3}
    seqs, row, kv_row = lengths(case), case["heads"] * case["dim"], case["kv"] * case["dim"]
    rows = sum(n for _, n in seqs)
    held = 9 / 16 * kv_row  # bytes of a cached row of keys or values
    if case["kind"] == "append":
        # the rows in, the queries out; the rows into the cache, and back as values
        return {"bytes": int(rows * (2 * kv_row * size + 2 * row * size + 2 * held + 2 * held + 2 * kv_row * size)), "flops": rows * 3 * (row + kv_row)}
    if case["kind"] == "evict":
        cells, moved = 0, 0
        for c, n in seqs:
            length = c + n
            if length > case["limit"]:
                cells += length + 3 * case["keep"]  # sums read, the kept ones' and their slots written
                moved += case["keep"] - case["first"]
        return {"bytes": int(cells * case["kv"] * 4 + moved * 4 * held), "flops": cells * case["kv"]}
    w = case["window"]
    pairs = sum(sum(min(c + j + 1, w) if w else c + j + 1 for j in range(n)) for c, n in seqs)
    keys = sum(min(c + n, w + n - 1) if w else c + n for c, n in seqs)
    if case["kind"] == "weights":
        return {"bytes": int(keys * (held + 8 * case["kv"]) + rows * (row * size + 4 * case["heads"])), "flops": 2 * row * pairs}
    return {"bytes": int(keys * 2 * held + 2 * rows * row * size + 4 * rows * case["heads"]), "flops": 4 * row * pairs}


# --------------------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    if case["kind"] == "rope":
        return _prepare_rope(case, dev, g, normal)
    heads, kv, dim, page, dtype = case["heads"], case["kv"], case["dim"], case["page"], DTYPES[case["type"]]
    seqs = lengths(case)
    ctx = torch.tensor([c for c, _ in seqs], dtype=torch.int32, device=dev)
    new = [n for _, n in seqs]
    row_start = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    rows = sum(new)
    # every sequence has pages for its whole context, in no order, and the pool has some more
    need = [-(-(c + n) // page) for c, n in seqs]
    pages, width = sum(need) + 7, max(need)
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(seqs), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    spread = torch.exp(0.7 * normal(1, kv, 1, dim))  # some channels of the keys are larger than others
    s = {"case": case, "ctx": ctx, "row_start": row_start, "table": table, "max_new": max(new)}
    s["k_scale"], s["v_scale"] = 2.0 ** -6 * torch.exp(0.1 * normal(kv)), 2.0 ** -6 * torch.exp(0.1 * normal(kv))
    s["k4"], s["k_block"] = _stored(normal, pages, kv, page, dim, spread, s["k_scale"])
    s["v4"], s["v_block"] = _stored(normal, pages, kv, page, dim, 1.0, s["v_scale"])
    if case["kind"] != "evict":
        s["q"] = normal(rows, heads, dim).to(dtype)
    if case["kind"] == "append":
        s["k"], s["v"] = (normal(rows, kv, dim) * spread[:, :, 0]).to(dtype), normal(rows, kv, dim).to(dtype)
        s["freq"] = _frequencies(10000.0, case["rot"], dev)
        s["positions"] = ctx.long() + (torch.randint(case["gone"], (len(seqs),), generator=g, device=dev) if case["gone"] else 0)
        s["q_out"] = torch.empty_like(s["q"])
        s["k_out"], s["v_out"] = torch.empty_like(s["k"]), torch.empty_like(s["v"])
    elif case["kind"] == "attention":
        s["out"] = torch.empty_like(s["q"])
        s["lse"] = torch.empty(rows, heads, device=dev)
    elif case["kind"] == "weights":
        s["mass"] = torch.rand(len(seqs), kv, width * page, generator=g, device=dev)
        s["lse"] = _sequences(s, lambda i, score: torch.logsumexp(score, -1), heads)
    else:
        # a few keys have most of the weight; some none at all
        cap = width * page
        s["mass"] = torch.exp(2.0 * normal(len(seqs), kv, cap)) * (torch.rand(len(seqs), kv, cap, generator=g, device=dev) < 0.98)
        s["kept"] = torch.empty(len(seqs), kv, case["limit"], dtype=torch.int32, device=dev)
        s["ctx_out"] = torch.empty_like(ctx)
    if own:
        import leafcutterllm_b200 as lc
        s["cache"] = lc.Kv4Cache(s["k4"], s["v4"], s["k_block"], s["v_block"], s["k_scale"], s["v_scale"])
        s["rows"] = lc.Kv8Rows(s["table"], s["ctx"], s["row_start"], s["max_new"])
        if case["kind"] == "append":
            s["turns"] = torch.from_numpy(lc.rope_turns(10000.0, case["rot"]).view("int64")).to(dev)
        elif case["kind"] == "attention":
            s["workspace"] = torch.empty(s["cache"].attention_workspace(s["rows"], s["q"]), dtype=torch.uint8, device=dev)
    return s


def _stored(normal, pages, kv, page, dim, spread, scale):
    """Pages as earlier appends have left them."""
    x = normal(pages, kv, page, dim) * spread
    ints, blocks = _quantised(x, scale[None, :, None])
    return _packed(ints), blocks


def _prepare_rope(case, dev, g, normal):
    rows, dtype = case["rows"], DTYPES[case["type"]]
    q, k = normal(rows, case["heads"], case["dim"]).to(dtype), normal(rows, case["kv"], case["dim"]).to(dtype)
    # stretches of some sequences, far into their documents
    starts = torch.randint(int(case["original"] * case["factor"]) or 4096, (1 + rows // 700,), generator=g, device=dev)
    at = torch.arange(rows, device=dev)
    s = {"case": case, "q": q, "k": k, "positions": starts[at // 700] + at % 700, "q_out": torch.empty_like(q), "k_out": torch.empty_like(k)}
    s["freq"], s["magnitude"] = _scaled(case, dev)
    if own:
        import leafcutterllm_b200 as lc
        turns, s["magnitude"] = lc.rope_turns_scaled(case["theta"], case["rot"], case["scaling"], case["factor"], case["original"])
        s["turns"] = torch.from_numpy(turns.view("int64")).to(dev)
    return s


def _frequencies(theta, rot, dev):
    return torch.tensor([theta ** (-2.0 * d / rot) for d in range(rot // 2)], dtype=torch.float64, device=dev)


def _scaled(case, dev):
    """Frequencies of a context that is longer than the trained one, and what the turned values are multiplied by."""
    theta, rot, factor, original = case["theta"], case["rot"], case["factor"], case["original"]
    f = _frequencies(theta, rot, dev)
    if case["scaling"] == "none":
        return f, 1.0
    if case["scaling"] == "linear":
        return f / factor, 1.0
    if case["scaling"] == "ntk":
        return _frequencies(theta * factor ** (rot / (rot - 2)), rot, dev), 1.0
    if case["scaling"] == "llama3":  # long waves are stretched, short ones stay, a mixture between
        turns = original * f / (2.0 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0.0, 1.0)
        return keep * f + (1.0 - keep) * f / factor, 1.0
    # yarn: the same by the index of the pair, and softer attention
    pair = lambda turns: rot * math.log(original / (turns * 2.0 * math.pi)) / (2.0 * math.log(theta))  # noqa: E731
    low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
    ramp = ((torch.arange(rot // 2, dtype=torch.float64, device=dev) - low) / max(high - low, 0.001)).clamp(0.0, 1.0)
    return f * (1.0 - ramp) + f / factor * ramp, 0.1 * math.log(factor) + 1.0


# --------------------------------------------------------------------------------------------------------------- passes

def run(s):
    return {"rope": _run_rope, "append": _run_append, "attention": _run_attention, "weights": _run_weights, "evict": _run_evict}[s["case"]["kind"]](s)


def _run_rope(s):
    case = s["case"]
    if own:
        import leafcutterllm_b200 as lc
        q, k = lc.rope_dev(s["q"], s["positions"], s["turns"], layout=case["layout"], magnitude=s["magnitude"], inverse=case["inverse"], out=s["q_out"],
                           y=s["k"], y_out=s["k_out"])
        return {"q": q, "k": k}
    freq = -s["freq"] if case["inverse"] else s["freq"]
    return {n: _turned(s[n], s["positions"], freq, case["layout"], s["magnitude"]).to(s[n].dtype) for n in ("q", "k")}


def _run_append(s):
    if own:
        c, rows = s["cache"], s["rows"]
        q = c.append(rows, s["k"], s["v"], turns=s["turns"], q=s["q"], q_out=s["q_out"], positions=s["positions"], layout=s["case"]["layout"])
        k, v = c.read(rows, s["k_out"], s["v_out"])
        return {"q": q, "k": k, "v": v}
    case, page = s["case"], s["case"]["page"]
    seq, j, slot = _places(s["row_start"], s["ctx"], s["k"].shape[0])
    at, token, pos = s["table"].long()[seq, slot // page], slot % page, s["positions"][seq] + j
    turned = lambda x: _turned(x, pos, s["freq"], case["layout"], 1.0)  # noqa: E731
    out = {"q": turned(s["q"]).to(s["q"].dtype)}
    for n, x in (("k", turned(s["k"])), ("v", s["v"].double())):
        ints, blocks = _quantised(x, s[n + "_scale"][None])
        s[n + "4"][at, :, token], s[n + "_block"][at, :, token] = _packed(ints), blocks
        out[n] = _values(s[n + "4"][at, :, token], s[n + "_block"][at, :, token], s[n + "_scale"][None]).to(s[n].dtype)
    return out


def _run_attention(s):
    if own:
        out = s["cache"].attention(s["rows"], s["q"], s["out"], lse=s["lse"], window=s["case"]["window"], workspace=s["workspace"])
        return {"out": out, "lse": s["lse"]}
    out = torch.empty_like(s["q"])
    case = s["case"]

    def weighted(i, score):
        top = score.amax(-1, keepdim=True)
        p = score.sub_(top).exp_()
        total = p.sum(-1, keepdim=True)
        r0, n = s["bounds"][i]
        o = torch.matmul(p.reshape(p.shape[0], -1, p.shape[-1]), _cached(s, i, "v").transpose(0, 1)).reshape(*p.shape[:-1], case["dim"]) / total
        out[r0:r0 + n] = o.permute(2, 0, 1, 3).reshape(n, case["heads"], case["dim"]).to(out.dtype)
        return total.log().add_(top)[..., 0]
    lse = _sequences(s, weighted, case["heads"])
    return {"out": out, "lse": lse}


def _run_weights(s):
    if own:
        return s["cache"].weights(s["rows"], s["q"], s["lse"], s["mass"], window=s["case"]["window"])

    def add(i, score):
        kv, group, n, keys = score.shape
        r0 = s["bounds"][i][0]
        lse = s["lse"][r0:r0 + n].reshape(n, kv, group).permute(1, 2, 0)
        s["mass"][i, :, :keys] += score.sub_(lse[..., None]).exp_().sum((1, 2))
    _sequences(s, add, None)
    return s["mass"]


def _run_evict(s):
    case = s["case"]
    if own:
        kept, ctx = s["cache"].evict(s["rows"], s["mass"], case["keep"], limit=case["limit"], recent=case["recent"], first=case["first"], kept=s["kept"], ctx_out=s["ctx_out"])
        return {"kept": kept, "ctx": ctx, "mass": s["mass"], "k": s["k4"], "v": s["v4"], "k_block": s["k_block"], "v_block": s["v_block"]}
    page, keep, kv = case["page"], case["keep"], case["kv"]
    kept, ctx = torch.full_like(s["kept"], -1), s["ctx_out"].clone()
    head = torch.arange(kv, device=ctx.device)[:, None]
    for i, (c, n) in enumerate(lengths(case)):
        length = c + n
        if length <= case["limit"]:
            kept[i, :, :length] = torch.arange(length, dtype=torch.int32, device=ctx.device)
            ctx[i] = length
            continue
        score = s["mass"][i, :, :length].clone()
        score[:, :case["first"]] = math.inf
        score[:, length - case["recent"]:] = math.inf
        slot = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :keep].sort(-1).values  # [kv, keep]
        kept[i, :, :keep] = slot
        ctx[i] = keep
        mass = s["mass"][i].gather(1, slot)
        s["mass"][i, :, :length] = 0.0
        s["mass"][i, :, :keep] = mass
        to = torch.arange(keep, device=ctx.device)[None]
        table = s["table"][i].long()
        for name in ("k4", "v4", "k_block", "v_block"):
            s[name][table[to // page], head, to % page] = s[name][table[slot // page], head, slot % page]
    return {"kept": kept, "ctx": ctx, "mass": s["mass"], "k": s["k4"], "v": s["v4"], "k_block": s["k_block"], "v_block": s["v_block"]}


def _places(row_start, ctx, rows):
    """Sequence, index within its sequence and slot of each of `rows` rows."""
    r = torch.arange(rows, device=ctx.device)
    seq = (r[:, None] >= row_start[None, 1:]).sum(1)
    j = r - row_start.long()[seq]
    return seq, j, ctx.long()[seq] + j


def _turned(x, pos, freq, layout, magnitude):
    """Rows of heads, turned by their positions, in 64 bits: angles of far positions need them, and so do values next to a border."""
    angle, n = pos[:, None].double() * freq[None], 2 * freq.shape[0]
    c, s = (torch.cos(angle) * magnitude)[:, None], (torch.sin(angle) * magnitude)[:, None]
    y = x.double()
    a, b = (y[..., :n // 2], y[..., n // 2:n]) if layout == "half" else (y[..., 0:n:2], y[..., 1:n:2])
    a, b = a * c - b * s, a * s + b * c
    return torch.cat(((torch.cat((a, b), -1) if layout == "half" else torch.stack((a, b), -1).flatten(-2)), y[..., n:]), -1)


def _e4m3(x):
    """64-bit numbers of 0 or more, rounded to 3 bits behind the leading one (2^-9 at the least, 448 at most), to the nearest even."""
    step = torch.exp2((torch.frexp(x).exponent - 1).clamp(min=-6).double() - 3.0)
    return ((x / step).round() * step).clamp(max=448.0)


def _quantised(x, scale):
    """Integers [..., dim] and the scales' bytes [..., dim / 16]; `scale`: the heads' scales, [..., heads] of x's leading dims."""
    x = x.double().unflatten(-1, (-1, BLOCK))
    scale = scale.double()[..., None]
    block = _e4m3(x.abs().amax(-1) / (7.0 * scale))
    ints = torch.nan_to_num(x / (block * scale)[..., None]).round().clamp(-7, 7)
    return ints.to(torch.int8).flatten(-2), block.float().to(torch.float8_e4m3fn).view(torch.uint8)


def _packed(ints):
    u = (ints + 8).to(torch.uint8)
    return u[..., 0::2] | (u[..., 1::2] << 4)


def _values(packed, blocks, scale):
    """Cached rows in 32 bits."""
    ints = torch.stack((packed & 15, packed >> 4), -1).flatten(-2).float() - 8.0
    return (ints.unflatten(-1, (-1, BLOCK)) * blocks.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2) * scale[..., None]


def _cached(s, i, name):
    """Keys or values of sequence i, [length, kv, dim]."""
    c, n = lengths(s["case"])[i]
    slot = torch.arange(c + n, device=s["ctx"].device)
    at, token = s["table"][i].long()[slot // s["case"]["page"]], slot % s["case"]["page"]
    return _values(s[name + "4"][at, :, token], s[name + "_block"][at, :, token], s[name + "_scale"][None])


def _sequences(s, each, heads):
    """each(i, scores [kv, group, rows, keys] of sequence i, masked); its results [kv, group, rows] as [all rows, heads], if there are any."""
    case, r0, results = s["case"], 0, []
    kv, window = case["kv"], case["window"]
    group = case["heads"] // kv
    s["bounds"] = []
    for i, (c, n) in enumerate(lengths(case)):
        s["bounds"].append((r0, n))
        q = s["q"][r0:r0 + n].float().reshape(n, kv, group, -1).permute(1, 2, 0, 3).reshape(kv, group * n, -1)
        score = torch.matmul(q, _cached(s, i, "k").permute(1, 2, 0)).mul_(1.0 / math.sqrt(case["dim"])).reshape(kv, group, n, c + n)
        key, place = torch.arange(c + n, device=q.device), c + torch.arange(n, device=q.device)[:, None]
        hidden = key > place
        if window:
            hidden |= key <= place - window
        score.masked_fill_(hidden, -math.inf)
        results.append(each(i, score))
        r0 += n
    if heads is None:
        return None
    return torch.cat([r.permute(2, 0, 1).reshape(-1, heads) for r in results])


# ------------------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """From the definitions, a row, a head or a sequence at a time."""
    s = prepare(case, seed)
    return {"rope": _exact_rope, "append": _exact_append, "attention": _exact_attention, "weights": _exact_weights, "evict": _exact_evict}[case["kind"]](s, case)


def _exact_turn(x, pos, freq, layout, magnitude):
    """As complex numbers."""
    n = 2 * freq.shape[0]
    turn = torch.polar(torch.full((len(pos), len(freq)), magnitude, dtype=torch.float64, device=x.device), pos.double()[:, None] * freq)[:, None]
    y = x.to(torch.float64).clone()
    first, second = (slice(0, n // 2), slice(n // 2, n)) if layout == "half" else (slice(0, n, 2), slice(1, n, 2))
    z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
    y[..., first], y[..., second] = z.real, z.imag
    return y


def _exact_rope(s, case):
    freq = s["freq"] * (-1 if case["inverse"] else 1)
    return {n: _exact_turn(s[n], s["positions"], freq, case["layout"], s["magnitude"]) for n in ("q", "k")}


def _exact_rounded(x, scale):
    """The values that rows x [n, dim] are held as, for one head's scale: the nearest of all e4m3 numbers, then of the 15 integers."""
    codes = torch.arange(127, device=x.device)
    grid = torch.where(codes < 8, codes * 2.0 ** -9, (1.0 + codes % 8 / 8.0) * torch.exp2((codes // 8).double() - 7.0)).double()
    x = x.reshape(x.shape[0], -1, BLOCK)
    want = x.abs().amax(-1) / (7.0 * scale)
    up = torch.searchsorted(grid, want.contiguous()).clamp(1, 126)
    low, high = grid[up - 1], grid[up]
    near = torch.where((want - low < high - want) | ((want - low == high - want) & ((up - 1) % 2 == 0)), low, high)
    step = (near * scale)[..., None]
    held = torch.where(step > 0, (x / step).round().clamp(-7, 7) * step, torch.zeros_like(x))
    return held.reshape(x.shape[0], -1)


def _exact_append(s, case):
    out = {"q": [], "k": [], "v": []}
    r = 0
    for i, (_, n) in enumerate(lengths(case)):
        pos = s["positions"][i] + torch.arange(n, device=s["ctx"].device)
        out["q"].append(_exact_turn(s["q"][r:r + n], pos, s["freq"], case["layout"], 1.0))
        for name, x in (("k", _exact_turn(s["k"][r:r + n], pos, s["freq"], case["layout"], 1.0)), ("v", s["v"][r:r + n].double())):
            out[name].append(torch.stack([_exact_rounded(x[:, h], float(s[name + "_scale"][h])) for h in range(case["kv"])], 1))
        r += n
    return {name: torch.cat(parts) for name, parts in out.items()}


def _exact_sequence(s, case, i, h, name):
    """Keys or values of sequence i and kv head h."""
    c, n = lengths(case)[i]
    used = s["table"][i, :-(-(c + n) // case["page"])].long()
    p = s[name + "4"][used, h].reshape(-1, case["dim"] // 2)[:c + n]
    ints = torch.zeros(c + n, case["dim"], dtype=torch.float64, device=p.device)
    ints[:, 0::2], ints[:, 1::2] = (p % 16).double() - 8, (p // 16).double() - 8
    block = s[name + "_block"][used, h].reshape(-1, case["dim"] // BLOCK)[:c + n].view(torch.float8_e4m3fn).double()
    return ints * block.repeat_interleave(BLOCK, -1) * float(s[name + "_scale"][h])


def _exact_scores(s, case, i, h, r):
    c, n = lengths(case)[i]
    group, window = case["heads"] // case["kv"], case["window"]
    at = torch.arange(c + n, device=s["q"].device)
    sees = at[None] <= c + torch.arange(n, device=at.device)[:, None]
    if window:
        sees &= at[None] > c + torch.arange(n, device=at.device)[:, None] - window
    q = s["q"][r:r + n, h * group:(h + 1) * group].double()
    score = torch.einsum("ngd,kd->gnk", q, _exact_sequence(s, case, i, h, "k")) / math.sqrt(case["dim"])
    return score.masked_fill(~sees[None], -math.inf)


def _exact_attention(s, case):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=s["q"].device)
    r, group = 0, case["heads"] // case["kv"]
    for i, (_, n) in enumerate(lengths(case)):
        for h in range(case["kv"]):
            score, mine = _exact_scores(s, case, i, h, r), slice(h * group, (h + 1) * group)
            lse[r:r + n, mine] = torch.logsumexp(score, -1).T
            out[r:r + n, mine] = torch.einsum("gnk,kd->ngd", torch.softmax(score, -1), _exact_sequence(s, case, i, h, "v"))
        r += n
    return {"out": out, "lse": lse}


def _exact_weights(s, case):
    mass = s["mass"].double()
    r, group = 0, case["heads"] // case["kv"]
    for i, (c, n) in enumerate(lengths(case)):
        for h in range(case["kv"]):
            lse = s["lse"][r:r + n, h * group:(h + 1) * group].double().T
            mass[i, h, :c + n] += torch.exp(_exact_scores(s, case, i, h, r) - lse[..., None]).sum((0, 1))
        r += n
    return mass


def _exact_evict(s, case):
    """The sums of what stays; places and moved bytes are whole numbers."""
    mass = s["mass"].double()
    for i, (c, n) in enumerate(lengths(case)):
        length = c + n
        if length <= case["limit"]:
            continue
        between = mass[i, :, case["first"]:length - case["recent"]]
        most = case["keep"] - case["first"] - case["recent"]
        for h in range(case["kv"]):
            # the lowest sum that stays, all above it, and of its equals the first ones
            x = between[h]
            least = x.kthvalue(len(x) - most + 1).values if most else torch.tensor(math.inf, device=x.device, dtype=x.dtype)
            stays = x > least
            equal = torch.nonzero(x == least)[:, 0]
            stays[equal[:most - int(stays.sum())]] = True
            row = torch.cat((mass[i, h, :case["first"]], x[stays], mass[i, h, length - case["recent"]:length]))
            mass[i, h, :length] = 0.0
            mass[i, h, :case["keep"]] = row
    return {"kept": None, "ctx": None, "mass": mass, "k": None, "v": None, "k_block": None, "v_block": None}
