"""The operators of a serving step over a key/value cache held in 8 bits, as cases of known size, in their plain form and in 64 bits.

A case is one pass of one kind:

  append     new rows of many sequences go into their pages (positions turned into rotations on the way, queries rotated with them), and the
             pages that they touched are read back as values;
  attention  the new rows of many sequences attend to what the cache holds of their sequence up to their own position;
  logprobs   log probabilities of given tokens under rows of logits, the rows' entropies and their best alternatives.

The cache: pages of int8, [page][kv head][token][dim], a 32-bit scale for each page and kv head; a value is the integer times its page's
scale. Row r of sequence i stands at position ctx[i] + r - row_start[i]; the page table says where a sequence's pages lie.

Lengths follow from the case alone; the values, the order of the pages and the tokens asked for come from the seed."""
import math
import random

import torch

own = False

THETA = 10000.0
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------- cases

def listed():
    def append(name, type, heads, kv, dim, page, seqs, new_lo, new_hi, ctx_lo, ctx_hi):
        return {"name": name, "kind": "append", "type": type, "heads": heads, "kv": kv, "dim": dim, "page": page, "seqs": seqs,
                "new_lo": new_lo, "new_hi": new_hi, "ctx_lo": ctx_lo, "ctx_hi": ctx_hi}

    def attention(name, type, heads, kv, dim, page, seqs, new_lo, new_hi, ctx_lo, ctx_hi, window=0):
        return dict(append(name, type, heads, kv, dim, page, seqs, new_lo, new_hi, ctx_lo, ctx_hi), kind="attention", window=window)

    def logprobs(name, type, rows, vocab, top):
        return {"name": name, "kind": "logprobs", "type": type, "rows": rows, "vocab": vocab, "top": top}

    return [
        # one user's next token on the TinyLlama shape: latency
        append("append-one", "f32", 32, 4, 64, 16, 1, 1, 1, 700, 700),
        # continuous batching on the 7B shape: 64 users' next tokens
        append("append-batch", "f32", 32, 32, 128, 16, 64, 1, 1, 128, 4096),
        # prompts of unequal length arriving together, some behind a cached prefix that ends inside a page
        append("append-prompts", "bf16", 32, 8, 128, 32, 5, 300, 2100, 0, 1300),
        # one user's next token on the TinyLlama shape: latency
        attention("attend-one", "f32", 32, 4, 64, 16, 1, 1, 1, 700, 700),
        # the headline decode step: the 7B shape behind 2048 tokens
        attention("attend-7b", "f32", 32, 32, 128, 16, 1, 1, 1, 2047, 2047),
        # continuous batching, grouped heads: 64 users with 128 to 4096 tokens each
        attention("attend-batch", "bf16", 32, 8, 128, 16, 64, 1, 1, 128, 4096),
        # drafts of four tokens checked behind two very long documents, grouped heads of the 70B shape
        attention("attend-long", "bf16", 64, 8, 128, 64, 2, 4, 4, 60001, 131000),
        # the 2048-token prompt of the 7B shape
        attention("attend-prompt", "f32", 32, 32, 128, 16, 1, 2048, 2048, 0, 0),
        # long prompts in chunks behind what earlier chunks have left
        attention("attend-chunks", "bf16", 32, 8, 128, 32, 3, 700, 2048, 1000, 6100),
        # one user's last row: latency
        logprobs("logprobs-one", "f32", 1, 32000, 5),
        # a batch of 64 users who all want alternatives
        logprobs("logprobs-batch", "f32", 64, 32000, 20),
        # a scored prompt over a large vocabulary
        logprobs("logprobs-prompt", "bf16", 2048, 128256, 4),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(("append", "attention", "attention", "logprobs"))
    type = rng.choice(sorted(DTYPES))
    if kind == "logprobs":
        vocab = spread(500, 131072)
        return {"kind": kind, "type": type, "rows": spread(1, max(2, min(2048, 2 ** 26 // vocab))), "vocab": vocab, "top": rng.choice((0, 1, 5, 20, rng.randint(1, 32)))}
    heads, kv, dim = rng.choice(((32, 4, 64), (32, 32, 128), (32, 8, 128), (64, 8, 128), (8, 1, 128), (12, 4, 96)))
    case = {"kind": kind, "type": type, "heads": heads, "kv": kv, "dim": dim, "page": rng.choice((16, 16, 32, 64, 128))}
    if kind == "append":
        seqs = spread(1, 64)
        new = 1 if rng.random() < 0.4 else spread(2, max(2, 4096 // seqs))
        ctx = spread(1, 8192)
    elif rng.random() < 0.6:  # single tokens and drafts
        seqs = spread(1, 64)
        new = rng.choice((1, 1, 1, 2, 5))
        ctx = spread(16, min(65536, 2 ** 28 // (kv * dim * seqs)))
    else:
        seqs = spread(1, 6)
        new = spread(16, 2048 // seqs)
        ctx = spread(1, 4096)
    case.update(seqs=seqs, new_lo=max(1, int(new * rng.uniform(0.3, 1.0))), new_hi=new, ctx_lo=int(ctx * rng.uniform(0.0, 1.0)), ctx_hi=ctx)
    if kind == "attention":
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
    if case["kind"] == "logprobs":
        cells = case["rows"] * case["vocab"]
        return {"bytes": cells * size + case["rows"] * (8 + 8 + 12 * case["top"]), "flops": 4 * cells}
    seqs, row, kv_row = lengths(case), case["heads"] * case["dim"], case["kv"] * case["dim"]
    rows = sum(n for _, n in seqs)
    if case["kind"] == "append":
        # the rows in, the queries out; the rows as integers, the older rows of their pages looked at; and all of these pages' rows back
        old = sum(c % case["page"] for c, _ in seqs)
        return {"bytes": rows * (2 * kv_row * size + 2 * row * size) + 2 * kv_row * (rows + old) + (rows + old) * 2 * kv_row * (1 + size), "flops": rows * 3 * (row + kv_row)}
    w = case["window"]
    pairs = sum(sum(min(c + j + 1, w) if w else c + j + 1 for j in range(n)) for c, n in seqs)
    keys = sum(min(c + n, w + n - 1) if w else c + n for c, n in seqs)
    return {"bytes": keys * 2 * kv_row + 2 * rows * row * size, "flops": 4 * row * pairs}


# --------------------------------------------------------------------------------------------------------------- inputs

def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    if case["kind"] == "logprobs":
        return _prepare_logprobs(case, dev, g, normal)
    heads, kv, dim, page, dtype = case["heads"], case["kv"], case["dim"], case["page"], DTYPES[case["type"]]
    seqs = lengths(case)
    ctx = torch.tensor([c for c, _ in seqs], dtype=torch.int32, device=dev)
    new = [n for _, n in seqs]
    row_start = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
    rows = sum(new)
    width = max(-(-(c + n) // page) for c, n in seqs)
    # every sequence has pages for its whole context, in no order, and the pool has some more
    need = [-(-(c + n) // page) for c, n in seqs]
    pages = sum(need) + 7
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    table = torch.full((len(seqs), width), -1, dtype=torch.int32, device=dev)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    spread = torch.exp(0.7 * normal(1, kv, 1, dim))  # some channels of the keys are larger than others
    s = {"case": case, "ctx": ctx, "row_start": row_start, "table": table, "max_new": max(new),
         "q": normal(rows, heads, dim).to(dtype)}
    k8, v8 = _integers(normal, pages, kv, page, dim, spread), _integers(normal, pages, kv, page, dim, 1.0)
    s["k8"], s["k_scale"] = k8[0], k8[1] * torch.exp(0.1 * normal(pages, kv))
    s["v8"], s["v_scale"] = v8[0], v8[1] * torch.exp(0.1 * normal(pages, kv))
    if case["kind"] == "append":
        s["k"], s["v"] = (normal(rows, kv, dim) * spread[:, :, 0]).to(dtype), normal(rows, kv, dim).to(dtype)
        s["freq"] = torch.tensor([THETA ** (-2.0 * d / dim) for d in range(dim // 2)], dtype=torch.float64, device=dev)
        # the pages that get rows, from their first row on
        first = [c // page * page for c, _ in seqs]
        back = [c + n - f for (c, n), f in zip(seqs, first)]
        s["first"] = torch.tensor(first, dtype=torch.int32, device=dev)
        s["back_start"] = torch.tensor([0] + back, device=dev).cumsum(0).to(torch.int32)
        s["max_back"] = max(back)
        s["q_out"] = torch.empty_like(s["q"])
        s["k_out"] = torch.empty(sum(back), kv, dim, dtype=dtype, device=dev)
        s["v_out"] = torch.empty_like(s["k_out"])
    else:
        s["out"] = torch.empty_like(s["q"])
    if own:
        import leafcutterllm_b200 as lc
        s["cache"] = lc.Kv8Cache(s["k8"], s["v8"], s["k_scale"], s["v_scale"])
        s["rows"] = lc.Kv8Rows(s["table"], s["ctx"], s["row_start"], s["max_new"])
        if case["kind"] == "append":
            s["turns"] = torch.from_numpy(lc.rope_turns(THETA, dim).view("int64")).to(dev)
            s["back"] = lc.Kv8Rows(s["table"], s["first"], s["back_start"], s["max_back"])
        else:
            s["workspace"] = torch.empty(s["cache"].attention_workspace(s["rows"], s["q"]), dtype=torch.uint8, device=dev)
    return s


def _integers(normal, pages, kv, page, dim, spread):
    """Pages as an earlier append has left them: the largest value of a page and head is 127 times its scale."""
    x = normal(pages, kv, page, dim) * spread
    top = x.abs().amax(dim=(2, 3), keepdim=True)
    return (x * (127.0 / top)).round_().to(torch.int8), top.reshape(pages, kv) / 127.0


def _prepare_logprobs(case, dev, g, normal):
    rows, vocab, top = case["rows"], case["vocab"], case["top"]
    # a model's logits: wide noise, and a few tokens of each row that stand out
    x = torch.empty(rows, vocab, dtype=DTYPES[case["type"]], device=dev)
    x.copy_(normal(rows, vocab).mul_(2.0))
    best = torch.randint(vocab, (rows, 6), generator=g, device=dev)
    x.scatter_(1, best, (8.0 + 3.0 * normal(rows, 6)).to(x.dtype))
    # mostly one of the likely tokens is asked for, now and then any
    any_token = torch.randint(vocab, (rows,), generator=g, device=dev)
    tokens = torch.where(torch.rand(rows, generator=g, device=dev) < 0.8, best[:, 0], any_token)
    s = {"case": case, "logits": x, "tokens": tokens,
         "logprob": torch.empty(rows, device=dev), "entropy": torch.empty(rows, device=dev),
         "top_logprob": torch.empty(rows, top, device=dev), "top_id": torch.empty(rows, top, dtype=torch.int64, device=dev)}
    return s


# --------------------------------------------------------------------------------------------------------------- passes

def run(s):
    kind = s["case"]["kind"]
    if kind == "append":
        if own:
            s["cache"].append(s["rows"], s["k"], s["v"], turns=s["turns"], q=s["q"], q_out=s["q_out"])
            s["cache"].read(s["back"], s["k_out"], s["v_out"])
            q, k, v = s["q_out"], s["k_out"], s["v_out"]
        else:
            q = _append(s)
            k, v = _read(s)
        return {"q": q, "k": k, "v": v, "k_scale": s["k_scale"], "v_scale": s["v_scale"]}
    if kind == "attention":
        if own:
            return s["cache"].attention(s["rows"], s["q"], s["out"], window=s["case"]["window"], workspace=s["workspace"])
        return _attention(s)
    if own:
        import leafcutterllm_b200 as lc
        out = lc.token_logprobs_dev(s["logits"], s["tokens"], s["logprob"], s["entropy"], s["top_logprob"], s["top_id"])
    else:
        out = _logprobs(s)
    return dict(zip(("logprob", "entropy", "top_logprob", "top_id"), out))


def _places(row_start, ctx, rows):
    """Sequence, index within its sequence and position of each of `rows` rows."""
    r = torch.arange(rows, device=ctx.device)
    seq = (r[:, None] >= row_start[None, 1:]).sum(1)
    j = r - row_start.long()[seq]
    return seq, j, ctx.long()[seq] + j


def _turned(x, pos, freq):
    """Rows of heads, turned by their positions, in 64 bits: angles of far positions need them, and so do values next to a border."""
    angle = pos[:, None].double() * freq[None]
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat((a * c - b * s, a * s + b * c), dim=-1)


def _append(s):
    page = s["case"]["page"]
    seq, j, pos = _places(s["row_start"], s["ctx"], s["k"].shape[0])
    at, slot = s["table"].long()[seq, pos // page], pos % page
    # the older rows of a sequence's first page
    ctx, n = s["ctx"].long(), s["row_start"].long().diff()
    old_page = s["table"].long().gather(1, (ctx // page)[:, None].clamp(max=s["table"].shape[1] - 1))[:, 0]
    has_old = (ctx % page > 0) & (n > 0)
    old_page, old_slots = old_page[has_old], (ctx % page)[has_old]
    for pool, scale, x in ((s["k8"], s["k_scale"], _turned(s["k"], pos, s["freq"])), (s["v8"], s["v_scale"], s["v"].double())):
        finite = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
        top = torch.zeros(scale.shape, dtype=torch.float64, device=x.device)
        top.scatter_reduce_(0, at[:, None].expand(-1, top.shape[1]), finite.abs().amax(-1), "amax")
        before = torch.zeros_like(scale)
        before[old_page] = scale[old_page]
        after = torch.maximum(before, (top / 127.0).float())
        ints = pool[old_page].double()
        ratio = before[old_page].double()[:, :, None, None] * ints / after[old_page].double()[:, :, None, None]
        is_old = torch.arange(page, device=x.device)[None, None, :, None] < old_slots[:, None, None, None]
        pool[old_page] = torch.where(is_old, torch.nan_to_num(ratio, 0.0).round(), ints).to(torch.int8)
        y = x / after[at].double()[:, :, None]
        y = torch.where((after[at] > 0)[:, :, None], y, torch.zeros_like(y))
        pool[at, :, slot] = torch.nan_to_num(y, nan=0.0).round().clamp(-127, 127).to(torch.int8)
        scale[at] = after[at]
    return _turned(s["q"], pos, s["freq"]).to(s["q"].dtype)


def _read(s):
    page = s["case"]["page"]
    seq, _, pos = _places(s["back_start"], s["first"], s["k_out"].shape[0])
    at, slot = s["table"].long()[seq, pos // page], pos % page
    return tuple((pool[at, :, slot].float() * scale[at][:, :, None]).to(s["k_out"].dtype)
                 for pool, scale in ((s["k8"], s["k_scale"]), (s["v8"], s["v_scale"])))


def _attention(s):
    case = s["case"]
    page, kv, dim, window = case["page"], case["kv"], case["dim"], case["window"]
    rows, heads = s["q"].shape[0], s["q"].shape[1]
    seq, j, pos = _places(s["row_start"], s["ctx"], rows)
    n, most, group = s["ctx"].shape[0], s["max_new"], heads // kv
    length = s["ctx"].long() + s["row_start"].long().diff()
    keys = torch.arange(s["table"].shape[1] * page, device=pos.device)
    at = s["table"].long()[:, keys // page].clamp(min=0)                       # [n, keys]
    value = lambda pool, scale: pool[at, :, keys % page].float() * scale[at][..., None]  # noqa: E731  [n, keys, kv, dim]
    held = keys[None] < length[:, None]
    q = torch.zeros(n, most, heads, dim, device=pos.device)
    q[seq, j] = s["q"].float()
    q = q.reshape(n, most, kv, group, dim).permute(0, 2, 3, 1, 4).reshape(n, kv, group * most, dim)
    k = value(s["k8"], s["k_scale"]).permute(0, 2, 3, 1)
    score = torch.matmul(q, k).reshape(n, kv, group, most, -1) * (1.0 / math.sqrt(dim))
    del k
    place = s["ctx"].long()[:, None] + torch.arange(most, device=pos.device)   # [n, most]
    sees = held[:, None, :] & (keys[None, None] <= place[:, :, None])
    if window:
        sees &= keys[None, None] > place[:, :, None] - window
    score.masked_fill_(~sees[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_(min=-3.0e38)
    p = score.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    v = value(s["v8"], s["v_scale"]).masked_fill_(~held[:, :, None, None], 0.0).permute(0, 2, 1, 3)
    out = torch.matmul(p.reshape(n, kv, group * most, -1), v).reshape(n, kv, group, most, dim)
    out = torch.where(total > 0, out / total, torch.zeros_like(out))
    return out.permute(0, 3, 1, 2, 4).reshape(n, most, heads, dim)[seq, j].to(s["q"].dtype)


def _logprobs(s):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    d = x - top
    p = d.exp()
    total = p.sum(-1, dtype=torch.float64)
    entropy = total.log() - torch.where(p > 0, p * d, torch.zeros_like(p)).sum(-1, dtype=torch.float64) / total
    del p
    lse = total.log()[:, None]
    logprob = (d.gather(1, s["tokens"][:, None]).double() - lse)[:, 0].float()
    if s["case"]["top"] == 0:
        return logprob, entropy.float(), s["top_logprob"], s["top_id"]
    # values as whole numbers of the same order, then the lower index first
    bits = (x + 0.0).view(torch.int32).long()
    key = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))
    key = key * (1 << 31) + ((1 << 31) - 1 - torch.arange(x.shape[1], device=x.device))
    best = (1 << 31) - 1 - (key.topk(s["case"]["top"], dim=-1).values & ((1 << 31) - 1))
    return logprob, entropy.float(), (d.gather(1, best).double() - lse).float(), best


# ------------------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """From the definitions, a sequence (or a stretch of rows) at a time."""
    s = prepare(case, seed)
    if case["kind"] == "logprobs":
        return _exact_logprobs(s, case)
    if case["kind"] == "attention":
        return _exact_attention(s, case)
    return _exact_append(s, case)


def _exact_append(s, case):
    page, kv, dim, dev = case["page"], case["kv"], case["dim"], s["ctx"].device
    f = torch.tensor([math.exp(-2.0 * d / dim * math.log(THETA)) for d in range(dim // 2)], dtype=torch.float64, device=dev)
    scales = {"k": s["k_scale"].double(), "v": s["v_scale"].double()}
    out = {"q": [], "k": [], "v": []}
    r = 0
    for i, (c, n) in enumerate(lengths(case)):
        angle = torch.arange(c, c + n, dtype=torch.float64, device=dev)[:, None] * f[None]
        turn = torch.polar(torch.ones_like(angle), angle)[:, None]
        def rotated(x):
            x = x.to(torch.float64)
            z = torch.complex(x[..., :dim // 2], x[..., dim // 2:]) * turn
            return torch.cat((z.real, z.imag), -1)
        out["q"].append(rotated(s["q"][r:r + n]))
        new = {"k": rotated(s["k"][r:r + n]), "v": s["v"][r:r + n].double()}
        for name in ("k", "v"):
            pos = c
            while pos < c + n:  # page after page
                number = int(s["table"][i, pos // page])
                first, end = pos % page, min(page, pos % page + c + n - pos)
                x = new[name][pos - c:pos - c + end - first].permute(1, 0, 2)                  # [kv, rows, dim]
                scale = (x.abs().amax((1, 2)) / 127).float().double()                          # the scale is held in 32 bits
                ints = s[name + "8"][number, :, :first].double()
                if first:
                    before = scales[name][number]
                    scale = torch.maximum(scale, before)
                    ints = torch.round(ints * before[:, None, None] / scale[:, None, None])
                ints = torch.cat((ints, torch.round(x / scale[:, None, None])), 1)
                scales[name][number] = scale
                out[name].append((ints * scale[:, None, None]).permute(1, 0, 2))
                pos += end - first
        r += n
    return {**{k: torch.cat(v) for k, v in out.items()}, "k_scale": scales["k"], "v_scale": scales["v"]}


def _exact_attention(s, case):
    page, kv, group, window = case["page"], case["kv"], case["heads"] // case["kv"], case["window"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    r = 0
    for i, (c, n) in enumerate(lengths(case)):
        used = s["table"][i, :-(-(c + n) // page)].long()
        at = torch.arange(c + n, device=out.device)
        hidden = at[None] > c + torch.arange(n, device=out.device)[:, None]
        if window:
            hidden |= at[None] <= c + torch.arange(n, device=out.device)[:, None] - window
        for h in range(kv):
            k = (s["k8"][used, h].double() * s["k_scale"][used, h].double()[:, None, None]).reshape(-1, case["dim"])[:c + n]
            v = (s["v8"][used, h].double() * s["v_scale"][used, h].double()[:, None, None]).reshape(-1, case["dim"])[:c + n]
            q = s["q"][r:r + n, h * group:(h + 1) * group].double()
            score = torch.einsum("ngd,kd->gnk", q, k) / math.sqrt(case["dim"])
            weight = torch.softmax(score.masked_fill(hidden[None], -math.inf), -1)
            out[r:r + n, h * group:(h + 1) * group] = torch.einsum("gnk,kd->ngd", weight, v)
        r += n
    return out


def _exact_logprobs(s, case):
    x, parts = s["logits"], {"logprob": [], "entropy": [], "top_logprob": [], "top_id": None}
    step = max(1, 2 ** 26 // case["vocab"])
    for a in range(0, case["rows"], step):
        y = x[a:a + step].double()
        y = y - torch.logsumexp(y, -1, keepdim=True)
        parts["logprob"].append(y.gather(1, s["tokens"][a:a + step, None])[:, 0])
        parts["entropy"].append(-(y.exp() * y).sum(-1))
        parts["top_logprob"].append(torch.sort(y, dim=-1, descending=True).values[:, :case["top"]])
    return {k: torch.cat(v) if v else None for k, v in parts.items()}
