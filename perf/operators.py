"""Workloads of three operators of a decode step over many requests: attention of rows that share a prompt prefix, low-rank
adapters beside a shared projection, and controls on logits (penalties, biases, grammar masks) with greedy selection.

Shapes of heads and projections are those of the model presets; the other sizes are generic. With ``own`` false a pass is
computed in elementary torch operations, in 32 bits and rounded once; with ``own`` true it is the framework's call.
"""

import math

import torch

own = False

# query heads, key heads, head width (hidden width) of the model presets
HEADS = {"small": (16, 8, 128), "large": (32, 8, 128), "larger": (64, 8, 128), "narrow": (14, 2, 64)}
VOCAB = 151936


# --------------------------------------------------------------------------------------------------- cases


def _attention(name, heads, page, groups, alone, shortest, longest):
    """``groups``: "rows x prefix tokens, ..." of the runs of rows that share a prefix; ``alone``: rows behind them that share
    none; every row has ``shortest`` to ``longest`` tokens of its own behind its prefix."""
    return {"name": name, "kind": "attention", "heads": heads, "page": page, "groups": groups, "alone": alone,
            "shortest": shortest, "longest": longest}


def _adapters(name, rows, inner, outer, adapters, ranks, bare, run):
    """``outer``: features of the parts of the projection ("2048+1024+1024"); ``ranks``: the adapters' ranks in turn;
    ``bare``: one row in so many runs has no adapter (0: none); ``run``: consecutive rows with one adapter."""
    return {"name": name, "kind": "adapters", "rows": rows, "inner": inner, "outer": outer, "adapters": adapters,
            "ranks": ranks, "bare": bare, "run": run}


def _logits(name, what, dtype, rows, vocab, history, biases, masks):
    """``what``: "select" (one greedy token a row, and its adjusted logit) or "adjust" (the adjusted logits). ``history``: longest prompt and answer;
    ``biases``: entries a row; ``masks``: one row in so many is held to a grammar (0: none)."""
    return {"name": name, "kind": "logits", "what": what, "dtype": dtype, "rows": rows, "vocab": vocab, "history": history,
            "biases": biases, "masks": masks}


def listed():
    return [
        # a few users of one assistant with a short system prompt, just started: launches and latency
        _attention("prefix_few", "small", 64, "4x512", 0, 1, 40),
        # a busy assistant with a long system prompt
        _attention("prefix_busy", "large", 64, "64x2048", 0, 20, 600),
        # questions about one long document: the shared part is nearly all the work
        _attention("prefix_document", "large", 64, "256x8192", 0, 30, 300),
        # several prompts at once, and requests that share none; seven query heads to a key head, small pages, ragged sizes
        _attention("prefix_groups", "narrow", 16, "23x1392,9x464,2x6000,40x752", 13, 1, 700),
        # four users with an adapter each, q, k and v projections of the small model
        _adapters("adapters_few", 4, 1024, "2048+1024+1024", 4, "16", 0, 1),
        # a decode step of many users with adapters of different ranks, some without
        _adapters("adapters_decode", 64, 4096, "4096+1024+1024", 40, "8,16,32,64", 7, 1),
        # a prefill chunk of some prompts
        _adapters("adapters_prefill", 1999, 4096, "4096", 5, "16,32", 3, 271),
        # one popular adapter of a high rank, output projection of a wide model
        _adapters("adapters_popular", 160, 8192, "5120", 2, "128,120", 0, 80),
        # three users with penalties, one of them answering in a grammar
        _logits("select_few", "select", "bfloat16", 3, VOCAB, 300, 5, 3),
        # a saturated step: penalties on everybody's history, biases, a third in grammars
        _logits("select_busy", "select", "bfloat16", 256, VOCAB, 1500, 60, 3),
        # adjusted 32-bit logits of another vocabulary, to be ranked or logged by the caller
        _logits("adjust_odd", "adjust", "float32", 33, 50021, 700, 300, 2),
        # ... of a saturated step
        _logits("adjust_busy", "adjust", "bfloat16", 128, VOCAB, 1000, 20, 4),
    ]


def _between(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Another case of the listed kinds, its sizes anywhere between the smallest and the largest listed ones."""
    most = {}
    for c in listed():
        most[c["kind"]] = max(most.get(c["kind"], 0), _cost(c))
    while True:
        kind = rng.choice(["attention", "adapters", "logits"])
        if kind == "attention":
            heads = rng.choice(list(HEADS))
            groups = ",".join(f"{_between(rng, 2, 256)}x{_between(rng, 16, 8192)}" for _ in range(rng.choice([1, 1, 2, 3, 5, 8])))
            lo = _between(rng, 1, 400)
            c = _attention(None, heads, rng.choice([16, 32, 64, 128]), groups, rng.choice([0, 0, _between(rng, 1, 40)]), lo, lo + _between(rng, 1, 700))
            if sum(n for n, _ in _groups(c)) + c["alone"] > 300:
                continue
        elif kind == "adapters":
            hidden = rng.choice([896, 1024, 2048, 4096, 5120])
            outer = rng.choice([f"{hidden}", f"{2 * hidden}+1024+1024", "4096+1024+1024", "896+128+128", "5120"])
            ranks = rng.choice(["16", "8,16,32,64", "32", "128,120", "4,64", "24"])
            long = rng.random() < 0.4
            rows = _between(rng, 200, 2048) if long else _between(rng, 1, 200)
            c = _adapters(None, rows, hidden, outer, _between(rng, 1, 8 if long else 64), ranks, rng.choice([0, 2, 3, 7]),
                          _between(rng, 60, 900) if long else rng.choice([1, 1, 2, 5]))
        else:
            c = _logits(None, rng.choice(["select", "adjust"]), rng.choice(["bfloat16", "bfloat16", "float32"]), _between(rng, 1, 256),
                        rng.choice([VOCAB, 4096, 50021, 32000, _between(rng, 1000, 200000)]), _between(rng, 1, 2000),
                        rng.choice([0, _between(rng, 1, 300)]), rng.choice([0, 1, 2, 5]))
        del c["name"]
        if _cost(c) <= most[kind]:
            return c


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 5e12, w["flops"] / 4e14)


# --------------------------------------------------------------------------------------------------- sizes of a case


def _spread(lo, hi, i):
    return lo + int((hi - lo + 1) * ((i * 0.6180339887498949 + 0.31) % 1.0))


def _groups(case):
    return [tuple(int(v) for v in g.split("x")) for g in case["groups"].split(",")]


def _rows(case):
    """(prefix, tokens of its own) of every row."""
    out = [p for n, p in _groups(case) for _ in range(n)] + [0] * case["alone"]
    return [(p, _spread(case["shortest"], case["longest"], i)) for i, p in enumerate(out)]


def _parts(case):
    return tuple(int(v) for v in case["outer"].split("+"))


def _rank(case, adapter):
    ranks = [int(v) for v in case["ranks"].split(",")]
    return ranks[adapter % len(ranks)]


def _index(case):
    """The adapter of every row (-1: none), in runs of consecutive rows."""
    out = []
    for i in range(case["rows"]):
        run = i // case["run"]
        out.append(-1 if case["bare"] and run % case["bare"] == case["bare"] - 1 else run * 7 % case["adapters"])
    return out


def _history(case):
    """(prompt, answer) tokens of every row."""
    most = case["history"]
    return [(_spread(0, most, i), _spread(0, most // 2, i + 5)) for i in range(case["rows"])]


def _masked(case):
    """Rows that are held to a grammar."""
    return [i for i in range(case["rows"]) if case["masks"] and i % case["masks"] == case["masks"] - 1]


def work(case):
    if case["kind"] == "attention":
        hq, hk, d = HEADS[case["heads"]]
        rows, page = _rows(case), case["page"]
        cached = sum(p // page * page for _, p in _groups(case)) + sum(p % page + s for p, s in rows)     # whole pages are shared
        return {"bytes": cached * hk * d * 4 + len(rows) * hq * d * 4, "flops": sum(p + s for p, s in rows) * 4 * hq * d}
    if case["kind"] == "adapters":
        parts, k, index = _parts(case), case["inner"], _index(case)
        used = sorted({a for a in index if a >= 0})
        weights = sum(_rank(case, a) * (len(parts) * k + sum(parts)) for a in used)
        flops = sum(2 * _rank(case, a) * (len(parts) * k + sum(parts)) for a in index if a >= 0)
        inner = k * sum(1 for a in index if a >= 0)
        return {"bytes": 2 * (weights + inner + 2 * case["rows"] * sum(parts)), "flops": flops}
    size = 4 if case["dtype"] == "float32" else 2
    each = case["rows"] * case["vocab"]
    read = each * size + sum(a + b for a, b in _history(case)) * 4 + case["rows"] * case["biases"] * 8 + len(_masked(case)) * case["vocab"] // 8
    return {"bytes": read + (each * size if case["what"] == "adjust" else 8 * case["rows"]), "flops": 2 * each}


# --------------------------------------------------------------------------------------------------- inputs


def _attention_inputs(case, seed):
    hq, hk, d = HEADS[case["heads"]]
    page, rows, groups = case["page"], _rows(case), _groups(case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    # whole pages are shared: what lies behind the last whole page of a prefix belongs to each row
    owner, at = [], 0
    for n, p in groups:
        owner += [at] * n
        at += n
    owner += list(range(at, len(rows)))
    total = sum(-(-(p + s) // page) for p, s in rows)
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32).cpu()
    table = torch.zeros(len(rows), max(-(-(p + s) // page) for p, s in rows), dtype=torch.int32)
    used = 0
    for r, (p, s) in enumerate(rows):
        shared = p // page if owner[r] != r else 0
        table[r, :shared] = table[owner[r], :shared]
        own_pages = -(-(p + s) // page) - shared
        table[r, shared:shared + own_pages] = order[used:used + own_pages]
        used += own_pages

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32).to(torch.bfloat16)

    k, v = torch.empty(used, page, hk, d, dtype=torch.bfloat16, device="cuda"), torch.empty(used, page, hk, d, dtype=torch.bfloat16, device="cuda")
    for t in (k, v):
        for i in range(0, used, 4096):
            t[i:i + 4096] = normal(min(4096, used - i), page, hk, d)
    # pages are numbered anew: the cache holds only those that some row reads
    new = torch.full((total,), -1, dtype=torch.int32)
    new[order[:used].long()] = torch.arange(used, dtype=torch.int32)[torch.randperm(used, generator=torch.Generator().manual_seed(seed))]
    width = [-(-(p + s) // page) for p, s in rows]
    for r, w in enumerate(width):
        table[r, :w] = new[table[r, :w].long()]
    lens = torch.tensor([p + s for p, s in rows], dtype=torch.int32)
    return {"q": 1.5 * normal(len(rows), hq, d), "k": k, "v": v, "table": table.cuda(), "lens": lens.cuda(),
            "groups": [(n, p // page * page) for n, p in groups], "longest": max(p + s for p, s in rows)}


def _adapter_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    parts, k, n = _parts(case), case["inner"], case["adapters"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)

    pairs = []
    for a in range(n):
        r = _rank(case, a)
        pairs.append([((normal(r, k) / math.sqrt(k)).to(torch.bfloat16), (normal(f, r) / math.sqrt(r)).to(torch.bfloat16)) for f in parts])
    return {"x": normal(case["rows"], k).to(torch.bfloat16), "y": normal(case["rows"], sum(parts)).to(torch.bfloat16), "pairs": pairs,
            "scales": [0.25 * (1 + a % 5) for a in range(n)], "index": _index(case)}


def _logit_inputs(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rows, vocab = case["rows"], case["vocab"]
    dtype = torch.float32 if case["dtype"] == "float32" else torch.bfloat16

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda", dtype=torch.float32)

    logits = torch.randn(rows, vocab, generator=g, device="cuda", dtype=torch.float32) * 2.5
    lens = _history(case)
    most = max(1, max(a + b for a, b in lens))
    # frequent tokens are frequent: the third power of a uniform number; what was said before is likely again
    history = (uniform(rows, most) ** 3 * vocab).long().clamp_(max=vocab - 1)
    logits.scatter_add_(1, history, torch.full((rows, most), 0.5, device="cuda"))
    ids = []
    if case["biases"]:
        ids = (uniform(rows, case["biases"]) * (vocab // case["biases"])).long() + torch.arange(case["biases"], device="cuda") * (vocab // case["biases"])
    masked = _masked(case)
    words = -(-vocab // 32)
    mask = torch.zeros(0, words, dtype=torch.int32, device="cuda")
    if masked:
        mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (len(masked), words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
    index = [-1] * rows
    for i, r in enumerate(masked):
        index[r] = i

    def each(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype, device="cuda")

    return {"logits": logits.to(dtype), "history": history.to(torch.int32), "prompt_lens": each([a for a, _ in lens]),
            "lens": each([a + b for a, b in lens]), "repetition": 1 + 0.3 * uniform(rows), "frequency": 0.4 * uniform(rows) - 0.1,
            "presence": 0.6 * uniform(rows) - 0.1,
            "bias_ids": ids.to(torch.int32).reshape(-1) if case["biases"] else each([]),
            "bias_values": 8 * uniform(rows * case["biases"]) - 4, "bias_starts": each([i * case["biases"] for i in range(rows + 1)]),
            "masks": mask, "mask_index": each(index)}


_INPUTS = {"attention": _attention_inputs, "adapters": _adapter_inputs, "logits": _logit_inputs}


def prepare(case, seed):
    s = {"case": case, **_INPUTS[case["kind"]](case, seed)}
    if case["kind"] == "adapters":
        index = s["index"]
        if own:
            from crosspool_b200.ops import lora

            s["stack"] = lora.AdapterStack(case["adapters"], case["inner"], _parts(case), max(_rank(case, a) for a in range(case["adapters"])))
            for a, pair in enumerate(s.pop("pairs")):
                s["stack"].load(a, [p[0] for p in pair], [p[1] for p in pair], s["scales"][a])
            s["plan"] = lora.adapter_plan(index, s["stack"])
        else:
            rows = {}
            for i, a in enumerate(index):
                rows.setdefault(a, []).append(i)
            s["rows"] = {a: torch.tensor(r, device="cuda") for a, r in rows.items() if a >= 0}
    elif own and case["kind"] == "attention":
        from crosspool_b200.ops import attention

        hq, hk, d = HEADS[case["heads"]]
        s["plan"] = attention.shared_prefix_plan([n for n, _ in s["groups"]], [p for _, p in s["groups"]], rows=s["q"].shape[0], q_heads=hq,
                                                 kv_heads=hk, head_dim=d, max_len=s["longest"])
    elif own:
        from crosspool_b200.ops import logits

        s["controls"] = logits.LogitControls(**{n: s[n] for n in (
            "history", "lens", "prompt_lens", "repetition", "frequency", "presence", "bias_ids", "bias_values", "bias_starts", "masks", "mask_index")})
    return s


# --------------------------------------------------------------------------------------------------- passes


def run(state):
    s, case = state, state["case"]
    if case["kind"] == "attention":
        if own:
            from crosspool_b200.ops import attention

            return attention.paged_decode_shared(s["q"], s["k"], s["v"], s["table"], s["lens"], s["plan"])
        return _plain_attention(s)
    if case["kind"] == "adapters":
        if own:
            from crosspool_b200.ops import lora

            return lora.lora_add(s["y"], s["x"], s["stack"], s["plan"])
        return _plain_adapters(s)
    if own:
        from crosspool_b200.ops import logits

        if case["what"] == "select":
            values = torch.empty(case["rows"], dtype=torch.float32, device="cuda")
            return logits.select_tokens(s["logits"], s["controls"], values=values), values
        return logits.adjust_logits(s["logits"], s["controls"])
    v = _plain_controls(s)
    if case["what"] == "select":
        tokens = v.argmax(dim=1)
        return tokens.to(torch.int32), v.gather(1, tokens[:, None])[:, 0]
    return v.to(s["logits"].dtype)


def _plain_attention(s):
    """softmax(q k^T / sqrt(d)) v of every row over its prefix (keys of the group's first row) and its own tokens."""
    q, page = s["q"], s["k"].shape[1]
    rows, hq, d = q.shape
    hk = s["k"].shape[2]
    k, v = s["k"].view(-1, hk, d), s["v"].view(-1, hk, d)
    qf = q.float().view(rows, hk, hq // hk, d) * d ** -0.5
    out = torch.empty(rows, hk, hq // hk, d, dtype=torch.float32, device=q.device)
    inside = torch.arange(page, device=q.device)
    spans, at = [], 0
    for n, p in s["groups"]:
        spans.append((at, n, p))
        at += n
    if at < rows:
        spans.append((at, rows - at, 0))
    for at, n, p in spans:
        lens = s["lens"][at:at + n]
        t = s["table"][at:at + n].long()
        tail = ((t[:, p // page:, None] * page) + inside).view(n, -1)           # the rows' own tokens, and some behind their ends
        ks, vs = k[tail].float(), v[tail].float()
        sc = torch.matmul(qf[at:at + n], ks.permute(0, 2, 3, 1))
        hidden = torch.arange(tail.shape[1], device=q.device)[None] >= (lens - p)[:, None]
        sc = sc.masked_fill(hidden[:, None, None], -math.inf)
        top = sc.amax(-1, keepdim=True)
        if p:
            head = ((t[0, :p // page, None] * page) + inside).view(-1)
            kp, vp = k[head].float().transpose(0, 1), v[head].float().transpose(0, 1)
            qg = qf[at:at + n].permute(1, 0, 2, 3).reshape(hk, -1, d)
            sp = torch.matmul(qg, kp.transpose(1, 2)).view(hk, n, hq // hk, p)
            top = torch.maximum(top, sp.amax(-1, keepdim=True).transpose(0, 1))
            ep = torch.exp(sp - top.transpose(0, 1))
            acc = torch.matmul(ep.reshape(hk, -1, p), vp).view(hk, n, hq // hk, d).transpose(0, 1)
            total = ep.sum(-1, keepdim=True).transpose(0, 1)
        else:
            acc, total = 0.0, 0.0
        e = torch.exp(sc - top)
        out[at:at + n] = (acc + torch.matmul(e, vs.permute(0, 2, 1, 3))) / (total + e.sum(-1, keepdim=True))
    return out.view(rows, hq, d).to(q.dtype)


def _plain_adapters(s):
    """y + scale (x A^T) B^T for the rows of every adapter, part by part of the features."""
    out, x = s["y"].float(), s["x"].float()
    for a, rows in s["rows"].items():
        at, xr = 0, x[rows]
        for low, high in s["pairs"][a]:
            out[rows, at:at + high.shape[0]] += s["scales"][a] * torch.matmul(torch.matmul(xr, low.float().t()), high.float().t())
            at += high.shape[0]
    return out.to(s["y"].dtype)


def _plain_controls(s):
    """Penalties on the tokens of the history, then biases, then the grammar's mask."""
    v = s["logits"].float()
    rows, vocab = v.shape
    place = torch.arange(s["history"].shape[1], device=v.device)[None]
    ids = s["history"].long()
    said = torch.zeros(rows, vocab, dtype=torch.int32, device=v.device)
    said.scatter_add_(1, ids, (place < s["lens"][:, None]).int())
    count = torch.zeros(rows, vocab, dtype=torch.int32, device=v.device)
    count.scatter_add_(1, ids, ((place >= s["prompt_lens"][:, None]) & (place < s["lens"][:, None])).int())
    r = s["repetition"][:, None]
    v = torch.where(said > 0, torch.where(v > 0, v / r, v * r), v)
    v = v - s["frequency"][:, None] * count
    v = torch.where(count > 0, v - s["presence"][:, None], v)
    if s["bias_ids"].numel():
        n = s["bias_ids"].numel() // rows
        bias = torch.zeros(rows, vocab, dtype=torch.float32, device=v.device)
        bias.scatter_(1, s["bias_ids"].view(rows, n).long(), s["bias_values"].view(rows, n))
        v = v + bias
    if s["masks"].shape[0]:
        bits = (s["masks"][:, :, None] >> torch.arange(32, device=v.device, dtype=torch.int32)) & 1
        allowed = bits.view(s["masks"].shape[0], -1)[:, :vocab].bool()[s["mask_index"].clamp(min=0).long()]
        v = v.masked_fill(~allowed & (s["mask_index"] >= 0)[:, None], -math.inf)
    return v


# --------------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = _INPUTS[case["kind"]](case, seed)
    if case["kind"] == "attention":
        return _exact_attention(s)
    if case["kind"] == "adapters":
        return _exact_adapters(case, s)
    v = _exact_controls(case, s)
    return (None, v.amax(dim=1)) if case["what"] == "select" else v


def _exact_attention(s):
    """Row after row over all of its tokens, in the order of its table."""
    page, hk, d = s["k"].shape[1:]
    out = []
    for q, table, n in zip(s["q"].double(), s["table"].long(), s["lens"].tolist()):
        used = table[:-(-n // page)]
        k, v = s["k"][used].reshape(-1, hk, d)[:n].double(), s["v"][used].reshape(-1, hk, d)[:n].double()
        w = torch.softmax(torch.einsum("hgd,thd->hgt", q.view(hk, -1, d), k) / math.sqrt(d), dim=-1)
        out.append(torch.einsum("hgt,thd->hgd", w, v).reshape(-1, d))
    return torch.stack(out)


def _exact_adapters(case, s):
    y, x = s["y"].double(), s["x"].double()
    index = torch.tensor(s["index"], device=y.device)
    for a, pair in enumerate(s["pairs"]):
        delta = torch.cat([(x @ low.double().t()) @ high.double().t() for low, high in pair], dim=1)
        y = torch.where((index == a)[:, None], y + s["scales"][a] * delta, y)
    return y


def _exact_controls(case, s):
    logits = s["logits"].double()
    bits = (s["masks"].long() & 0xFFFFFFFF).cpu()
    lens, prompts = s["lens"].tolist(), s["prompt_lens"].tolist()
    for r in range(case["rows"]):
        row = logits[r]
        said = s["history"][r, :lens[r]].long()
        old = torch.unique(said)
        rep = s["repetition"][r].double()
        row[old] = torch.where(row[old] > 0, row[old] / rep, row[old] * rep)
        new, times = torch.unique(said[prompts[r]:], return_counts=True)
        row[new] -= s["frequency"][r].double() * times + s["presence"][r].double()
        n = case["biases"]
        if n:
            row[s["bias_ids"][r * n:(r + 1) * n].long()] += s["bias_values"][r * n:(r + 1) * n].double()
        m = int(s["mask_index"][r])
        if m >= 0:
            ids = torch.arange(case["vocab"])
            off = ((bits[m][ids // 32] >> (ids % 32)) & 1) == 0
            row[off.to(row.device)] = -math.inf
    return logits
