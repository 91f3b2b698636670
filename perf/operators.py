"""Cases of the operators that surround the skinny GEMMs in a verify step, and their plain forms.

A verify step runs a few token rows per request through qkv_proj, attention, o_proj, the MLP and the
lm_head. The projections are this library's GEMMs; the operators here are the ones between them:

* ``rope``            rotary positions on the rows' query and key heads;
* ``rope_cache``      the same, with the rotated keys and the values written to a paged cache;
* ``prefix_attn``     attention of the rows over that cache, where all requests share a long prefix;
* ``logits_process``  penalties for repeated tokens, biases and grammar masks on the lm_head's logits.

``run`` computes them from elementary torch operations, or through ``torch.ops.gfx906_skinny`` where
``own`` is true.
"""

import math

import torch

own = False

_ops = None

DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
BYTES = {"float16": 2, "bfloat16": 2, "float32": 4}


def _library():
    global _ops
    if _ops is None:
        from __graft_entry__ import load_package

        _ops = load_package().ops()
    return _ops


# ------------------------------------------------------------------------------------------------
# The cases
# ------------------------------------------------------------------------------------------------
def _rope(name, op, rows, q_heads, kv_heads, dim, rot, dtype, interleaved, scaling, top, page=16):
    return {"name": name, "op": op, "rows": rows, "q_heads": q_heads, "kv_heads": kv_heads,
            "dim": dim, "rot": rot, "dtype": dtype, "interleaved": interleaved, "scaling": scaling,
            "top": top, "page": page}


def _attn(name, requests, rows, prefix, own_len, q_heads, kv_heads, dim, dtype, page, tree=False):
    return {"name": name, "op": "prefix_attn", "requests": requests, "rows": rows, "prefix": prefix,
            "own_len": own_len, "q_heads": q_heads, "kv_heads": kv_heads, "dim": dim,
            "dtype": dtype, "page": page, "tree": tree}


def _logits(name, requests, rows, vocab, shard, history, dtype, biases, mask):
    return {"name": name, "op": "logits_process", "requests": requests, "rows": rows,
            "vocab": vocab, "shard": shard, "history": history, "dtype": dtype, "biases": biases,
            "mask": mask}


def listed():
    return [
        # The eight rows of one verify step, cut out of the qkv_proj output (24 query and 4 KV
        # heads of 256, of which the first 64 dimensions turn): what one layer does between its
        # first GEMM and its attention. Latency counts.
        _rope("rope verify rows", "rope", 8, 24, 4, 256, 64, "float16", False, "none", 32768),
        # A long prompt's chunk at far positions, interleaved pairs, frequencies scaled for it.
        _rope("rope prompt", "rope", 4099, 32, 8, 128, 128, "bfloat16", True, "yarn", 1 << 20),
        # The same eight rows with their keys and values going to the cache.
        _rope("rope_cache verify rows", "rope_cache", 8, 24, 4, 256, 64, "float16", False, "none",
              32768, 16),
        # A prompt chunk that fills the cache.
        _rope("rope_cache prompt", "rope_cache", 2048, 32, 8, 128, 128, "bfloat16", False, "linear",
              131072, 64),
        # One request at the start of its answer, one row: the smallest call there is.
        _attn("attn one short row", 1, 1, 0, 33, 24, 4, 256, "float16", 16),
        # One request, eight verified rows, a long cache of its own.
        _attn("attn one long request", 1, 8, 0, 32775, 24, 4, 256, "float16", 16),
        # Eight requests with one row each behind a system prompt of 32 thousand tokens.
        _attn("attn eight on a prefix", 8, 8, 32768, 600, 24, 4, 256, "float16", 16),
        # Four draft trees of eight rows behind a medium prompt, small heads.
        _attn("attn draft trees", 4, 32, 4093, 257, 16, 2, 64, "float16", 32, True),
        # A serving batch: 64 requests, one row each, on a prefix of 32 thousand tokens.
        _attn("attn batch on a prefix", 64, 64, 32768, 1500, 32, 8, 128, "bfloat16", 64),
        # One request's single row over one rank's shard of the lm_head.
        _logits("logits shard, one row", 1, 1, 151936, 18992, 300, "float16", 0, False),
        # The eight rows of a verify step over the whole vocabulary, all processors on.
        _logits("logits verify rows", 1, 8, 151936, 151936, 8192, "float16", 300, True),
        # A serving batch of 128 rows with long histories.
        _logits("logits batch", 128, 128, 151936, 151936, 16384, "float16", 32, True),
    ]


def _spread(rng, lo, hi):
    """A whole number of [lo, hi], even over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "rope_cache", "prefix_attn", "prefix_attn", "logits_process",
                     "logits_process"])
    dtype = rng.choice(["float16", "bfloat16"])
    if op in ("rope", "rope_cache"):
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 3, 4, 6, 8])
        dim = rng.choice([64, 80, 96, 128, 192, 256])
        rot = rng.choice([dim, dim // 2, dim // 4])
        cap = (4099 if op == "rope" else 2048) * 48 * 128
        rows = min(_spread(rng, 1, 4099), cap // ((heads + 2 * kv) * dim))
        case = _rope("", op, rows, heads, kv, dim, rot - rot % 2, dtype, rng.random() < 0.5,
                     rng.choice(["none", "linear", "yarn"]), _spread(rng, 4096, 1 << 20),
                     rng.choice([16, 32, 64]))
    elif op == "prefix_attn":
        kv = rng.choice([1, 2, 4, 8])
        heads = kv * rng.choice([1, 2, 4, 6, 8])
        dim = rng.choice([64, 80, 128, 128, 256])
        requests = _spread(rng, 1, 64)
        rows = min(64, requests * rng.choice([1, 1, 2, 4, 7, 8]))
        prefix = rng.choice([0, 1, 1, 1]) * _spread(rng, 16, 32768)
        own_len = _spread(rng, rows // requests + 1, 2000 if requests > 1 else 32775)
        case = _attn("", requests, rows, prefix, own_len, heads, kv, dim, dtype,
                     rng.choice([16, 32, 64, 128]), rng.random() < 0.25)
        top = work(next(c for c in listed() if c["name"] == "attn batch on a prefix"))
        while any(work(case)[n] > top[n] for n in top):
            case["prefix"], case["own_len"] = case["prefix"] // 2, case["own_len"] // 2 + 8
    else:
        requests = _spread(rng, 1, 128)
        rows = min(128, requests * rng.choice([1, 1, 2, 4, 8]))
        vocab = rng.choice([32000, 50257, 128256, 151936])
        shard = rng.choice([vocab, vocab, vocab // 2, vocab // 8])
        case = _logits("", requests, rows, vocab, shard, _spread(rng, 1, 16384),
                       rng.choice(["float16", "bfloat16", "float32"]),
                       rng.choice([0, 1, 17, 300]), rng.random() < 0.5)
        most = work(next(c for c in listed() if c["name"] == "logits batch"))["bytes"]
        while work(case)["bytes"] > most:
            case["rows"] = rows = rows - 1
            case["requests"] = min(requests, rows)
    del case["name"]
    return case


def _ragged(most, count, least=1):
    """`count` lengths up to `most`, spread over its upper three quarters; the first is `most`."""
    return [max(least, most - int((i * 0.6180339887 % 1.0) * 0.75 * most)) for i in range(count)]


def _rows_of(case):
    """How many of the rows each request has."""
    n, b = case["rows"], case["requests"]
    return [n // b + (1 if i < n % b else 0) for i in range(b)]


def work(case):
    es, op = BYTES[case["dtype"]], case["op"]
    if op in ("rope", "rope_cache"):
        heads = case["q_heads"] + case["kv_heads"] * (1 if op == "rope" else 2)
        turned = case["q_heads"] + case["kv_heads"]
        return {"bytes": case["rows"] * (2 * heads * case["dim"] * es + (8 if op == "rope" else 16))
                + 2 * case["rot"], "flops": 3 * case["rows"] * turned * case["rot"]}
    if op == "prefix_attn":
        rows, lens = _rows_of(case), _ragged(case["own_len"], case["requests"], 8)
        keys = case["prefix"] + sum(lens)
        pairs = case["rows"] * case["prefix"] + sum(n * m for n, m in zip(rows, lens))
        head = case["dim"] * es
        return {"bytes": 2 * keys * case["kv_heads"] * head + 2 * case["rows"] * case["q_heads"] * head
                + 4 * case["rows"] * case["q_heads"] + 4 * (keys // case["page"]),
                "flops": 4 * pairs * case["q_heads"] * case["dim"]}
    cells = case["rows"] * case["shard"]
    return {"bytes": cells * (es + 4) + 4 * sum(_ragged(case["history"], case["requests"]))
            + (cells // 8 if case["mask"] else 0) + 8 * case["rows"] * case["biases"],
            "flops": 6 * cells}


# ------------------------------------------------------------------------------------------------
# Inputs
# ------------------------------------------------------------------------------------------------
def _frequencies(rot, scaling, top):
    """Inverse frequencies (float32) of base 10^6 and the factor on cos and sin."""
    i = torch.arange(rot // 2, dtype=torch.float64)
    f = 1e6 ** (-2.0 * i / rot)
    if scaling == "linear":
        return (f / 4.0).float(), 1.0
    if scaling == "yarn":
        # frequencies that turn less than once over the trained length are stretched, those that
        # turn often are kept, with a linear ramp between
        turns = f * (top / 8.0) / (2 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0, 1)
        return (f * keep + f / 8.0 * (1 - keep)).float(), 0.1 * math.log(8.0) + 1.0
    return f.float(), 1.0


def _prepare_rope(case, g):
    t, hq, hk, d = case["rows"], case["q_heads"], case["kv_heads"], case["dim"]
    dt = DTYPES[case["dtype"]]
    # one projection's output; query, key and value heads are views of its columns
    qkv = torch.randn(t, (hq + 2 * hk) * d, device="cuda", generator=g).to(dt)
    q = qkv[:, :hq * d].unflatten(1, (hq, d))
    k = qkv[:, hq * d:(hq + hk) * d].unflatten(1, (hk, d))
    v = qkv[:, (hq + hk) * d:].unflatten(1, (hk, d))
    inv, factor = _frequencies(case["rot"], case["scaling"], case["top"])
    start = torch.randint(0, max(1, case["top"] - t), (1,), device="cuda", generator=g)
    s = {"case": case, "q": q, "k": k, "v": v, "positions": start + torch.arange(t, device="cuda"),
         "inv_freq": inv.cuda(), "scale": factor, "interleaved": case["interleaved"]}
    if case["op"] == "rope_cache":
        page = case["page"]
        pages = -(-t // page) + 3
        order = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(t, device="cuda") + int(page // 3)
        s["slots"] = order[at // page] * page + at % page
        s["k_cache"] = torch.randn(pages, page, hk, d, device="cuda", generator=g).to(dt)
        s["v_cache"] = torch.randn(pages, page, hk, d, device="cuda", generator=g).to(dt)
    return s


def _prepare_attn(case, g):
    b, t, hq, hk, d = (case[n] for n in ("requests", "rows", "q_heads", "kv_heads", "dim"))
    page, dt = case["page"], DTYPES[case["dtype"]]
    lens = _ragged(case["own_len"], b, 8)
    shared, each = -(-case["prefix"] // page), -(-max(lens) // page)
    need = [-(-n // page) for n in lens]
    total = shared + sum(need) + 2
    order = torch.randperm(total, device="cuda", generator=g).int()
    # a request's row of the page table ends where its pages do; the rest is unused
    pages = torch.full((b, each), -1, dtype=torch.int32)
    at = shared
    index = torch.zeros(b, each, dtype=torch.int64)
    for i, n in enumerate(need):
        index[i, :n] = torch.arange(at, at + n)
        pages[i, :n] = 0
        at += n
    pages = torch.where(pages.cuda() < 0, pages.cuda(), order[index.cuda()])
    starts = [0]
    for n in _rows_of(case):
        starts.append(starts[-1] + n)
    # keys carry an offset per channel, as those of trained models do
    k = torch.randn(total, page, hk, d, device="cuda", generator=g, dtype=torch.float32).to(dt)
    k += (0.5 * torch.randn(hk, d, device="cuda", generator=g)).to(dt)
    v = torch.randn(total, page, hk, d, device="cuda", generator=g, dtype=torch.float32).to(dt)
    s = {"case": case, "q": (1.5 * torch.randn(t, hq, d, device="cuda", generator=g)).to(dt),
         "k_cache": k, "v_cache": v, "prefix_pages": order[:shared].contiguous(),
         "prefix_len": torch.tensor([case["prefix"]], dtype=torch.int32, device="cuda"),
         "pages": pages, "own_lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
         "row_start": torch.tensor(starts, dtype=torch.int32, device="cuda"),
         "scale": d ** -0.5, "tree": None}
    if case["tree"]:
        # row i of a request hangs below a random earlier row: it sees itself and its ancestors
        masks = []
        parent = torch.randint(0, 1 << 30, (t,), device="cuda", generator=g).tolist()
        for n in _rows_of(case):
            seen = []
            for i in range(n):
                up = parent[len(masks) + i] % (i + 1) - 1
                seen.append((seen[up] if up >= 0 else 0) | 1 << i)
            masks += seen
        s["tree"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
    return s


def _prepare_logits(case, g):
    b, r, vocab, shard = case["requests"], case["rows"], case["vocab"], case["shard"]
    lens = _ragged(case["history"], b)
    # few tokens are frequent and many are rare
    u = torch.rand(b, case["history"], device="cuda", generator=g)
    tokens = (vocab * u ** 4).int().clamp(max=vocab - 1)
    tokens = (tokens * 7919 % vocab).int() if vocab < 200000 else tokens
    rows = _rows_of(case)
    seq = [i for i, n in enumerate(rows) for _ in range(n)]
    # row i of a request sees its history up to the drafted token before it
    total = [max(1, lens[i] - n + 1 + j) for i, n in enumerate(rows) for j in range(n)]
    logits = (3.0 * torch.randn(r, shard, device="cuda", generator=g)).to(DTYPES[case["dtype"]])
    pick = lambda lo, hi: lo + (hi - lo) * torch.rand(r, device="cuda", generator=g)  # noqa: E731
    s = {"case": case, "logits": logits, "tokens": tokens,
         "row_seq": torch.tensor(seq, dtype=torch.int32, device="cuda"),
         "prompt_lens": torch.tensor([lens[i] // 2 for i in seq], dtype=torch.int32, device="cuda"),
         "total_lens": torch.tensor(total, dtype=torch.int32, device="cuda"),
         "repetition": pick(1.0, 1.3), "frequency": pick(-0.2, 0.6), "presence": pick(0.0, 0.5),
         "bias_ids": None, "bias_values": None, "mask": None,
         "vocab_start": (vocab // shard - 1) * shard // 2 if shard < vocab else 0}
    if case["biases"]:
        n = case["biases"]
        ids = torch.randint(0, vocab, (r, n), device="cuda", generator=g).int()
        used = torch.arange(n, device="cuda") < torch.randint(0, n + 1, (r, 1), device="cuda", generator=g)
        s["bias_ids"] = torch.where(used, ids, torch.full_like(ids, -1))
        s["bias_values"] = 4.0 * torch.randn(r, n, device="cuda", generator=g)
    if case["mask"]:
        # a grammar allows nearly everything inside a string and little elsewhere
        words = -(-vocab // 32)
        share = torch.rand(r, 1, 1, device="cuda", generator=g) < 0.5
        bits = torch.rand(r, words, 32, device="cuda", generator=g) < torch.where(share, 0.97, 0.02)
        weight = (1 << torch.arange(32, device="cuda", dtype=torch.int64))
        s["mask"] = (bits * weight).sum(-1).to(torch.int32)
    return s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    make = {"rope": _prepare_rope, "rope_cache": _prepare_rope, "prefix_attn": _prepare_attn,
            "logits_process": _prepare_logits}[case["op"]]
    return make(case, g)


# ------------------------------------------------------------------------------------------------
# One pass
# ------------------------------------------------------------------------------------------------
def _turn(x, cos, sin, rot, interleaved):
    x = x.float()
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    c, s = cos[:, None], sin[:, None]
    u, w = a * c - b * s, b * c + a * s
    turned = torch.stack((u, w), -1).flatten(-2) if interleaved else torch.cat((u, w), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _rope_plain(s):
    angle = s["positions"].double()[:, None] * s["inv_freq"].double()
    cos, sin = (angle.cos() * s["scale"]).float(), (angle.sin() * s["scale"]).float()
    rot, dt = 2 * s["inv_freq"].numel(), s["q"].dtype
    q = _turn(s["q"], cos, sin, rot, s["interleaved"]).to(dt)
    k = _turn(s["k"], cos, sin, rot, s["interleaved"]).to(dt)
    if s["case"]["op"] == "rope":
        return q, k
    hk, d = k.shape[1:]
    s["k_cache"].view(-1, hk, d)[s["slots"]] = k
    s["v_cache"].view(-1, hk, d)[s["slots"]] = s["v"]
    return q, s["k_cache"], s["v_cache"]


def _attn_plain(s):
    q, kc, vc = s["q"], s["k_cache"], s["v_cache"]
    t, hq, d = q.shape
    page, hk = kc.shape[1:3]
    qg = q.float().view(t, hk, hq // hk, d) * s["scale"]
    rows = torch.arange(t, device=q.device)
    # the request of each row, and the row's place among its request's rows
    seq = torch.searchsorted(s["row_start"][1:].long(), rows, right=True)
    first, count = s["row_start"][seq], s["row_start"][seq + 1] - s["row_start"][seq]
    place = rows - first
    # every row sees the whole prefix
    kp = kc[s["prefix_pages"].long()].reshape(-1, hk, d).float()
    vp = vc[s["prefix_pages"].long()].reshape(-1, hk, d).float()
    sp = torch.einsum("thgd,phd->thgp", qg, kp)
    hidden = torch.arange(kp.shape[0], device=q.device) >= s["prefix_len"]
    sp.masked_fill_(hidden, -math.inf)
    # its request's own tokens up to itself, or those of its branch
    table = s["pages"][seq].long().clamp(min=0)
    ko = kc[table].reshape(t, -1, hk, d).float()
    vo = vc[table].reshape(t, -1, hk, d).float()
    so = torch.einsum("thgd,tphd->thgp", qg, ko)
    at = torch.arange(ko.shape[1], device=q.device)
    new = at - (s["own_lens"][seq] - count)[:, None]
    if s["tree"] is None:
        sees = new <= place[:, None]
    else:
        sees = (new < 0) | ((s["tree"][:, None] >> new.clamp(0, 63)) & 1 > 0) & (new < 64)
    sees &= at < s["own_lens"][seq][:, None]
    so.masked_fill_(~sees[:, None, None], -math.inf)
    top = sp.amax(-1) if kp.shape[0] else torch.full_like(so[..., 0], -math.inf)
    top = torch.maximum(top, so.amax(-1))
    base = torch.where(top == -math.inf, torch.zeros_like(top), top)
    pp, po = (sp - base[..., None]).exp(), (so - base[..., None]).exp()
    total = pp.sum(-1) + po.sum(-1)
    out = torch.einsum("thgp,phd->thgd", pp, vp) + torch.einsum("thgp,tphd->thgd", po, vo)
    out = torch.where(total[..., None] > 0, out / total[..., None], torch.zeros_like(out))
    lse = base + total.log()
    return out.reshape(t, hq, d).to(q.dtype), lse.reshape(t, hq)


def _logits_plain(s):
    x = s["logits"].float()
    r, v = x.shape
    history = s["tokens"][s["row_seq"].long()].long() - s["vocab_start"]
    at = torch.arange(history.shape[1], device=x.device)
    valid = (at < s["total_lens"][:, None]) & (history >= 0) & (history < v)
    answer = valid & (at >= s["prompt_lens"][:, None])
    bin_ = lambda which: torch.zeros(r, v + 1, device=x.device).scatter_add_(  # noqa: E731
        1, torch.where(which, history, torch.full_like(history, v)), torch.ones_like(history, dtype=torch.float32))[:, :v]
    seen, count = bin_(valid) > 0, bin_(answer)
    rep = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / rep, x * rep), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    if s["bias_ids"] is not None:
        ids = s["bias_ids"].long() - s["vocab_start"]
        inside = (s["bias_ids"] >= 0) & (ids >= 0) & (ids < v)
        added = torch.zeros(r, v + 1, device=x.device, dtype=torch.float64)
        added.scatter_add_(1, torch.where(inside, ids, torch.full_like(ids, v)), s["bias_values"].double())
        x = x + added[:, :v].float()
    if s["mask"] is not None:
        token = torch.arange(v, device=x.device) + s["vocab_start"]
        allowed = (s["mask"][:, token >> 5] >> (token & 31)) & 1
        x = torch.where(allowed > 0, x, torch.full_like(x, -math.inf))
    return x


def run(state):
    op, s = state["case"]["op"], state
    if not own:
        plain = {"prefix_attn": _attn_plain, "logits_process": _logits_plain}.get(op, _rope_plain)
        return plain(s)
    ops = _library()
    if op == "rope":
        return ops.rope(s["q"], s["k"], s["positions"], s["inv_freq"], s["scale"], s["interleaved"])
    if op == "rope_cache":
        q = ops.rope_cache(s["q"], s["k"], s["v"], s["positions"], s["inv_freq"], s["slots"],
                           s["k_cache"], s["v_cache"], s["scale"], s["interleaved"])
        return q, s["k_cache"], s["v_cache"]
    if op == "prefix_attn":
        return ops.prefix_attn(s["q"], s["k_cache"], s["v_cache"], s["prefix_pages"],
                               s["prefix_len"], s["pages"], s["own_lens"], s["row_start"],
                               s["scale"], s["tree"])
    return ops.logits_process(s["logits"], s["tokens"], s["row_seq"], s["prompt_lens"],
                              s["total_lens"], s["repetition"], s["frequency"], s["presence"],
                              s["bias_ids"], s["bias_values"], s["mask"], s["vocab_start"])


# ------------------------------------------------------------------------------------------------
# The definitions in 64 bits
# ------------------------------------------------------------------------------------------------
def _exact_rope(s):
    rot = 2 * s["inv_freq"].numel()
    angle = s["positions"].double()[:, None, None] * s["inv_freq"].double()
    phase = torch.polar(torch.full_like(angle, s["scale"]), angle)

    def turned(x):
        x = x.double().clone()
        i = torch.arange(rot // 2, device=x.device)
        lo, hi = (2 * i, 2 * i + 1) if s["interleaved"] else (i, i + rot // 2)
        z = torch.complex(x[..., lo], x[..., hi]) * phase
        x[..., lo], x[..., hi] = z.real, z.imag
        return x

    q, k = turned(s["q"]), turned(s["k"])
    if s["case"]["op"] == "rope":
        return q, k
    page = s["k_cache"].shape[1]
    kc, vc = s["k_cache"].double(), s["v_cache"].double()
    kc[s["slots"] // page, s["slots"] % page] = k
    vc[s["slots"] // page, s["slots"] % page] = s["v"].double()
    return q, kc, vc


def _exact_attn(s):
    case, page = s["case"], s["case"]["page"]
    group, p = case["q_heads"] // case["kv_heads"], case["prefix"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.full(s["q"].shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    at = 0
    for i, (n, m) in enumerate(zip(_rows_of(case), _ragged(case["own_len"], case["requests"], 8))):
        token = torch.arange(m, device="cuda")
        where = s["pages"][i].long()[token // page] * page + token % page
        token = torch.arange(p, device="cuda")
        if p:
            where = torch.cat((s["prefix_pages"].long()[token // page] * page + token % page, where))
        for j in range(n):
            last = m - n
            branch = (1 << (j + 1)) - 1 if s["tree"] is None else int(s["tree"][at])
            pick = [x for x in range(n) if branch >> x & 1]
            seen = torch.cat((torch.arange(p + last, device="cuda"),
                              p + last + torch.tensor(pick, dtype=torch.int64, device="cuda")))
            rows = where[seen]
            for h in range(case["kv_heads"]):
                k = s["k_cache"].flatten(0, 1)[rows, h].double()
                v = s["v_cache"].flatten(0, 1)[rows, h].double()
                heads = slice(h * group, (h + 1) * group)
                score = s["q"][at, heads].double() @ k.T * s["scale"]
                out[at, heads] = torch.softmax(score, -1) @ v
                lse[at, heads] = torch.logsumexp(score, -1)
            at += 1
    return out, lse


def _exact_logits(s):
    x = s["logits"].double()
    v, lo = x.shape[1], s["vocab_start"]
    for i in range(x.shape[0]):
        n, p = int(s["total_lens"][i]), int(s["prompt_lens"][i])
        text = s["tokens"][int(s["row_seq"][i]), :n].long()
        every = torch.bincount(text, minlength=lo + v)[lo:lo + v]
        count = torch.bincount(text[p:], minlength=lo + v)[lo:lo + v].double()
        rep = float(s["repetition"][i])
        y = x[i]
        y = torch.where(every > 0, torch.where(y > 0, y / rep, y * rep), y)
        y = y - float(s["frequency"][i]) * count - float(s["presence"][i]) * (count > 0)
        if s["bias_ids"] is not None:
            ids, values = s["bias_ids"][i].long(), s["bias_values"][i].double()
            keep = (ids >= lo) & (ids < lo + v)
            y = y.index_add(0, ids[keep] - lo, values[keep])
        if s["mask"] is not None:
            word = s["mask"][i].long()[:, None] >> torch.arange(32, device="cuda") & 1
            y = y.masked_fill(word.flatten()[lo:lo + v] == 0, -math.inf)
        x[i] = y
    return x


def exact(case, seed):
    s = prepare(case, seed)
    make = {"prefix_attn": _exact_attn, "logits_process": _exact_logits}.get(case["op"], _exact_rope)
    return make(s)
