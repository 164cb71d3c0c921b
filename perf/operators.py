"""Operators of a paged cache: what writes its pages, attention that reads them, and copies of pages.

* ``norm_rope``: a projection's rows [tokens, (nq + 2 nkv) hd]; bias; RMS norm with a weight on every query and key head; rotation of
  entry i with entry i + hd/2; queries come out as rows of their own, keys and values go to their page slots.
* ``store4``: the same, the norms optional, with keys and values held in 4 bits; and the stored values read back.
* ``decode4``: one query a request over pages held in 4 bits.
* ``portion4``: portions of prompts over pages held in 4 bits, causal.
* ``pages``: copies of pages in every layer's pool.

Pages are [num_pages, nkv, page, row]. Four bits: a row holds its entries in groups of 32, each with a scale s and a centre c (bfloat16)
and a number n from 0 to 15 for each entry, which stands for c + s (n - 8); s = (max - min) / 15, c = min + 8 s. With G groups, a row
is 16 G bytes of numbers and then (s, c) of each group. Keys: entry d of group g lies in 32-bit word (d % 32 // 8) G + g at bit
4 (d % 8); values: in 16-bit word (d % 32 // 4) G + g at bit 4 (d % 4).
"""

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
EPS = 1e-5
GROUP = 32
POSITIONS = 16384


# ------------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the norms and the rotation of one layer of a prompt of 2048 tokens, at the heads of the 8B preset
        {"name": "norms and rotation, prompt", "op": "norm_rope", "dtype": "bfloat16", "tokens": 2048, "nq": 32, "nkv": 8, "hd": 128, "page": 16,
         "bias": False},
        # a 32-bit model with few heads of an odd size, a bias, and a step of prompt rests and single tokens
        {"name": "norms and rotation, 32 bits", "op": "norm_rope", "dtype": "float32", "tokens": 333, "nq": 12, "nkv": 4, "hd": 96, "page": 8,
         "bias": True},
        # one layer's keys and values of a decode step of 64 requests
        {"name": "store, decode step", "op": "store4", "dtype": "bfloat16", "tokens": 64, "nq": 32, "nkv": 8, "hd": 128, "page": 16, "bias": False,
         "norms": False},
        # one layer's keys and values of a prompt, behind head norms
        {"name": "store, prompt", "op": "store4", "dtype": "bfloat16", "tokens": 2048, "nq": 32, "nkv": 8, "hd": 128, "page": 16, "bias": True,
         "norms": True},
        # a chat of one user: the smallest call, where latency counts
        {"name": "decode, one request", "op": "decode4", "dtype": "bfloat16", "requests": 1, "context": 2048, "nq": 32, "nkv": 8, "hd": 128, "page": 16,
         "window": 0, "softcap": 0.0, "sinks": False, "slopes": False},
        # a full batch with long contexts of different lengths: the bytes of the cache count
        {"name": "decode, 64 requests", "op": "decode4", "dtype": "bfloat16", "requests": 64, "context": 8192, "nq": 32, "nkv": 8, "hd": 128, "page": 16,
         "window": 0, "softcap": 0.0, "sinks": False, "slopes": False},
        # a windowed layer with capped scores and sinks, small heads, an odd context
        {"name": "decode, window and sinks", "op": "decode4", "dtype": "bfloat16", "requests": 5, "context": 5003, "nq": 16, "nkv": 8, "hd": 64, "page": 32,
         "window": 1024, "softcap": 30.0, "sinks": True, "slopes": False},
        # the last portion of a prompt of 8192 tokens
        {"name": "portion behind a context", "op": "portion4", "dtype": "bfloat16", "requests": 1, "portion": 2048, "context": 8192, "nq": 32, "nkv": 8,
         "hd": 128, "page": 16, "window": 0, "softcap": 0.0, "sinks": False, "slopes": False},
        # the rests of eight prompts in one step, small heads, a penalty on the distance
        {"name": "portions of eight requests", "op": "portion4", "dtype": "bfloat16", "requests": 8, "portion": 211, "context": 1500, "nq": 16, "nkv": 4,
         "hd": 64, "page": 16, "window": 0, "softcap": 0.0, "sinks": False, "slopes": True},
        # a 32-bit model, whose results may not depend on how a prompt is cut
        {"name": "portion, 32 bits", "op": "portion4", "dtype": "float32", "requests": 2, "portion": 50, "context": 1000, "nq": 12, "nkv": 4, "hd": 64,
         "page": 16, "window": 0, "softcap": 0.0, "sinks": True, "slopes": False},
        # eight requests fork: each one's last page, in all 32 layers
        {"name": "pages, forks", "op": "pages", "dtype": "bfloat16", "layers": 32, "pool": 128, "copies": 8, "nkv": 8, "page": 16, "row": 128},
        # a long request is given pages of its own, held in 4 bits
        {"name": "pages, a long request", "op": "pages", "dtype": "uint8", "layers": 32, "pool": 1200, "copies": 512, "nkv": 8, "page": 16, "row": 80},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "store4", "decode4", "decode4", "portion4", "portion4", "pages"])
    nkv = rng.choice([1, 2, 4, 8])
    heads = {"nq": nkv * rng.choice([1, 2, 3, 4, 7, 8] if nkv <= 4 else [1, 2, 4]), "nkv": nkv, "page": rng.choice([8, 16, 16, 16, 32, 64])}
    if op in ("norm_rope", "store4"):
        case = {"op": op, "dtype": rng.choice(["bfloat16", "bfloat16", "float32"]), "tokens": _log(rng, 1, 2048), **heads,
                "hd": rng.choice([64, 80, 96, 128]), "bias": rng.random() < 0.5}
        return dict(case, norms=rng.random() < 0.5) if op == "store4" else case
    rules = {"window": rng.choice([0, 0, 0, 100, 1024]), "softcap": rng.choice([0.0, 0.0, 30.0]), "sinks": rng.random() < 0.3, "slopes": rng.random() < 0.3}
    if op == "decode4":
        return {"op": op, "dtype": "bfloat16", "requests": _log(rng, 1, 64), "context": _log(rng, 64, 8192), **heads, "hd": rng.choice([64, 128]), **rules}
    if op == "portion4":
        if rng.random() < 0.25:
            return {"op": op, "dtype": "float32", "requests": rng.choice([1, 2, 3]), "portion": _log(rng, 1, 60), "context": _log(rng, 64, 1000), **heads,
                    "hd": rng.choice([32, 64, 128]), **rules}
        requests = rng.choice([1, 1, 2, 3, 5, 8])
        portion = _log(rng, 2, 2048 // requests)
        return {"op": op, "dtype": "bfloat16", "requests": requests, "portion": portion, "context": portion + _log(rng, 1, 6144), **heads,
                "hd": rng.choice([64, 128]), **rules}
    case = {"op": op, "dtype": rng.choice(["bfloat16", "float32", "uint8"]), "nkv": nkv, "page": heads["page"], "row": rng.choice([40, 64, 80, 128])}
    layers = rng.randint(1, 32)
    page_bytes = nkv * case["page"] * case["row"] * {"bfloat16": 2, "float32": 4, "uint8": 1}[case["dtype"]]
    pool = _log(rng, 20, max(21, min(1200, (300 << 20) // (layers * page_bytes))))
    return dict(case, layers=layers, pool=pool, copies=_log(rng, 1, pool // 2))


def _lengths(case):
    """Keys of each request after the step: the first has the whole context, the others three quarters of it and less, all different."""
    n, full = case["requests"], case["context"]
    least = case.get("portion", 1)
    return [full] + [max(least, full - full // 4 - (i * 977) % max(1, full // 2)) for i in range(1, n)]


def _portions(case):
    """Tokens that each request brings."""
    lengths = _lengths(case)
    most = case.get("portion", 1)
    return [min(n, most - (i * 37) % max(1, most // 3)) for i, n in enumerate(lengths)]


def _groups(hd):
    return -(-hd // GROUP)


# ------------------------------------------------------------------------------------------------------------------ four bits
def _places(hd, which, device):
    """(byte, shift) of every entry of a row."""
    d = torch.arange(hd, device=device)
    group, within, G = d // GROUP, d % GROUP, _groups(hd)
    if which == "k":
        return 4 * (within // 8 * G + group) + within % 8 // 2, 4 * (within % 2)
    return 2 * (within // 4 * G + group) + within % 4 // 2, 4 * (within % 2)


def _quantise(x):
    """(n, s, c): [..., G, 32], [..., G], [..., G] of float32 rows [..., hd]; the last group may lack entries (n = 8)."""
    hd, G = x.shape[-1], _groups(x.shape[-1])
    pad = G * GROUP - hd
    grouped = torch.nn.functional.pad(x, (0, pad)).unflatten(-1, (G, GROUP))
    there = (torch.arange(G * GROUP, device=x.device) < hd).view(G, GROUP)
    lo = grouped.masked_fill(~there, math.inf).amin(-1)
    hi = grouped.masked_fill(~there, -math.inf).amax(-1)
    s = ((hi - lo) / 15).to(torch.bfloat16).to(F32)
    s = torch.where(s < 2.0 ** -126, torch.zeros_like(s), s)
    c = (lo + 8 * s).to(torch.bfloat16).to(F32)
    inverse = torch.where(s > 0, 1 / s, torch.zeros_like(s))
    n = (torch.round((grouped - c[..., None]) * inverse[..., None]) + 8).clamp(0, 15)
    return torch.where(there, n, torch.full_like(n, 8.0)), s, c


def _stands_for(n, s, c, hd):
    return (c[..., None] + s[..., None] * (n - 8)).flatten(-2)[..., :hd]


def _pack(n, s, c, which, hd):
    """uint8 rows [..., 20 G]."""
    G = _groups(hd)
    byte, shift = _places(G * GROUP, which, n.device)
    numbers = n.flatten(-2).to(torch.uint8)
    order = torch.argsort(byte * 8 + shift)              # low and high half of byte 0, of byte 1, ...
    halves = numbers[..., order].unflatten(-1, (16 * G, 2))
    packed = halves[..., 0] + 16 * halves[..., 1]
    pairs = torch.stack([s, c], -1).to(torch.bfloat16).contiguous().view(torch.uint8).flatten(-2)
    return torch.cat([packed, pairs], -1)


def _unpack(rows, which, hd):
    """float32 values [..., hd] of uint8 rows."""
    G = _groups(hd)
    byte, shift = _places(hd, which, rows.device)
    n = (rows[..., byte] >> shift.to(torch.uint8)) & 15
    pairs = rows[..., 16 * G:].contiguous().view(torch.bfloat16).to(F32).unflatten(-1, (G, 2))
    of = torch.arange(hd, device=rows.device) // GROUP
    return pairs[..., 1][..., of] + pairs[..., 0][..., of] * (n.to(F32) - 8)


# -------------------------------------------------------------------------------------------------------------------- prepare
def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _tables(hd):
    f = 500000.0 ** (-torch.arange(0, hd, 2, dtype=F64, device="cuda") / hd)
    angles = torch.outer(torch.arange(POSITIONS, dtype=F64, device="cuda"), f)
    return angles.cos().to(F32), angles.sin().to(F32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, dtype = case["op"], getattr(torch, case["dtype"])
    state = {"case": case}
    if op == "pages":
        shape = (case["layers"], case["pool"], case["nkv"], case["page"], case["row"])
        make = (lambda: torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.uint8)) if dtype == torch.uint8 else \
            (lambda: torch.randn(shape, generator=g, device="cuda", dtype=dtype))
        order = torch.randperm(case["pool"], generator=torch.Generator().manual_seed(seed)).tolist()
        return dict(state, pools=[make(), make()], src=order[:case["copies"]], dst=order[case["copies"]:2 * case["copies"]])
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    if op in ("norm_rope", "store4"):
        tokens = case["tokens"]
        width = (nq + 2 * nkv) * hd
        pages = -(-tokens // page) + 3
        spread = 0.5 + torch.rand(width, generator=g, device="cuda")               # channels of different sizes, as projections have them
        state["rows"] = (_normal(g, tokens, width) * spread).to(dtype)
        state["q_out"] = torch.empty((tokens, nq * hd), dtype=dtype, device="cuda")
        state["bias"] = 0.3 * _normal(g, width) if case["bias"] else None
        normed = op == "norm_rope" or case["norms"]
        state["q_norm"], state["k_norm"] = (1 + 0.2 * _normal(g, hd), 1 + 0.2 * _normal(g, hd)) if normed else (None, None)
        state["positions"] = torch.randint(0, POSITIONS, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        state["slots"] = torch.randperm(pages * page, generator=g, device="cuda")[:tokens].to(torch.int32)
        state["cos"], state["sin"] = _tables(hd)
        if op == "norm_rope":
            state["k_pages"], state["v_pages"] = (torch.zeros((pages, nkv, page, hd), dtype=dtype, device="cuda") for _ in "kv")
        else:
            state["k_pages"], state["v_pages"] = (torch.zeros((pages, nkv, page, 20 * _groups(hd)), dtype=torch.uint8, device="cuda") for _ in "kv")
            state["k_read"], state["v_read"] = (torch.empty((tokens, nkv, hd), dtype=dtype, device="cuda") for _ in "kv")
        return state
    lengths, portions = _lengths(case), _portions(case)
    width = -(-max(lengths) // page)
    total = sum(-(-n // page) for n in lengths) + 2
    order = torch.randperm(total, generator=g, device="cuda", dtype=torch.int64)
    rows = total * nkv * page
    for which in "kv":                                                             # keys with a few channels that stand out, as keys have them
        channels = torch.ones(hd, device="cuda")
        if which == "k":
            channels[torch.randperm(hd, generator=g, device="cuda")[:max(1, hd // 32)]] = 3.0
        filled = torch.empty((rows, 20 * _groups(hd)), dtype=torch.uint8, device="cuda")
        for at in range(0, rows, 1 << 19):
            x = _normal(g, min(1 << 19, rows - at), hd) * channels
            filled[at:at + (1 << 19)] = _pack(*_quantise(x), which, hd)
        state[which + "_pages"] = filled.view(total, nkv, page, -1)
    table = torch.full((len(lengths), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lengths):
        have = -(-n // page)
        table[i, :have] = order[at:at + have].to(torch.int32).cpu()
        at += have
    tokens = sum(portions)
    start = [sum(portions[:i]) for i in range(len(portions))]
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    state["table"] = table.cuda()
    state["q_start"], state["q_len"], state["ctx_len"] = ints(start), ints(portions), ints(lengths)
    state["positions"] = ints([n - p + j for n, p in zip(lengths, portions) for j in range(p)])
    state["seq"] = ints([i for i, p in enumerate(portions) for _ in range(p)])
    state["q"] = _normal(g, tokens, nq * hd).to(dtype)
    state["out"] = torch.empty((tokens, nq * hd), dtype=dtype, device="cuda")
    state["sinks"] = _normal(g, nq) if case["sinks"] else None
    state["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / nq) for h in range(nq)], device="cuda") if case["slopes"] else None
    return state


# ------------------------------------------------------------------------------------------------------------------------ run
def _plain_rows(state, norms):
    """Queries, keys and values [tokens, heads, hd] in float32, behind bias, norms and rotation."""
    case = state["case"]
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    x = state["rows"].to(F32)
    if state["bias"] is not None:
        x = x + state["bias"]
    q, k, v = x.unflatten(-1, (nq + 2 * nkv, hd)).split([nq, nkv, nkv], dim=1)
    if norms:
        q, k = (t * torch.rsqrt(t.square().mean(-1, keepdim=True) + EPS) * w for t, w in ((q, state["q_norm"]), (k, state["k_norm"])))
    at = state["positions"].long()
    cos, sin = state["cos"][at][:, None], state["sin"][at][:, None]

    def turned(t):
        a, b = t.chunk(2, -1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return turned(q), turned(k), v


def _plain_write(state):
    case, page = state["case"], state["case"]["page"]
    four = case["op"] == "store4"
    q, k, v = _plain_rows(state, state["q_norm"] is not None)
    dtype = state["rows"].dtype
    at, off = state["slots"].long() // page, state["slots"].long() % page
    if not four:
        state["k_pages"][at, :, off] = k.to(dtype)
        state["v_pages"][at, :, off] = v.to(dtype)
        return [q.flatten(1).to(dtype), state["k_pages"], state["v_pages"]]
    for which, x in (("k", k), ("v", v)):
        state[which + "_pages"][at, :, off] = _pack(*_quantise(x), which, case["hd"])
    read = [_unpack(state[w + "_pages"][at, :, off], w, case["hd"]).to(dtype) for w in "kv"]
    return [q.flatten(1).to(dtype)] + read


def _plain_attention(state):
    """Every query against all keys of its request, in float32; requests side by side, padded to the longest."""
    case = state["case"]
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    table = state["table"].long().clamp(min=0)
    k, v = (_unpack(state[w + "_pages"][table], w, hd).permute(0, 2, 1, 3, 4).flatten(2, 3) for w in "kv")      # [requests, nkv, keys, hd]
    seq, starts = state["seq"].long(), state["q_start"].long()
    most = max(_portions(case))
    requests = table.shape[0]
    at = (torch.arange(state["q"].shape[0], device="cuda") - starts[seq])
    q = torch.zeros((requests, most, nq * hd), device="cuda")
    q[seq, at] = state["q"].to(F32)
    pos = torch.zeros((requests, most), dtype=torch.long, device="cuda")
    pos[seq, at] = state["positions"].long()
    q = q.unflatten(-1, (nkv, nq // nkv, hd)).permute(0, 2, 3, 1, 4).flatten(2, 3)                              # [requests, nkv, group * most, hd]
    x = (q @ k.transpose(-1, -2)).mul_(hd ** -0.5).unflatten(2, (nq // nkv, most))                              # [requests, nkv, group, most, keys]
    if case["softcap"]:
        x = x.div_(case["softcap"]).tanh_().mul_(case["softcap"])
    distance = pos[:, :, None] - torch.arange(k.shape[2], device="cuda")                                        # [requests, most, keys]
    if state["slopes"] is not None:
        x = x - state["slopes"].view(nkv, -1, 1, 1) * distance[:, None, None].to(F32)
    seen = (distance >= 0) & ((distance < case["window"]) if case["window"] else True)
    x = x.masked_fill_(~seen[:, None, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    if state["sinks"] is not None:
        sink = state["sinks"].view(nkv, -1, 1, 1)
        top = torch.maximum(top, sink)
    p = (x.sub_(top)).exp_()
    below = p.sum(-1, keepdim=True)
    if state["sinks"] is not None:
        below = below + (sink - top).exp()
    p = p.div_(below).flatten(2, 3)
    y = (p @ v).unflatten(2, (nq // nkv, most)).permute(0, 3, 1, 2, 4).flatten(2)
    return y[seq, at].to(state["q"].dtype)


def _own(state):
    from stride_b200.csrc import ops
    case = state["case"]
    op = case["op"]
    if op == "pages":
        ops.copy_pages(state["pools"], state["src"], state["dst"])
        return state["pools"]
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    if op in ("norm_rope", "store4"):
        write = ops.qk_norm_rope_write if op == "norm_rope" else ops.rope_kv_write_int4
        write(state["rows"], state["bias"], state["q_norm"], state["k_norm"], EPS, state["positions"], state["slots"], state["cos"], state["sin"],
              state["k_pages"], state["v_pages"], nq, nkv, hd, page, q_out=state["q_out"])
        q = state["q_out"]
        if op == "norm_rope":
            return [q, state["k_pages"], state["v_pages"]]
        ops.read_int4(state["k_pages"], state["v_pages"], state["slots"], state["k_read"], state["v_read"], nkv, hd, page)
        return [q, state["k_read"], state["v_read"]]
    geometry = (nq, nkv, hd, page, hd ** -0.5, case["window"])
    rules = (case["softcap"], state["sinks"], state["slopes"])
    where = (state["q"], nq * hd, state["out"], state["k_pages"], state["v_pages"], state["table"])
    if op == "decode4":
        if "scratch" not in state:
            state["scratch"] = torch.zeros(ops.decode_int4_scratch_floats(case["requests"], nq, nkv, hd, case["context"]), device="cuda")
        ops.paged_attention_decode_int4(*where, state["seq"], state["positions"], state["scratch"], *geometry, case["context"], *rules)
    elif case["dtype"] == "float32":
        ops.paged_attention_int4(*where, state["seq"], state["positions"], *geometry, *rules)
    else:
        keys = sum(_lengths(case))
        if "scratch" not in state:
            state["scratch"] = torch.zeros(ops.prefill_int4_scratch_ints(case["requests"], keys, nkv, hd), dtype=torch.int32, device="cuda")
        ops.paged_attention_prefill_int4(*where, state["q_start"], state["q_len"], state["ctx_len"], state["scratch"], case["requests"], keys,
                                         *geometry, *rules)
    return state["out"]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "pages":
        src, dst = (torch.tensor(state[n], device="cuda") for n in ("src", "dst"))
        for pool in state["pools"]:
            pool[:, dst] = pool[:, src]
        return state["pools"]
    return _plain_write(state) if op in ("norm_rope", "store4") else _plain_attention(state)


# ----------------------------------------------------------------------------------------------------------------------- work
def work(case):
    item = {"bfloat16": 2, "float32": 4, "uint8": 1}[case["dtype"]]
    if case["op"] == "pages":
        return {"bytes": 2 * 2 * case["layers"] * case["copies"] * case["nkv"] * case["page"] * case["row"] * item, "flops": 0}
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    row = 20 * _groups(hd)
    if case["op"] in ("norm_rope", "store4"):
        tokens = case["tokens"]
        bytes_ = tokens * ((nq + 2 * nkv) * hd * item + nq * hd * item + hd * 4 + 8)       # rows in, queries out, angles, position and slot
        bytes_ += tokens * 2 * nkv * (hd * item if case["op"] == "norm_rope" else row + hd * item)      # into the pages; and read back
        return {"bytes": bytes_, "flops": tokens * (nq + 2 * nkv) * hd * 8}
    lengths, portions = _lengths(case), _portions(case)
    window = case["window"] or 1 << 30
    keys = sum(min(n, window + p - 1) for n, p in zip(lengths, portions))
    pairs = 0
    for n, p in zip(lengths, portions):
        for pos in (range(n - p, n) if case["window"] else ()):
            pairs += min(pos + 1, window)
        if not case["window"]:
            pairs += p * (n - p) + p * (p + 1) // 2
    return {"bytes": keys * nkv * 2 * row + 2 * sum(portions) * nq * hd * item, "flops": 4 * nq * hd * pairs}


# ---------------------------------------------------------------------------------------------------------------------- exact
def _exact_row_values(rows, which, hd):
    """The numbers that rows of 4 bits stand for, entry by entry, in float64."""
    out = torch.empty((*rows.shape[:-1], hd), dtype=F64, device=rows.device)
    G = (hd + 31) // 32
    for d in range(hd):
        g, r = divmod(d, 32)
        bit = 32 * (r // 8 * G + g) + 4 * (r % 8) if which == "k" else 16 * (r // 4 * G + g) + 4 * (r % 4)
        n = (rows[..., bit // 8].long() >> (bit % 8)) % 16
        scale, centre = (rows[..., 16 * G + 4 * g + o:16 * G + 4 * g + o + 2].contiguous().view(torch.bfloat16)[..., 0].to(F64) for o in (0, 2))
        out[..., d] = centre + scale * (n - 8)
    return out


def _exact_four_bits(x):
    """float64 rows after a round trip through groups of 32 held in 4 bits."""
    out = torch.empty_like(x)
    for lo in range(0, x.shape[-1], 32):
        part = x[..., lo:lo + 32]
        low, high = part.min(-1, keepdim=True).values, part.max(-1, keepdim=True).values
        scale = ((high - low) / 15).to(torch.bfloat16).to(F64)
        centre = (low + 8 * scale).to(torch.bfloat16).to(F64)
        steps = torch.where(scale > 0, (part - centre) / scale, torch.zeros_like(part)).round().clamp(-8, 7)
        out[..., lo:lo + 32] = centre + scale * steps
    return out


def exact(case, seed):
    if case["op"] == "pages":
        state = prepare(case, seed)
        if case["dtype"] == "uint8":
            return None
        pools = [p.to(F64) for p in state["pools"]] if case["layers"] * case["pool"] * case["page"] * case["row"] * case["nkv"] < 1 << 28 else state["pools"]
        for pool in pools:
            for a, b in zip(state["src"], state["dst"]):
                pool[:, b] = pool[:, a]
        return pools
    state = prepare(case, seed)
    nq, nkv, hd, page = case["nq"], case["nkv"], case["hd"], case["page"]
    if case["op"] in ("norm_rope", "store4"):
        tokens, half = case["tokens"], hd // 2
        x = state["rows"].to(F64)
        x = (x if state["bias"] is None else x + state["bias"].to(F64)).view(tokens, nq + 2 * nkv, hd)
        at = state["positions"].long()
        cos, sin = state["cos"].to(F64)[at], state["sin"].to(F64)[at]
        heads = []
        for h in range(nq + 2 * nkv):
            y = x[:, h]
            if h < nq + nkv:
                w = state["q_norm"] if h < nq else state["k_norm"]
                if w is not None:
                    y = y / ((y * y).sum(-1, keepdim=True) / hd + EPS).sqrt() * w.to(F64)
                y = torch.cat([y[:, :half] * cos - y[:, half:] * sin, y[:, half:] * cos + y[:, :half] * sin], -1)
            heads.append(y)
        y = torch.stack(heads, 1)
        q, k, v = y[:, :nq].reshape(tokens, -1), y[:, nq:nq + nkv], y[:, nq + nkv:]
        if case["op"] == "store4":
            return [q, _exact_four_bits(k), _exact_four_bits(v)]
        pages = [torch.zeros(state["k_pages"].shape, dtype=F64, device="cuda") for _ in "kv"]
        for t, slot in enumerate(state["slots"].tolist()):
            pages[0][slot // page, :, slot % page], pages[1][slot // page, :, slot % page] = k[t], v[t]
        return [q] + pages
    out = torch.empty((sum(_portions(case)), nq * hd), dtype=F64, device="cuda")
    row = 0
    for i, (n, p) in enumerate(zip(_lengths(case), _portions(case))):
        ids = state["table"][i, :-(-n // page)].long()
        keys = torch.arange(n, device="cuda")
        for h in range(nkv):
            k = _exact_row_values(state["k_pages"][ids, h].reshape(-1, 20 * _groups(hd))[:n], "k", hd)
            v = _exact_row_values(state["v_pages"][ids, h].reshape(-1, 20 * _groups(hd))[:n], "v", hd)
            for head in range(h * (nq // nkv), (h + 1) * (nq // nkv)):
                q = state["q"][row:row + p, head * hd:(head + 1) * hd].to(F64)
                scores = q @ k.t() / math.sqrt(hd)
                if case["softcap"]:
                    scores = case["softcap"] * torch.tanh(scores / case["softcap"])
                pos = torch.arange(n - p, n, device="cuda")[:, None]
                if state["slopes"] is not None:
                    scores = scores - state["slopes"][head].to(F64) * (pos - keys)
                hidden = (keys > pos) | ((keys <= pos - case["window"]) if case["window"] else False)
                scores = scores.masked_fill(hidden, -math.inf)
                if state["sinks"] is not None:
                    scores = torch.cat([scores, state["sinks"][head].to(F64).expand(p, 1)], -1)
                weights = torch.softmax(scores, -1)[:, :n]
                out[row:row + p, head * hd:(head + 1) * hd] = weights @ v
        row += p
    return out
