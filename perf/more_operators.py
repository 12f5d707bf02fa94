"""The operators of serving in 8 bits, as they are timed: calls that a program makes of them, and the same
computed with elementary torch operations.

* ``cache``    keys and values of a step written into a cache of 8-bit codes, with a float32 scale for every
               position and key/value head (``ops.rope_store_int8``: q and k are rotated on the way), and the
               pages of the step's sequences read back for the prompt's attention (``ops.read_pages_int8``);
* ``attend``   attention of single tokens, or of a few drafted ones, over such a cache (``ops.attention_int8``);
* ``product``  rows times a matrix held in 8-bit codes with a scale for every row of it; the rows are put into
               codes with a scale for every token first, and the codes are multiplied as whole numbers
               (``ops.linear_int8``).

A value x of a row (a position's head, a token, a row of a matrix) has the code rint(x * (127 / top)) and the row
the scale top / 127, where top is the row's largest magnitude.

Head layouts and widths are those of the SmolLM2 shapes (135M: 9 query and 3 key/value heads of 64, width 576;
360M: 15 and 5, widths 960 and 2,560; 1.7B: 32 and 32, widths 2,048 and 8,192) and heads of 128.
"""
from __future__ import annotations

import math

import torch

own = False

PAGE = 64
_DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


# ---- the cases ----------------------------------------------------------------------------
def listed():
    return [
        # one token of each of eight sequences at contexts of up to 512: launches and latency
        _cache("cache_step_8", "bfloat16", 9, 3, 64, sequences=8, tokens=1, before=511),
        # a prompt of 2,048 tokens, 135M heads
        _cache("cache_prompt_2048", "bfloat16", 9, 3, 64, sequences=1, tokens=2048, before=0),
        # ragged chunks of four prompts behind what they hold already, a key/value head per query head (1.7B)
        _cache("cache_chunks", "bfloat16", 32, 32, 64, sequences=4, tokens=3001, before=1000),
        # one sequence at a short context: launches and latency
        _attend("attend_1x128", "bfloat16", 9, 3, 64, sequences=1, context=128),
        # eight sequences at contexts ending at 4,096
        _attend("attend_8x4096", "bfloat16", 9, 3, 64, sequences=8, context=4096),
        # a server's batch, a key/value head per query head (1.7B), ragged contexts
        _attend("attend_64x4001", "bfloat16", 32, 32, 64, sequences=64, context=4001, ragged=True),
        # four drafted tokens and the one before them per sequence, wide heads, a window
        _attend("attend_drafts_128", "bfloat16", 32, 8, 128, sequences=16, context=8190, tokens=5, window=4000),
        # true float32
        _attend("attend_float32", "float32", 9, 3, 64, sequences=16, context=2000),
        # q, k and v of one token, 135M: launches and latency
        _product("product_1", "bfloat16", m=1, n=960, k=576),
        # gate and up of eight sequences' tokens, 1.7B
        _product("product_8_gated", "bfloat16", m=8, n=8192, k=2048, gated=True),
        # an odd number of rows and columns, float32 operands
        _product("product_odd", "float32", m=333, n=961, k=2555),
        # gate and up of a step of prompts, 1.7B
        _product("product_4096_gated", "bfloat16", m=4096, n=8192, k=2048, gated=True),
    ]


def _cache(name, dtype, heads, kv_heads, dim, sequences, tokens, before):
    return {"name": name, "op": "cache", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "sequences": sequences, "tokens": tokens, "before": before}


def _attend(name, dtype, heads, kv_heads, dim, sequences, context, tokens=1, window=0, ragged=False):
    return {"name": name, "op": "attend", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "sequences": sequences, "context": context, "tokens": tokens, "window": window, "ragged": ragged}


def _product(name, dtype, m, n, k, gated=False):
    return {"name": name, "op": "product", "dtype": dtype, "m": m, "n": n, "k": k, "gated": gated}


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


_HEADS = ((9, 3, 64), (15, 5, 64), (32, 32, 64), (32, 8, 128), (16, 2, 128), (20, 1, 64), (12, 4, 96), (8, 8, 32))


def _draw_once(rng):
    op = rng.choice(("cache", "attend", "attend", "product"))
    dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
    heads, kv_heads, dim = rng.choice(_HEADS)
    if op == "cache":
        sequences = _log_int(rng, 1, 16)
        return _cache("", dtype, heads, kv_heads, dim, sequences=sequences, tokens=_log_int(rng, 1, 4096),
                      before=rng.choice((0, rng.randrange(1, 2000))))
    if op == "attend":
        tokens = rng.choice((1, 1, 1, 2, 5))
        context = _log_int(rng, tokens, 16384 if dtype == "bfloat16" else 4096)
        return _attend("", dtype, heads, kv_heads, dim, sequences=_log_int(rng, 1, 64), context=context, tokens=tokens,
                       window=rng.choice((0, 0, 0, 1 + context // 3)), ragged=rng.choice((True, False)))
    n, k = rng.choice(((960, 576), (576, 576), (960, 960), (2560, 960), (960, 2560), (2048, 2048), (8192, 2048), (2048, 8192),
                       (1001, 517), (130, 4104)))
    return _product("", dtype, m=_log_int(rng, 1, 4096), n=n, k=k, gated=rng.choice((True, False)))


def draw(rng):
    most = {op: max(_cost(c) for c in listed() if c["op"] == op) for op in ("cache", "attend", "product")}
    while True:
        case = _draw_once(rng)
        del case["name"]
        if _cost(case) <= most[case["op"]]:
            return case


def _cost(case):
    w = work(case)
    # (float32 attention costs some eight times the others)
    slow = 8.0 if case["op"] == "attend" and case["dtype"] == "float32" else 1.0
    return max(w["bytes"] / 6.4e12, slow * w["flops"] / 5e14)


# ---- sizes that follow from a case alone ----------------------------------------------------
def _spans(case):
    """(positions held before, new tokens) of every sequence of a cache case: the first brings the most."""
    tokens, before = case["tokens"], case["before"]
    return [((before - i * 61) % (before + 1) if before else 0, max(1, tokens - (i * 997) % tokens))
            for i in range(case["sequences"])]


def _lengths(case):
    """Positions that every sequence of an attention case holds, its new tokens among them."""
    context, least = case["context"], case["tokens"]
    if not case["ragged"]:
        return [context] * case["sequences"]
    return [context - (i * 7919) % max(1, (context - least) // 2 + 1) for i in range(case["sequences"])]


def work(case):
    if case["op"] == "product":
        size, rows = (2 if case["dtype"] == "bfloat16" else 4), case["n"] * (2 if case["gated"] else 1)
        return {"bytes": size * case["m"] * (case["k"] + case["n"]) + rows * case["k"] + 4 * rows,
                "flops": 2 * case["m"] * rows * case["k"]}
    size, heads, kv, dim = (2 if case["dtype"] == "bfloat16" else 4), case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "cache":
        spans = _spans(case)
        new, pages = sum(c for _, c in spans), sum(-(-(s + c) // PAGE) for s, c in spans)
        row = 2 * kv * (dim + 4)                          # codes and scales of a position
        return {"bytes": new * size * (2 * heads + 2 * kv) * dim + new * row + (pages * PAGE - new) * row
                + pages * PAGE * 2 * kv * dim * size + 8 * new + 4 * pages
                + 4 * min(new, max(s + c for s, c in spans)) * dim,
                "flops": new * dim * (3 * (heads + kv) + 4 * kv)}
    lengths, tokens, window = _lengths(case), case["tokens"], case["window"]
    seen = [[min(n - tokens + 1 + j, window or n) for j in range(tokens)] for n in lengths]
    positions = sum(min(n, window + tokens - 1 if window else n) for n in lengths)
    rows = len(lengths) * tokens
    return {"bytes": 2 * positions * kv * (dim + 4) + size * 2 * rows * heads * dim + 8 * rows
            + 4 * sum(-(-n // PAGE) for n in lengths),
            "flops": 4 * heads * dim * sum(map(sum, seen))}


# ---- inputs -----------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    state = {"cache": _prepare_cache, "attend": _prepare_attend, "product": _prepare_product}[case["op"]](case, gen)
    state["case"] = case
    if own:
        from nnis_b200.engine.workspace import Workspace
        state["workspace"] = Workspace(torch.device("cuda"))
    return state


def _page_table(lengths, gen):
    """Pages in random places, as a store that has served for a while hands them out: (table, number of pages)."""
    counts = [-(-n // PAGE) for n in lengths]
    pages = sum(counts) + 3
    ids = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(lengths), max(counts)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = ids[at:at + c]
        at += c
    return table, pages


def _codes(pages, kv_heads, dim, gen):
    """A store as rows with a normal distribution leave it: the largest code of a row is 127, scales vary."""
    shape = (pages, kv_heads, PAGE, dim)
    codes = torch.empty(shape, dtype=torch.float32, device="cuda").normal_(generator=gen)
    top = codes.abs().amax(-1, keepdim=True)
    codes = torch.round(codes * (127.0 / top)).to(torch.int8)
    spread = torch.rand(shape[:3], generator=gen, device="cuda") * 0.5 + 0.75
    return codes, top[..., 0] / 127.0 * spread


def _prepare_cache(case, gen):
    dtype, heads, kv, dim, spans = _DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"], _spans(case)
    n = sum(c for _, c in spans)
    table, pages = _page_table([s + c for s, c in spans], gen)
    k, k_scales = _codes(pages, kv, dim, gen)
    v, v_scales = _codes(pages, kv, dim, gen)
    qkv = torch.randn((n, (heads + 2 * kv) * dim), generator=gen, device="cuda").to(dtype)
    reach = max(s + c for s, c in spans)
    freq = 10000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device="cuda") / dim)
    angle = torch.arange(reach, dtype=torch.float64, device="cuda")[:, None] * freq
    held = [-(-(s + c) // PAGE) for s, c in spans]
    # where the read pages go: one sequence's behind another's
    local = torch.full_like(table, -1)
    at = 0
    for i, c in enumerate(held):
        local[i, :c] = torch.arange(at, at + c, dtype=torch.int32, device="cuda")
        at += c
    shape = (at, kv, PAGE, dim)
    return {"qkv": qkv, "table": table, "local": local, "k": k, "v": v, "k_scales": k_scales, "v_scales": v_scales,
            "pos": torch.cat([torch.arange(s, s + c, dtype=torch.int32, device="cuda") for s, c in spans]),
            "seq": torch.cat([torch.full((c,), i, dtype=torch.int32, device="cuda") for i, (_, c) in enumerate(spans)]),
            "cos": torch.cos(angle).float(), "sin": torch.sin(angle).float(),
            "q": torch.empty((n, heads * dim), dtype=dtype, device="cuda"),
            "k_read": torch.empty(shape, dtype=dtype, device="cuda"), "v_read": torch.empty(shape, dtype=dtype, device="cuda")}


def _prepare_attend(case, gen):
    dtype, heads, kv, dim, tokens = _DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    lengths = _lengths(case)
    table, pages = _page_table(lengths, gen)
    k, k_scales = _codes(pages, kv, dim, gen)
    v, v_scales = _codes(pages, kv, dim, gen)
    rows = len(lengths) * tokens
    q = (1.5 * torch.randn((rows, heads * dim), generator=gen, device="cuda")).to(dtype)
    return {"q": q, "table": table, "k": k, "v": v, "k_scales": k_scales, "v_scales": v_scales,
            "pos": torch.tensor([n - tokens + j for n in lengths for j in range(tokens)], dtype=torch.int32, device="cuda"),
            "seq": torch.arange(len(lengths), dtype=torch.int32, device="cuda").repeat_interleave(tokens),
            "out": torch.empty_like(q), "scale": 1.0 / math.sqrt(dim)}


def _prepare_product(case, gen):
    dtype, m, n, k = _DTYPES[case["dtype"]], case["m"], case["n"], case["k"]
    rows = n * (2 if case["gated"] else 1)
    # activations behind a norm: every token has a size of its own
    x = torch.randn((m, k), generator=gen, device="cuda") * (0.5 + torch.rand((m, 1), generator=gen, device="cuda"))
    w = torch.randn((rows, k), generator=gen, device="cuda") / math.sqrt(k)
    top = w.abs().amax(1)
    # a row of codes takes a multiple of 16 bytes; the rest of it is zero
    codes = torch.zeros((rows, -(-k // 16) * 16), dtype=torch.int8, device="cuda")
    codes[:, :k] = torch.round(w * (127.0 / top)[:, None]).to(torch.int8)
    return {"x": x.to(dtype), "w": codes, "w_scales": top / 127.0, "out": torch.empty((m, n), dtype=dtype, device="cuda")}


# ---- one pass -----------------------------------------------------------------------------------
def run(state):
    return {"cache": _run_cache, "attend": _run_attend, "product": _run_product}[state["case"]["op"]](state)


def _rows_to_codes(x):
    """float32 rows -> (codes as float32, scales)."""
    top = x.abs().amax(-1, keepdim=True)
    most = torch.full_like(top, 127.0)  # (a quotient of two tensors is rounded once; by a number it is a product with a reciprocal)
    return torch.round(x * (most / top)), top / most


def _run_cache(s):
    case = s["case"]
    heads, kv, dim, n = case["heads"], case["kv_heads"], case["dim"], s["qkv"].shape[0]
    if own:
        from nnis_b200.csrc import ops
        ops.rope_store_int8(s["qkv"], s["q"], s["pos"], s["seq"], s["table"], s["cos"], s["sin"], s["k"], s["v"],
                            s["k_scales"], s["v_scales"], heads, kv, dim, PAGE)
        ops.read_pages_int8(s["k"], s["v"], s["k_scales"], s["v_scales"], s["table"], s["local"], s["k_read"], s["v_read"])
        return s["q"], s["k_read"], s["v_read"]
    dtype = s["qkv"].dtype
    x = s["qkv"].float().view(n, heads + 2 * kv, dim)
    pos = s["pos"].long()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    a, b = x[:, :heads + kv, :dim // 2], x[:, :heads + kv, dim // 2:]
    turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1).to(dtype)
    k_codes, k_scales = _rows_to_codes(turned[:, heads:].float())
    v_codes, v_scales = _rows_to_codes(x[:, heads + kv:])
    pages, slots = s["table"][s["seq"].long(), pos // PAGE].long(), pos % PAGE
    s["k"][pages, :, slots] = k_codes.to(torch.int8)
    s["v"][pages, :, slots] = v_codes.to(torch.int8)
    s["k_scales"][pages, :, slots] = k_scales[..., 0]
    s["v_scales"][pages, :, slots] = v_scales[..., 0]
    q = turned[:, :heads].reshape(n, heads * dim)
    held = s["table"][s["local"] >= 0].long()
    return (q, (s["k"][held].float() * s["k_scales"][held][..., None]).to(dtype),
            (s["v"][held].float() * s["v_scales"][held][..., None]).to(dtype))


def _run_attend(s):
    case = s["case"]
    heads, kv, dim, tokens, window = case["heads"], case["kv_heads"], case["dim"], case["tokens"], case["window"]
    if own:
        from nnis_b200.csrc import ops
        ops.attention_int8(s["q"], s["q"].shape[1], s["k"], s["v"], s["k_scales"], s["v_scales"], s["pos"], s["seq"], s["table"],
                           s["out"], heads, kv, dim, window, s["scale"], s["workspace"])
        return s["out"]
    count, per = s["table"].shape[0], heads // kv
    table = s["table"].long().clamp_min(0)

    def rows_of(codes, scales):                                                # [sequences, kv, keys, dim]
        return (codes[table].float() * scales[table][..., None]).permute(0, 2, 1, 3, 4).reshape(count, kv, -1, dim)

    q = s["q"].float().view(count, tokens, kv, per, dim).transpose(1, 2).reshape(count, kv, tokens * per, dim) * s["scale"]
    scores = torch.matmul(q, rows_of(s["k"], s["k_scales"]).transpose(2, 3)).view(count, kv, tokens, per, -1)
    key, pos = torch.arange(scores.shape[-1], device=q.device), s["pos"].view(count, tokens, 1).long()
    hidden = key > pos
    if window:
        hidden = hidden | (key <= pos - window)
    scores = scores.masked_fill(hidden[:, None, :, None], -math.inf)
    weights = torch.exp(scores - scores.amax(-1, keepdim=True))
    weights = (weights / weights.sum(-1, keepdim=True)).view(count, kv, tokens * per, -1)
    out = torch.matmul(weights, rows_of(s["v"], s["v_scales"])).view(count, kv, tokens, per, dim)
    return out.transpose(1, 2).reshape(count * tokens, heads * dim).to(s["q"].dtype)


def _run_product(s):
    case = s["case"]
    if own:
        from nnis_b200.csrc import ops
        ops.linear_int8(s["x"], s["w"], s["w_scales"], None, s["out"], ops.GEMM_GATED if case["gated"] else ops.STORE, s["workspace"])
        return s["out"]
    codes, scales = _rows_to_codes(s["x"].float())
    # (64 bits: a sum of many products of codes passes 24 bits)
    sums = torch.matmul(codes.double(), s["w"][:, :case["k"]].double().T)
    y = sums.float() * scales * s["w_scales"]
    if case["gated"]:
        gate, up = y[:, :case["n"]], y[:, case["n"]:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    return y.to(s["x"].dtype)


# ---- the same from the definitions, in 64 bits -----------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    return {"cache": _exact_cache, "attend": _exact_attend, "product": _exact_product}[case["op"]](state)


def _exact_cache(s):
    """Sequence by sequence; keys are rounded to their type after the rotation, as a cache of that type holds them."""
    case, dtype = s["case"], s["qkv"].dtype
    heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
    qs, ks, vs, row = [], [], [], 0
    for i, (start, count) in enumerate(_spans(case)):
        x = s["qkv"][row:row + count].double().view(count, -1, d)
        row += count
        z = torch.complex(x[:, :heads + kv, :d // 2], x[:, :heads + kv, d // 2:])
        z = z * torch.complex(s["cos"].double(), s["sin"].double())[start:start + count, None]
        turned = torch.cat((z.real, z.imag), 2)
        qs.append(turned[:, :heads].reshape(count, heads * d))
        pages = s["table"][i][s["local"][i] >= 0].long()
        for new, codes, scales, out in ((turned[:, heads:].to(dtype).double(), s["k"], s["k_scales"], ks),
                                        (x[:, heads + kv:], s["v"], s["v_scales"], vs)):
            flat = (codes[pages].double() * scales[pages].double()[..., None]).transpose(0, 1).reshape(kv, -1, d)
            step = new.abs().amax(2, keepdim=True) / 127
            flat[:, start:start + count] = (torch.round(new / step) * step).transpose(0, 1)
            out.append(flat.view(kv, -1, PAGE, d).transpose(0, 1))
    return torch.cat(qs), torch.cat(ks), torch.cat(vs)


def _exact_attend(s):
    """Row by row over the row's own list of pages."""
    case = s["case"]
    heads, kv, d, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    out = torch.empty((s["q"].shape[0], kv, heads // kv, d), dtype=torch.float64, device=s["q"].device)
    tables, seqs, positions = s["table"].tolist(), s["seq"].tolist(), s["pos"].tolist()
    for r, (i, pos) in enumerate(zip(seqs, positions)):
        pages = torch.tensor(tables[i][:pos // PAGE + 1], device=s["q"].device)
        first = max(0, pos - window + 1) if window else 0
        keys, values = ((c[pages].double() * f[pages].double()[..., None]).transpose(0, 1).reshape(kv, -1, d)[:, first:pos + 1]
                        for c, f in ((s["k"], s["k_scales"]), (s["v"], s["v_scales"])))
        q = s["q"][r].double().view(kv, heads // kv, d)
        out[r] = torch.softmax(torch.einsum("hgd,hnd->hgn", q, keys) * s["scale"], dim=2) @ values
    return out.reshape(s["q"].shape[0], heads * d)


def _exact_product(s):
    case = s["case"]
    x = s["x"].double()
    step = x.abs().amax(1, keepdim=True) / 127
    y = torch.einsum("mk,nk->mn", torch.round(x / step), s["w"][:, :case["k"]].double()) * step * s["w_scales"].double()
    if not case["gated"]:
        return y
    gate, up = y.split(case["n"], dim=1)
    return gate * torch.sigmoid(gate) * up
