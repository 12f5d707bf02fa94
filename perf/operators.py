"""The operators of forked sequences and drafted tokens, as they are timed: calls that a program makes of
them, and the same computed with elementary torch operations.

* ``shared``  attention of a batch whose sequences begin with the same pages of the cache: the shared
              pages are read once for all rows (``ops.attention_shared`` with a plan that the program
              keeps while its sequences do);
* ``pages``   pages of keys and values copied inside the store for all layers in one call: the last,
              partly filled page of forked sequences, or whole pages that move (``ops.copy_pages``);
* ``verify``  drafted tokens accepted or rejected against the target's probabilities, and the next token
              picked, from given random numbers (``sampling.device.verify_drafts``).

Head layouts, layers and vocabulary are those of the SmolLM2 shapes (135M: 9 query and 3 key/value heads
of 64, 30 layers; 360M: 15 and 5; 1.7B: 32 and 32, 24 layers; 49,152 tokens) and heads of 128.
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
        # two samples of a short prompt, their first tokens: launches and latency
        _shared("shared_2x128", "bfloat16", 9, 3, 64, groups=1, members=2, alone=0, prefix=128, tail=16),
        # eight samples of one prompt at contexts ending at 4,096
        _shared("shared_8x4096", "bfloat16", 9, 3, 64, groups=1, members=8, alone=0, prefix=4032, tail=64),
        # a batch of 64 behind one long document, 360M heads
        _shared("shared_64x16384", "bfloat16", 15, 5, 64, groups=1, members=64, alone=0, prefix=16384, tail=256),
        # two prompts' samples beside three unrelated sequences, a key/value head per query head (1.7B)
        _shared("shared_two_prompts", "bfloat16", 32, 32, 64, groups=2, members=24, alone=3, prefix=4001, tail=300),
        # four drafted tokens and the one before them per sequence, wide heads
        _shared("shared_drafts_128", "bfloat16", 32, 8, 128, groups=1, members=16, alone=0, prefix=8190, tail=100, tokens=5),
        # true float32
        _shared("shared_float32", "float32", 9, 3, 64, groups=1, members=16, alone=0, prefix=2000, tail=48),
        # a session is forked once: its last page, 30 layers
        _pages("fork_session", "bfloat16", 30, 3, 64, pages=64, moves=1, sources=1, partial=True),
        # 63 forks of one sequence begin to write
        _pages("fork_63", "bfloat16", 30, 3, 64, pages=96, moves=63, sources=1, partial=True),
        # whole pages move together, 1.7B heads in float32
        _pages("compact_float32", "float32", 24, 32, 64, pages=64, moves=24, sources=24, partial=False),
        # one session with a drafting model, four tokens
        _verify("verify_session", 1, 4, 49152, temperature=0.8, model=True),
        # a server's batch with a drafting model
        _verify("verify_64x7", 64, 7, 49152, temperature=1.0, model=True),
        # drafts looked up in the text, none to ten a sequence, every third sequence greedy
        _verify("verify_lookup", 24, 10, 49152, temperature=0.7, model=False, ragged=True, greedy_every=3),
    ]


def _shared(name, dtype, heads, kv_heads, dim, groups, members, alone, prefix, tail, tokens=1):
    return {"name": name, "op": "shared", "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "groups": groups,
            "members": members, "alone": alone, "prefix": prefix, "tail": tail, "tokens": tokens}


def _pages(name, dtype, layers, kv_heads, dim, pages, moves, sources, partial):
    return {"name": name, "op": "pages", "dtype": dtype, "layers": layers, "kv_heads": kv_heads, "dim": dim, "pages": pages,
            "moves": moves, "sources": sources, "partial": partial}


def _verify(name, sequences, drafts, vocab, temperature, model, ragged=False, greedy_every=0):
    return {"name": name, "op": "verify", "sequences": sequences, "drafts": drafts, "vocab": vocab, "temperature": temperature,
            "model": model, "ragged": ragged, "greedy_every": greedy_every}


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def _draw_once(rng):
    op = rng.choice(("shared", "shared", "pages", "verify"))
    if op == "shared":
        heads, kv_heads, dim = rng.choice(((9, 3, 64), (15, 5, 64), (32, 32, 64), (32, 8, 128), (16, 2, 128), (20, 1, 64)))
        dtype = rng.choice(("bfloat16", "bfloat16", "bfloat16", "float32"))
        tokens = rng.choice((1, 1, 1, 2, 5))
        return _shared("", dtype, heads, kv_heads, dim, groups=rng.choice((1, 1, 1, 2, 3)), members=_log_int(rng, 2, 64),
                       alone=rng.choice((0, 0, 1, 4)), prefix=_log_int(rng, 64, 16384 if dtype == "bfloat16" else 4096),
                       tail=_log_int(rng, tokens + 1, 400), tokens=tokens)
    if op == "pages":
        layers, kv_heads = rng.choice(((30, 3), (32, 5), (24, 32), (1, 8)))
        moves = _log_int(rng, 1, 63)
        return _pages("", rng.choice(("bfloat16", "bfloat16", "float32")), layers, kv_heads, rng.choice((64, 64, 128)),
                      pages=2 * moves + rng.randrange(1, 8), moves=moves, sources=rng.choice((1, moves)),
                      partial=rng.choice((True, True, False)))
    return _verify("", _log_int(rng, 1, 64), rng.randrange(1, 9), rng.choice((49152, 32000, 49153, 100277)),
                   temperature=round(rng.uniform(0.5, 1.3), 3), model=rng.choice((True, True, False)),
                   ragged=rng.choice((True, False)), greedy_every=rng.choice((0, 0, 3)))


def draw(rng):
    most = {op: max((_cost(c) for c in listed() if c["op"] == op)) for op in ("shared", "pages", "verify")}
    while True:
        case = _draw_once(rng)
        del case["name"]
        if _cost(case) <= most[case["op"]]:
            return case


def _cost(case):
    w = work(case)
    # (float32 products cost some eight times the others)
    slow = 8.0 if case["op"] == "shared" and case["dtype"] == "float32" else 1.0
    return max(w["bytes"] / 6.4e12, slow * w["flops"] / 5e14)


# ---- sizes that follow from a case alone ----------------------------------------------------
def _lengths(case):
    """Positions that every sequence holds with its new tokens: groups first, then the ones alone."""
    least, tail = case["tokens"], case["tail"]
    count = case["groups"] * case["members"] + case["alone"]
    return [case["prefix"] + least + (i * 7919) % max(1, tail - least + 1) for i in range(count)]


def _shared_pages(case):
    return case["prefix"] // PAGE  # whole pages; the rest of the prefix is each sequence's own copy


def _rows_moved(case):
    return [1 + (i * 37 + 22) % (PAGE - 1) if case["partial"] else PAGE for i in range(case["moves"])]


def _counts(case):
    if not case["ragged"]:
        return [case["drafts"]] * case["sequences"]
    return [(i * 7 + 3) % (case["drafts"] + 1) for i in range(case["sequences"])]


def work(case):
    if case["op"] == "shared":
        size = 2 if case["dtype"] == "bfloat16" else 4
        lengths, tokens, shared = _lengths(case), case["tokens"], _shared_pages(case) * PAGE
        grouped = case["groups"] * case["members"]
        positions = case["groups"] * shared + sum(n - (shared if i < grouped else 0) for i, n in enumerate(lengths))
        rows = len(lengths) * tokens
        keys = sum(n - tokens + 1 + j for n in lengths for j in range(tokens))
        return {"bytes": size * (2 * positions * case["kv_heads"] * case["dim"] + 2 * rows * case["heads"] * case["dim"])
                + 8 * rows + 4 * sum(-(-n // PAGE) for n in lengths),
                "flops": 4 * case["heads"] * case["dim"] * keys}
    if case["op"] == "pages":
        size = 2 if case["dtype"] == "bfloat16" else 4
        rows = _rows_moved(case)
        per_row = 2 * case["layers"] * case["kv_heads"] * case["dim"] * size
        read = max(rows) if case["sources"] == 1 else sum(rows)
        return {"bytes": per_row * (read + sum(rows)) + 12 * len(rows), "flops": 0}
    counts = _counts(case)
    rows = sum(counts) + len(counts)
    values = case["vocab"] * (rows + (sum(counts) if case["model"] else 0))
    return {"bytes": 4 * values + 12 * rows + 24 * len(counts), "flops": 4 * values}


# ---- inputs -----------------------------------------------------------------------------------
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return {"shared": _prepare_shared, "pages": _prepare_pages, "verify": _prepare_verify}[case["op"]](case, gen)


def _prepare_shared(case, gen):
    dtype, heads, kv_heads, dim, tokens = _DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    lengths, shared, members = _lengths(case), _shared_pages(case), case["members"]
    grouped = case["groups"] * members
    used = case["groups"] * shared + sum(-(-n // PAGE) - (shared if i < grouped else 0) for i, n in enumerate(lengths))
    pages = used + 3
    ids = torch.randperm(pages, generator=gen, device="cuda").tolist()
    firsts = [[ids.pop() for _ in range(shared)] for _ in range(case["groups"])]
    tables = []
    for i, n in enumerate(lengths):
        begin = list(firsts[i // members]) if i < grouped else []
        tables.append(begin + [ids.pop() for _ in range(-(-n // PAGE) - len(begin))])
    cols = max(len(t) for t in tables)
    shape = (pages, kv_heads, PAGE, dim)
    k = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    v = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    rows = len(lengths) * tokens
    q = (1.5 * torch.randn((rows, heads * dim), generator=gen, device="cuda")).to(dtype)
    table = torch.tensor([t + [-1] * (cols - len(t)) for t in tables], dtype=torch.int32, device="cuda")
    seq = torch.arange(len(lengths), dtype=torch.int32, device="cuda").repeat_interleave(tokens)
    positions = [n - tokens + j for n in lengths for j in range(tokens)]
    state = {"case": case, "q": q, "k": k, "v": v, "table": table, "seq": seq, "cols": cols, "lengths": lengths,
             "pos": torch.tensor(positions, dtype=torch.int32, device="cuda"), "out": torch.empty_like(q),
             "scale": 1.0 / math.sqrt(dim),
             # (sequences, pages that all of them begin with) of every group
             "groups": [(list(range(g * members, (g + 1) * members)), shared) for g in range(case["groups"])]
             + [([i], 0) for i in range(grouped, len(lengths))]}
    if own:
        from nnis_b200.csrc import ops
        from nnis_b200.engine.workspace import Workspace
        state["plan"] = ops.attention_shared_plan(tables, [i for i in range(len(tables)) for _ in range(tokens)], positions,
                                                  heads, kv_heads, dim, dtype, torch.device("cuda"))
        state["workspace"] = Workspace(torch.device("cuda"))
    return state


def _prepare_pages(case, gen):
    shape = (case["layers"], case["pages"], case["kv_heads"], PAGE, case["dim"])
    dtype = _DTYPES[case["dtype"]]
    k = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    v = torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)
    ids = torch.randperm(case["pages"], generator=gen, device="cuda").tolist()
    sources, targets = ids[:case["sources"]], ids[case["sources"]:case["sources"] + case["moves"]]
    moves = [(sources[i % len(sources)], targets[i], r) for i, r in enumerate(_rows_moved(case))]
    return {"case": case, "k": k, "v": v, "moves": moves}


def _prepare_verify(case, gen):
    counts, vocab, t = _counts(case), case["vocab"], case["temperature"]
    b, drafted = len(counts), sum(counts)
    rows = drafted + b
    # spread as a trained model's: the likeliest token has about a fifth of the probability
    logits = 4.0 * torch.randn((rows, vocab), generator=gen, device="cuda")
    # a sequence's rows lie together, its drafts' logits too: row r of sequence s is draft row r - s
    first = [0]
    for c in counts:
        first.append(first[-1] + c + 1)
    of_draft = torch.tensor([first[s] + j for s, c in enumerate(counts) for j in range(c)], dtype=torch.long, device="cuda")
    draft_logits = None
    if case["model"]:
        noise = torch.randn((drafted, vocab), generator=gen, device="cuda")
        draft_logits = logits[of_draft] + 0.7 * noise
        uniform = torch.rand((drafted, vocab), generator=gen, device="cuda").clamp_(1e-12, 1.0 - 1e-7)
        drafts = torch.argmax(draft_logits / t - torch.log(-torch.log(uniform)), dim=1)
        del noise, uniform
    else:
        likely = torch.argmax(logits[of_draft], dim=1)
        other = torch.randint(0, vocab, (drafted,), generator=gen, device="cuda")
        drafts = torch.where(torch.rand(drafted, generator=gen, device="cuda") < 0.7, likely, other)
    every = case["greedy_every"]
    state = {"case": case, "logits": logits, "draft_logits": draft_logits, "drafts": drafts.to(torch.int32),
             "first": torch.tensor(first, dtype=torch.int32, device="cuda"),
             "temperatures": torch.tensor([0.0 if every and s % every == 0 else t for s in range(b)], dtype=torch.float32,
                                          device="cuda"),
             "accept_draws": torch.rand(drafted, generator=gen, device="cuda", dtype=torch.float64),
             "pick_draws": torch.rand(b, generator=gen, device="cuda", dtype=torch.float64),
             "accepted": torch.empty(b, dtype=torch.int32, device="cuda"),
             "picked": torch.empty(b, dtype=torch.int32, device="cuda"),
             "counts": torch.tensor(counts, dtype=torch.long, device="cuda"), "of_draft": of_draft}
    if own:
        from nnis_b200.engine.workspace import Workspace
        state["workspace"] = Workspace(torch.device("cuda"))
    return state


# ---- one pass -----------------------------------------------------------------------------------
def run(state):
    return {"shared": _run_shared, "pages": _run_pages, "verify": _run_verify}[state["case"]["op"]](state)


def _run_shared(s):
    case = s["case"]
    if own:
        from nnis_b200.csrc import ops
        ops.attention_shared(s["q"], s["q"].shape[1], s["k"], s["v"], s["pos"], s["table"], s["plan"], s["out"],
                             case["heads"], case["kv_heads"], case["dim"], s["scale"], s["workspace"])
        return s["out"]
    heads, kv, d, tokens = case["heads"], case["kv_heads"], case["dim"], case["tokens"]
    per = heads // kv
    outs = []
    for members, shared in s["groups"]:
        first, count = members[0] * tokens, len(members) * tokens
        q = s["q"][first:first + count].float().view(count, kv, per, d) * s["scale"]
        pos = s["pos"][first:first + count].long()
        table = s["table"][members[0]:members[0] + len(members)].long().clamp_min(0)
        own_pages = table[:, shared:].repeat_interleave(tokens, dim=0)                  # [rows, pages]
        k_own = s["k"][own_pages].float().permute(0, 2, 1, 3, 4).reshape(count, kv, -1, d)
        v_own = s["v"][own_pages].float().permute(0, 2, 1, 3, 4).reshape(count, kv, -1, d)
        at = shared * PAGE + torch.arange(k_own.shape[2], device=pos.device)
        own_scores = torch.matmul(q, k_own.transpose(2, 3))                              # [rows, kv, per, keys]
        own_scores = own_scores.masked_fill((at[None] > pos[:, None])[:, None, None], -math.inf)
        k_all = s["k"][table[0, :shared]].float().permute(1, 0, 2, 3).reshape(kv, -1, d)  # [kv, keys, d]
        v_all = s["v"][table[0, :shared]].float().permute(1, 0, 2, 3).reshape(kv, -1, d)
        stacked = q.permute(1, 0, 2, 3).reshape(kv, count * per, d)
        scores = torch.matmul(stacked, k_all.transpose(1, 2)).view(kv, count, per, -1).permute(1, 0, 2, 3)
        top = own_scores.amax(-1, keepdim=True)
        if shared:
            top = torch.maximum(top, scores.amax(-1, keepdim=True))
        own_weights, weights = torch.exp(own_scores - top), torch.exp(scores - top)
        total = own_weights.sum(-1, keepdim=True) + weights.sum(-1, keepdim=True)
        o = torch.matmul(own_weights, v_own)
        o = o + torch.matmul(weights.permute(1, 0, 2, 3).reshape(kv, count * per, -1), v_all) \
            .view(kv, count, per, d).permute(1, 0, 2, 3)
        outs.append((o / total).reshape(count, heads * d))
    return torch.cat(outs).to(s["q"].dtype)


def _run_pages(s):
    if own:
        from nnis_b200.csrc import ops
        ops.copy_pages(s["k"], s["v"], s["moves"])
        return s["k"], s["v"]
    for store in (s["k"], s["v"]):
        for src, dst, rows in s["moves"]:
            store[:, dst, :, :rows] = store[:, src, :, :rows]
    return s["k"], s["v"]


def _run_verify(s):
    if own:
        from nnis_b200.sampling import device
        device.verify_drafts(s["logits"], s["drafts"], s["first"], s["temperatures"], s["accept_draws"], s["pick_draws"],
                             s["accepted"], s["picked"], s["draft_logits"], s["workspace"])
        return s["accepted"], s["picked"]
    # (64 bits: a draw may fall next to a border between two tokens)
    counts, first, rows = s["counts"], s["first"].long(), s["logits"].shape[0]
    b = counts.numel()
    temps = s["temperatures"].double()
    greedy = temps == 0
    seq_of_row = torch.searchsorted(first, torch.arange(rows, device=counts.device), right=True) - 1
    inverse = torch.where(greedy, torch.ones_like(temps), 1.0 / temps)

    def probabilities(logits, seq):
        x = logits.double()
        e = torch.exp((x - x.amax(1, keepdim=True)) * inverse[seq][:, None])
        return e / e.sum(1, keepdim=True)

    p = probabilities(s["logits"], seq_of_row)
    best = torch.argmax(s["logits"], dim=1)
    drafts, of_draft = s["drafts"].long(), s["of_draft"]
    seq = seq_of_row[of_draft]
    p_draft = p[of_draft].gather(1, drafts[:, None])[:, 0]
    q = probabilities(s["draft_logits"], seq) if s["draft_logits"] is not None else None
    q_draft = q.gather(1, drafts[:, None])[:, 0] if q is not None else torch.ones_like(p_draft)
    takes = torch.where(greedy[seq], drafts == best[of_draft], s["accept_draws"] * q_draft < p_draft)
    place = of_draft - first[seq]
    refused = torch.where(takes, counts[seq], place)
    accepted = counts.clone().scatter_reduce_(0, seq, refused, "amin")
    at = first[:-1] + accepted
    weights = p[at]
    corrects = accepted < counts
    draft_row = (at - torch.arange(b, device=at.device)).clamp_max(max(drafts.numel() - 1, 0))
    if drafts.numel():
        if q is not None:
            left = (weights - q[draft_row]).clamp_min(0)
        else:
            left = weights.scatter(1, drafts[draft_row][:, None], 0.0)
        left = torch.where((left.sum(1) > 0)[:, None], left, weights)
        weights = torch.where(corrects[:, None], left, weights)
    running = torch.cumsum(weights, 1)
    drawn = torch.searchsorted(running, (s["pick_draws"] * running[:, -1])[:, None], right=True)[:, 0]
    last = weights.shape[1] - 1 - torch.argmax((weights.flip(1) > 0).to(torch.int8), dim=1)
    picked = torch.where(greedy, best[at], torch.minimum(drawn, last))
    return accepted.to(torch.int32), picked.to(torch.int32)


# ---- the same from the definitions, in 64 bits -----------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "shared":
        return _exact_shared(state)
    if case["op"] == "pages":
        k, v = state["k"].clone(), state["v"].clone()
        for src, dst, rows in state["moves"]:
            for new, old in ((k, state["k"]), (v, state["v"])):
                new[:, dst, :, :rows].copy_(old[:, src, :, :rows])
        return k, v
    return _exact_verify(state)


def _exact_shared(s):
    """Row by row over the row's own list of pages."""
    case = s["case"]
    heads, kv, d = case["heads"], case["kv_heads"], case["dim"]
    out = torch.empty((s["q"].shape[0], heads, d), dtype=torch.float64, device=s["q"].device)
    tables, seqs, positions = s["table"].tolist(), s["seq"].tolist(), s["pos"].tolist()
    for r, (i, pos) in enumerate(zip(seqs, positions)):
        pages = torch.tensor(tables[i][:pos // PAGE + 1], device=s["q"].device)
        for h in range(kv):
            keys = s["k"][pages, h].double().reshape(-1, d)[:pos + 1]
            values = s["v"][pages, h].double().reshape(-1, d)[:pos + 1]
            q = s["q"][r].double().view(kv, heads // kv, d)[h]
            out[r, h * (heads // kv):(h + 1) * (heads // kv)] = torch.softmax(q @ keys.T * s["scale"], dim=1) @ values
    return out.reshape(s["q"].shape[0], heads * d)


def _exact_verify(s):
    """Sequence by sequence, draft by draft."""
    first, temps = s["first"].tolist(), s["temperatures"].tolist()
    drafts, accept, picks = s["drafts"].tolist(), s["accept_draws"].tolist(), s["pick_draws"].tolist()
    accepted, picked = [], []
    for b, t in enumerate(temps):
        count, row0 = first[b + 1] - first[b] - 1, first[b]
        a, left = 0, None
        while True:
            z = s["logits"][row0 + a].double()
            if t == 0:
                best = int(torch.nonzero(z == z.max())[0])
                if a < count and drafts[row0 - b + a] == best:
                    a += 1
                    continue
                accepted.append(a)
                picked.append(best)
                break
            p = torch.softmax(z / t, dim=0)
            if a == count:
                left = p
            else:
                d = drafts[row0 - b + a]
                if s["draft_logits"] is not None:
                    q = torch.softmax(s["draft_logits"][row0 - b + a].double() / t, dim=0)
                else:
                    q = torch.zeros_like(p)
                    q[d] = 1.0
                if accept[row0 - b + a] * float(q[d]) < float(p[d]):
                    a += 1
                    continue
                left = torch.clamp(p - q, min=0.0)
                if float(left.sum()) <= 0:
                    left = p
            running = torch.cumsum(left, 0)
            over = torch.nonzero(running > picks[b] * float(running[-1]))
            accepted.append(a)
            picked.append(int(over[0]) if over.numel() else int(torch.nonzero(left)[-1]))
            break
    make = lambda x: torch.tensor(x, dtype=torch.int32, device=s["logits"].device)
    return make(accepted), make(picked)
