"""Measured cases of the rotary and chunk operators: rotary_embedding, fill_kv_pages_rotary and paged_attention_chunk.

``listed()`` names the cases, ``draw(rng)`` makes more of the same ranges, ``prepare`` builds the tensors that a serving
program holds before the call, and ``run`` is one call: in elementary torch operations where ``own`` is false, through the
package where it is true.  ``exact`` gives the outputs in 64 bits from the operators' definitions.

The three follow one another in a serving step: the projections of the new tokens leave as one [T, (Hq + 2 Hkv) D] matrix
whose column ranges are the queries, keys and values (so all three are strided views); fill_kv_pages_rotary rotates the
queries and keys by the tokens' positions and appends keys and values to the page pools; paged_attention_chunk lets the
rotated queries attend to the pools.  rotary_embedding is the rotation alone, as an image encoder or a dense cache wants it.
"""

import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------------------------------
# A case holds plain values only, so lists of whole numbers (token counts, lengths, sections) are texts: "16,24,24".
def _text(numbers):
    return ",".join(str(n) for n in numbers)


def _ints(text):
    return [int(n) for n in text.split(",")] if text else []


def _rotary(name, tokens, heads, head_dim, dtype, rotary_dim=None, sections=(), order="blocked", pairing="half", theta=5e5,
            magnitude=1.0, first=0):
    return {"name": name, "op": "rotary", "tokens": tokens, "heads": heads, "head_dim": head_dim, "dtype": dtype,
            "rotary_dim": rotary_dim or head_dim, "sections": _text(sections), "order": order, "pairing": pairing, "theta": theta,
            "magnitude": magnitude, "first": first}


def _append(name, new, history, hq, hkv, head_dim, tpp, dtype, slots=False, queries=True, rotary_dim=None, sections=(),
            order="blocked", pairing="half", theta=5e5, magnitude=1.0):
    return {"name": name, "op": "append", "new": _text(new), "history": _text(history), "hq": hq, "hkv": hkv, "head_dim": head_dim,
            "tpp": tpp, "dtype": dtype, "slots": slots, "queries": queries, "rotary_dim": rotary_dim or head_dim,
            "sections": _text(sections), "order": order, "pairing": pairing, "theta": theta, "magnitude": magnitude}


def _chunk(name, new, history, hq, hkv, head_dim, tpp, dtype, causal=True, window=0):
    return {"name": name, "op": "chunk", "new": _text(new), "history": _text(history), "hq": hq, "hkv": hkv, "head_dim": head_dim,
            "tpp": tpp, "dtype": dtype, "causal": causal, "window": window}


def _spread(count, lo, hi, step):
    """``count`` fixed lengths spread over [lo, hi], none of them in order."""
    return [lo + (i * step) % (hi - lo + 1) for i in range(count)]


def listed():
    return [
        # the queries of one step of a small batch, deep in their contexts; half of each head is rotated, adjacent pairs
        _rotary("rotary_step", 16, 32, 128, "fp16", rotary_dim=64, pairing="adjacent", first=120000),
        # patches of one large image in an encoder: two axes (row, column), heads of 80, an odd number of patches
        _rotary("rotary_image", 5329, 16, 80, "bf16", sections=(20, 20), theta=1e4),
        # the queries of a long video prompt: three axes (time, row, column)
        _rotary("rotary_video", 32768, 32, 128, "bf16", sections=(16, 24, 24), theta=1e6),
        # one decode step of 64 sequences: a token each, at the end of contexts of 200 to 8000 tokens
        _append("append_step", [1] * 64, _spread(64, 200, 8000, 2711), 32, 8, 128, 16, "bf16"),
        # a ragged batch of prompts that start anywhere in a page, flat slot ids, three interleaved axes, heads of 64
        _append("append_ragged", [1, 700, 33, 1, 259, 1023, 5, 410], [77, 0, 1001, 3333, 18, 511, 4090, 129], 24, 8, 64, 32, "fp16",
                slots=True, sections=(12, 10, 10), order="interleaved", theta=1e6),
        # chunked prefill of eight prompts: 2048 tokens each on top of 0 to 4096
        _append("append_prefill", [2048] * 8, _spread(8, 0, 4096, 1499), 32, 8, 128, 16, "bf16", magnitude=1.2079),
        # one sequence whose five proposed tokens are verified: the smallest call
        _chunk("chunk_verify_one", [5], [1000], 32, 8, 128, 16, "bf16"),
        # 64 sequences with four proposed tokens each: every page of the batch is read for a few rows
        _chunk("chunk_verify_batch", [4] * 64, _spread(64, 1024, 4096, 1237), 32, 8, 128, 16, "bf16"),
        # decode steps and three prompt chunks in one call, 16 heads of 64 on as many kv heads, fp16
        _chunk("chunk_mixed", [1] * 45 + [777, 1500, 300], _spread(48, 64, 6000, 1663), 16, 16, 64, 32, "fp16"),
        # sliding window of 1000 tokens, seven query heads per kv head
        _chunk("chunk_window", [1537, 1537, 1537, 1537], [0, 500, 2999, 8191], 28, 4, 128, 32, "bf16", window=1000),
        # chunked prefill of eight prompts: 2048 tokens each on top of 0 to 4096
        _chunk("chunk_prefill", [2048] * 8, _spread(8, 0, 4096, 1499), 32, 8, 128, 16, "bf16"),
        # the next 512 tokens of a prompt of 128 Ki tokens, 64 query heads
        _chunk("chunk_long", [512], [130560], 64, 8, 128, 16, "bf16"),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_rotation(rng, head_dim):
    rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2])
    half = rotary_dim // 2
    kind = rng.choice(["text", "text", "blocked", "interleaved"])
    if kind == "text":
        sections, order = [], "blocked"
    else:
        order = kind
        sections = [half // 2, half - half // 2] if kind == "blocked" and rng.random() < 0.4 else [half - 2 * (half // 3), half // 3, half // 3]
    return {"rotary_dim": rotary_dim, "sections": _text(sections), "order": order, "pairing": rng.choice(["half", "half", "adjacent"]),
            "theta": rng.choice([1e4, 5e5, 1e6]), "magnitude": rng.choice([1.0, 1.0, 1.2079])}


def _draw_batch(rng, max_seqs, budget):
    """New-token counts and history lengths: steps, verification, prompt chunks, or a mix."""
    kind = rng.choice(["step", "verify", "prompt", "mixed"])
    seqs = _log_int(rng, 1, max_seqs)
    if kind == "step":
        new = [1] * seqs
    elif kind == "verify":
        new = [rng.randint(2, 16) for _ in range(seqs)]
    elif kind == "prompt":
        seqs = min(seqs, 12)
        new = [_log_int(rng, 17, 2048) for _ in range(seqs)]
    else:
        new = [1 if rng.random() < 0.8 else _log_int(rng, 2, 1500) for _ in range(seqs)]
    history = [0 if rng.random() < 0.1 else _log_int(rng, 16, 8000) for _ in range(seqs)]
    while sum(history) + sum(new) > budget:
        history = [h // 2 for h in history]
        new = [max(1, n // 2) for n in new]
    return new, history


def draw(rng):
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    op = rng.choice(["rotary", "append", "chunk", "chunk"])
    if op == "rotary":
        head_dim = rng.choice([64, 80, 96, 128, 128, 256])
        heads = rng.choice([1, 8, 16, 24, 32, 40])
        tokens = _log_int(rng, 1, 32768 * 32 * 128 // (heads * head_dim))
        case = {"op": "rotary", "tokens": min(tokens, 100000), "heads": heads, "head_dim": head_dim, "dtype": dtype,
                "first": rng.choice([0, 5000, 900000])}
        case.update(_draw_rotation(rng, head_dim))
        return case
    hq, hkv = rng.choice([(32, 8), (32, 8), (64, 8), (16, 16), (28, 4), (8, 1), (40, 8), (12, 4)])
    tpp = rng.choice([16, 16, 32])
    if op == "append":
        head_dim = rng.choice([64, 96, 128, 128, 256])
        new, history = _draw_batch(rng, 256, 16384 * 128 * 40 // (head_dim * (hq + hkv)) + 256)
        case = {"op": "append", "new": _text(new), "history": _text(history), "hq": hq, "hkv": hkv, "head_dim": head_dim, "tpp": tpp, "dtype": dtype,
                "slots": rng.random() < 0.4, "queries": rng.random() < 0.8}
        case.update(_draw_rotation(rng, head_dim))
        return case
    head_dim = rng.choice([64, 80, 128, 128, 128, 256])
    new, history = _draw_batch(rng, 128, 120000 * 8 * 128 // (hkv * head_dim * 2))
    causal = rng.random() < 0.85
    window = _log_int(rng, 32, 4096) if causal and rng.random() < 0.25 else 0
    return {"op": "chunk", "new": _text(new), "history": _text(history), "hq": hq, "hkv": hkv, "head_dim": head_dim, "tpp": tpp, "dtype": dtype,
            "causal": causal, "window": window}


# ---------------------------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------------------------
def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _normal(g, shape, dtype, spread=1.0):
    return (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32) * spread).to(dtype)


def _pages(case, g):
    """Page table over the whole lengths, pages in random order, and the pool's page count (a tenth more than used)."""
    tpp = case["tpp"]
    lens = [n + h for n, h in zip(_ints(case["new"]), _ints(case["history"]))]
    counts = [(length + tpp - 1) // tpp for length in lens]
    used = sum(counts)
    total = used + used // 10 + 1
    perm = torch.randperm(total, generator=g, device="cuda")[:used].to(torch.int32)
    table = torch.zeros((len(lens), max(counts)), dtype=torch.int32, device="cuda")
    at = 0
    for s, c in enumerate(counts):
        table[s, :c] = perm[at:at + c]
        at += c
    return table, total, lens


def _inv_freq(case):
    half = case["rotary_dim"] // 2
    return (case["theta"] ** (-torch.arange(half, dtype=torch.float64) / half)).float().cuda()


def _axis_positions(case, base):
    """Text positions, or with several axes the (frame, row, column) of a token in frames of 24 x 32 patches; two axes are
    the row and column in an image 73 patches wide."""
    axes = len(_ints(case["sections"]))
    if axes <= 1:
        return base
    if axes == 2:
        return torch.stack([base // 73, base % 73])
    return torch.stack([base // 768, base % 768 // 32, base % 32])


def _axis_of_frequency(case):
    half, sections = case["rotary_dim"] // 2, _ints(case["sections"])
    if len(sections) <= 1:
        return [0] * half
    if case["order"] == "blocked":
        return [a for a, n in enumerate(sections) for _ in range(n)]
    axes = len(sections)
    return [i % axes if i // axes < sections[i % axes] else 0 for i in range(half)]


def prepare(case, seed):
    g = _generator(seed)
    dtype = DTYPES[case["dtype"]]
    d = case["head_dim"]
    if case["op"] == "rotary":
        tokens, heads = case["tokens"], case["heads"]
        # queries are the leading columns of a projection that also holds a quarter as many keys' worth of columns
        width = heads + max(1, heads // 4)
        x = _normal(g, (tokens, width, d), dtype)[:, :heads]
        shift = int(torch.randint(0, 64, (1,), generator=g, device="cuda").item())
        base = torch.arange(tokens, device="cuda") + case["first"] + shift
        return {"case": case, "x": x, "positions": _axis_positions(case, base).to(torch.int32), "inv_freq": _inv_freq(case),
                "axis": torch.tensor(_axis_of_frequency(case), device="cuda")}
    hq, hkv, tpp = case["hq"], case["hkv"], case["tpp"]
    table, total, lens = _pages(case, g)
    state = {"case": case, "page_table": table, "total_pages": total}
    new = torch.tensor(_ints(case["new"]), dtype=torch.int64, device="cuda")
    hist = torch.tensor(_ints(case["history"]), dtype=torch.int64, device="cuda")
    tokens = sum(_ints(case["new"]))
    # keys of a layer have channels of very different size; values and queries are near normal
    channel = torch.exp(torch.randn((1, 1, hkv, d), generator=g, device="cuda") * 0.3)
    k_tok = _normal(g, (total, tpp, hkv, d), torch.float32).mul_(channel).to(dtype)
    state["k_pool"] = k_tok.view(total, tpp, hkv, d // 8, 8).permute(0, 2, 3, 1, 4).contiguous()
    del k_tok
    state["v_pool"] = _normal(g, (total, hkv, d, tpp), dtype)
    if case["op"] == "append":
        first = torch.cumsum(new, 0) - new
        seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), new)
        position = torch.arange(tokens, device="cuda") - first[seq] + hist[seq]
        qkv = _normal(g, (tokens, hq + 2 * hkv, d), dtype)
        state.update(q=qkv[:, :hq], k=qkv[:, hq:hq + hkv], v=qkv[:, hq + hkv:], inv_freq=_inv_freq(case),
                     positions=_axis_positions(case, position).to(torch.int32), write_positions=position.to(torch.int32),
                     seq_map=seq.to(torch.int32), axis=torch.tensor(_axis_of_frequency(case), device="cuda"))
        state["slots"] = table[seq, position // tpp].to(torch.int64) * tpp + position % tpp
        return state
    state["q"] = _normal(g, (tokens, hq, d), dtype, 1.5)
    state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    state["cu"] = torch.tensor([0] + torch.tensor(_ints(case["new"])).cumsum(0).tolist(), dtype=torch.int32, device="cuda")
    return state


# ---------------------------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------------------------
def _plain_rotate(x, state):
    """x [T, H, D] rotated, in 32 bits (the angles in 64), not yet rounded."""
    case = state["case"]
    half = case["rotary_dim"] // 2
    pos = state["positions"] if state["positions"].dim() == 2 else state["positions"][None]
    per_freq = pos[state["axis"]].t()  # [T, half]
    angle = per_freq.double() * state["inv_freq"].double()
    cos = (torch.cos(angle) * case["magnitude"]).float()[:, None]
    sin = (torch.sin(angle) * case["magnitude"]).float()[:, None]
    xf = x.float()
    if case["pairing"] == "half":
        a, b = xf[..., :half], xf[..., half:2 * half]
        parts = [a * cos - b * sin, b * cos + a * sin]
    else:
        a, b = xf[..., 0:2 * half:2], xf[..., 1:2 * half:2]
        parts = [torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)]
    return torch.cat(parts + [xf[..., 2 * half:]], dim=-1)


def _plain_chunk(state):
    case = state["case"]
    hq, hkv, d, tpp = case["hq"], case["hkv"], case["head_dim"], case["tpp"]
    group = hq // hkv
    out = torch.empty((sum(_ints(case["new"])), hq, d), dtype=state["q"].dtype, device="cuda")
    row = 0
    for s, (n, h) in enumerate(zip(_ints(case["new"]), _ints(case["history"]))):
        length = n + h
        pages = state["page_table"][s, :(length + tpp - 1) // tpp].long()
        keys = state["k_pool"][pages].permute(1, 2, 4, 0, 3).reshape(hkv, d, -1)[..., :length].float()      # [Hkv, D, L]
        values = state["v_pool"][pages].permute(1, 0, 3, 2).reshape(hkv, -1, d)[:, :length].float()         # [Hkv, L, D]
        step = max(1, (1 << 29) // (hq * length))  # rows of queries at a time: at most 2 GiB of scores
        for r0 in range(0, n, step):
            r1 = min(n, r0 + step)
            q = state["q"][row + r0:row + r1].float().view(r1 - r0, hkv, group, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
            scores = torch.matmul(q, keys).mul_(1.0 / math.sqrt(d)).view(hkv, group, r1 - r0, length)
            if case["causal"]:
                at = torch.arange(h + r0, h + r1, device="cuda")[:, None]
                key = torch.arange(length, device="cuda")[None]
                hidden = key > at
                if case["window"]:
                    hidden = hidden | (key <= at - case["window"])
                scores.masked_fill_(hidden, float("-inf"))
            scores -= scores.amax(-1, keepdim=True)
            weights = scores.exp_()
            total = weights.sum(-1, keepdim=True)
            mixed = torch.matmul(weights.view(hkv, -1, length), values).view(hkv, group, r1 - r0, d) / total
            out[row + r0:row + r1] = mixed.permute(2, 0, 1, 3).reshape(r1 - r0, hq, d).to(out.dtype)
        row += n
    return out


def _plain(state):
    case = state["case"]
    if case["op"] == "rotary":
        return _plain_rotate(state["x"], state).to(state["x"].dtype)
    if case["op"] == "chunk":
        return _plain_chunk(state)
    k_pool, v_pool, tpp, d = state["k_pool"], state["v_pool"], case["tpp"], case["head_dim"]
    if case["slots"]:
        page, slot = state["slots"] // tpp, state["slots"] % tpp
    else:
        at = state["write_positions"].long()
        page, slot = state["page_table"][state["seq_map"].long(), at // tpp].long(), at % tpp
    keys = _plain_rotate(state["k"], state).to(k_pool.dtype)
    k_pool[page, :, :, slot] = keys.reshape(keys.shape[0], case["hkv"], d // 8, 8)
    v_pool[page, :, :, slot] = state["v"]
    if not case["queries"]:
        return [k_pool, v_pool]
    return [k_pool, v_pool, _plain_rotate(state["q"], state).to(state["q"].dtype)]


def run(state):
    if not own:
        return _plain(state)
    import proxy_attention_lab_b200 as pal

    case = state["case"]
    if case["op"] == "chunk":
        return pal.paged_attention_chunk(state["q"], state["k_pool"], state["v_pool"], state["page_table"], state["lens"], state["cu"],
                                         causal=case["causal"], window=case["window"] or None)
    rotation = dict(sections=_ints(case["sections"]) or None, section_order=case["order"], pairing=case["pairing"], magnitude=case["magnitude"])
    if case["op"] == "rotary":
        return pal.rotary_embedding(state["x"], state["positions"], state["inv_freq"], **rotation)
    where = dict(slot_mapping=state["slots"]) if case["slots"] else dict(
        page_table=state["page_table"], current_token_write_positions=state["write_positions"], query_to_seq_map=state["seq_map"])
    return list(pal.fill_kv_pages_rotary(state["k"], state["v"], state["k_pool"], state["v_pool"], inv_freq=state["inv_freq"],
                                         positions=state["positions"], queries=state["q"] if case["queries"] else None, **where, **rotation))


# ---------------------------------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------------------------------
def work(case):
    d = case["head_dim"]
    if case["op"] == "rotary":
        t, h, axes = case["tokens"], case["heads"], max(1, len(_ints(case["sections"])))
        return {"bytes": 4 * t * h * d + 4 * t * axes + 2 * case["rotary_dim"], "flops": 3 * t * h * case["rotary_dim"]}
    hq, hkv = case["hq"], case["hkv"]
    t = sum(_ints(case["new"]))
    if case["op"] == "append":
        axes = max(1, len(_ints(case["sections"])))
        heads = 2 * hkv + (hq if case["queries"] else 0)
        turned = heads - hkv
        return {"bytes": 4 * t * heads * d + t * (4 * axes + (8 if case["slots"] else 8)), "flops": 3 * t * turned * case["rotary_dim"]}
    pairs = read = 0
    for n, h in zip(_ints(case["new"]), _ints(case["history"])):
        w = case["window"]
        if not case["causal"]:
            pairs += n * (n + h)
        elif w:
            pairs += sum(min(h + i + 1, w) for i in range(n))
        else:
            pairs += n * h + n * (n + 1) // 2
        read += min(n + h, n + w - 1) if w else n + h
    return {"bytes": 4 * read * hkv * d + 4 * t * hq * d + 4 * (read // case["tpp"] + 2 * len(_ints(case["new"]))), "flops": 4 * pairs * hq * d}


# ---------------------------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------------------------
def _exact_rotation(x, state):
    """Every pair (a, b) is the complex number a + ib, turned by position * frequency and stretched by the magnitude."""
    case = state["case"]
    r = case["rotary_dim"]
    x = x.double()
    pos = state["positions"].double().reshape(-1, x.shape[0])
    freq = state["inv_freq"].double()
    angle = torch.zeros((x.shape[0], r // 2), dtype=torch.float64, device=x.device)
    bounds = 0
    sections = _ints(case["sections"])
    count = len(sections)
    for a in range(pos.shape[0]):
        if count <= 1:
            mine = torch.arange(r // 2, device=x.device)
        elif case["order"] == "blocked":
            mine = torch.arange(bounds, bounds + sections[a], device=x.device)
            bounds += sections[a]
        else:
            index = torch.arange(r // 2, device=x.device)
            taken = [(index % count == b) & (index < count * sections[b]) for b in range(1, count)]
            mine = (taken[a - 1] if a else ~torch.stack(taken).any(0)).nonzero().flatten()
        angle[:, mine] = pos[a][:, None] * freq[mine]
    turn = torch.polar(torch.full_like(angle, case["magnitude"]), angle)[:, None]
    turned = x[..., :r]
    if case["pairing"] == "adjacent":
        z = torch.view_as_complex(turned.unflatten(-1, (r // 2, 2)).contiguous()) * turn
        y = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(turned[..., :r // 2].contiguous(), turned[..., r // 2:].contiguous()) * turn
        y = torch.cat([z.real, z.imag], -1)
    return torch.cat([y, x[..., r:]], -1)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotation(state["x"], state)
    d, tpp, hkv = case["head_dim"], case["tpp"], case["hkv"]
    if case["op"] == "append":
        slots = state["slots"]
        k_tok = state["k_pool"].double().permute(0, 3, 1, 2, 4).reshape(-1, hkv, d)   # one row per slot
        v_tok = state["v_pool"].double().permute(0, 3, 1, 2).reshape(-1, hkv, d)
        k_tok.index_copy_(0, slots, _exact_rotation(state["k"], state))
        v_tok.index_copy_(0, slots, state["v"].double())
        outs = [k_tok.view(-1, tpp, hkv, d // 8, 8).permute(0, 2, 3, 1, 4).contiguous(), v_tok.view(-1, tpp, hkv, d).permute(0, 2, 3, 1).contiguous()]
        return outs + ([_exact_rotation(state["q"], state)] if case["queries"] else [])
    hq, group = case["hq"], case["hq"] // hkv
    out = torch.empty((sum(_ints(case["new"])), hq, d), dtype=torch.float64, device="cuda")
    row = 0
    for s, (n, h) in enumerate(zip(_ints(case["new"]), _ints(case["history"]))):
        length = n + h
        token = torch.arange(length, device="cuda")
        page, slot = state["page_table"][s].long()[token // tpp], token % tpp
        lowest = (token[h:] - case["window"] + 1).clamp(min=0) if case["window"] else torch.zeros(n, dtype=torch.long, device="cuda")
        highest = token[h:] if case["causal"] else torch.full((n,), length - 1, device="cuda")
        for head in range(hkv):
            keys = state["k_pool"][page, head, :, slot].reshape(length, d).double()
            values = state["v_pool"][page, head, :, slot].double()
            for r0 in range(0, n, 1024):
                rows = slice(r0, min(n, r0 + 1024))
                q = state["q"][row + r0:row + rows.stop, head * group:(head + 1) * group].double()
                score = torch.einsum("ngd,ld->ngl", q, keys) / math.sqrt(d)
                seen = (token[None] >= lowest[rows, None]) & (token[None] <= highest[rows, None])
                score = torch.where(seen[:, None], score, -math.inf)
                weight = torch.exp(score - torch.logsumexp(score, -1, keepdim=True))
                out[row + r0:row + rows.stop, head * group:(head + 1) * group] = torch.einsum("ngl,ld->ngd", weight, values)
        row += n
    return out
