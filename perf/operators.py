"""Cases, plain forms and calls of the decode-step operators around a shared prompt.

Three operators, in the order a step runs them:

* ``qkv_norm_post``: per-head RMS norms of q and k, rotation and the append to the paged cache;
* ``shared_prefix_attention``: decode attention of sequences whose contexts begin with the same keys;
* ``adjust_logits``: penalties for repeated tokens, biases and a grammar mask, ahead of the sampler.

With ``own`` false ``run`` computes them from elementary torch operations in 32 bits; with ``own``
true it calls relay_b200.ops. ``exact`` states each of them once more in 64 bits.
"""
import math

import torch

own = False

EPS = 1e-6
THETA = 500000.0


# ---- sizes ------------------------------------------------------------------------------------


def _spread(lo, hi, n):
    """n whole numbers from lo to hi, in a scrambled but fixed order, both ends among them where n > 1."""
    if n == 1:
        return [hi]
    step = next(s for s in (7, 11, 13, 17, 19, 23) if math.gcd(s, n) == 1)
    return [lo + (hi - lo) * ((i * step) % n) // (n - 1) for i in range(n)]


def _group_sizes(tokens, groups):
    """`tokens` split over `groups`, at least one each, unevenly."""
    weights = [1 + (3 * g) % 5 for g in range(groups)]
    rest, total = tokens - groups, sum(weights)
    sizes = [1 + rest * w // total for w in weights]
    sizes[0] += tokens - sum(sizes)
    return sizes


def _chunks(case):
    return _spread(case["chunk_lo"], case["chunk_hi"], case["seqs"])


def listed():
    return [
        # one sequence's decode token: launch latency
        {"name": "qkv_1x1_d128", "op": "qkv", "seqs": 1, "chunk_lo": 1, "chunk_hi": 1, "max_pos": 4096, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "block": 16, "bias": False},
        # a full decode batch, contexts up to 128 k: large rotation angles
        {"name": "qkv_256x1_d128", "op": "qkv", "seqs": 256, "chunk_lo": 1, "chunk_hi": 1, "max_pos": 131072, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "block": 16, "bias": False},
        # prompt chunks of a model with as many KV heads as query heads, biased projections and half of each head rotated
        {"name": "qkv_5xragged_d64_rot32", "op": "qkv", "seqs": 5, "chunk_lo": 33, "chunk_hi": 777, "max_pos": 6000, "heads": 16,
         "kv_heads": 16, "dim": 64, "rot": 32, "block": 32, "bias": True},
        # a large prefill step: eight prompts at once
        {"name": "qkv_8x2048_d128", "op": "qkv", "seqs": 8, "chunk_lo": 2048, "chunk_hi": 2048, "max_pos": 2048, "heads": 32,
         "kv_heads": 8, "dim": 128, "rot": 128, "block": 16, "bias": False},
        # four requests behind a short system prompt, a few tokens in: launch latency
        {"name": "prefix_4x500", "op": "prefix", "tokens": 4, "groups": 1, "prefix_lo": 500, "prefix_hi": 500, "suffix_lo": 1,
         "suffix_hi": 40, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16},
        # an ordinary batch behind a few-shot prompt
        {"name": "prefix_32x4096", "op": "prefix", "tokens": 32, "groups": 1, "prefix_lo": 4096, "prefix_hi": 4096, "suffix_lo": 64,
         "suffix_hi": 512, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16},
        # rollouts of one prompt: many samples, a long shared part, different lengths behind it
        {"name": "prefix_256x8192", "op": "prefix", "tokens": 256, "groups": 1, "prefix_lo": 8192, "prefix_hi": 8192, "suffix_lo": 128,
         "suffix_hi": 640, "heads": 32, "kv_heads": 8, "dim": 128, "block": 16},
        # several prompts, some shared by many requests and some by few, odd lengths, seven heads to a KV head
        {"name": "prefix_96_in_6_groups_d64", "op": "prefix", "tokens": 96, "groups": 6, "prefix_lo": 17, "prefix_hi": 5003,
         "suffix_lo": 1, "suffix_hi": 901, "heads": 14, "kv_heads": 2, "dim": 64, "block": 32},
        # questions about one long document
        {"name": "prefix_8x65537", "op": "prefix", "tokens": 8, "groups": 1, "prefix_lo": 65537, "prefix_hi": 65537, "suffix_lo": 20,
         "suffix_hi": 300, "heads": 40, "kv_heads": 8, "dim": 128, "block": 16},
        # a small model with small pages
        {"name": "prefix_48x777_d32", "op": "prefix", "tokens": 48, "groups": 2, "prefix_lo": 300, "prefix_hi": 777, "suffix_lo": 1,
         "suffix_hi": 100, "heads": 16, "kv_heads": 4, "dim": 32, "block": 8},
        # one request under a grammar: launch latency
        {"name": "logits_1x128256", "op": "logits", "rows": 1, "vocab": 128256, "history_lo": 800, "history_hi": 800, "biases": 4,
         "mask": True},
        # a full batch with long histories
        {"name": "logits_256x128256", "op": "logits", "rows": 256, "vocab": 128256, "history_lo": 40, "history_hi": 8192, "biases": 16,
         "mask": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    most = {op: max(work(c)["bytes"] + work(c)["flops"] / 200 for c in listed() if c["op"] == op) for op in ("qkv", "prefix", "logits")}
    while True:
        op = rng.choice(("qkv", "prefix", "prefix", "logits"))
        if op == "logits":
            history = _log_int(rng, 1, 32768)
            case = {"op": op, "rows": _log_int(rng, 1, 256), "vocab": _log_int(rng, 1000, 160000), "history_lo": rng.randint(0, history),
                    "history_hi": history, "biases": rng.choice((0, 1, 5, 64, 300)), "mask": rng.random() < 0.7}
        else:
            heads, kv_heads = rng.choice(((32, 8), (16, 16), (14, 2), (40, 8), (12, 4), (16, 1), (9, 3)))
            case = {"op": op, "heads": heads, "kv_heads": kv_heads, "block": rng.choice((8, 16, 16, 32, 64))}
            if op == "qkv":
                chunk, dim = rng.choice((1, _log_int(rng, 1, 4096))), rng.choice((32, 64, 80, 128, 128, 256))
                case |= {"seqs": _log_int(rng, 1, 256), "chunk_lo": rng.randint(1, chunk), "chunk_hi": chunk,
                         "max_pos": chunk + _log_int(rng, 1, 131072), "dim": dim, "rot": rng.choice((dim, dim, dim // 2)),
                         "bias": rng.random() < 0.5}
            else:
                tokens, prefix, suffix = _log_int(rng, 1, 256), _log_int(rng, 8, 65536), _log_int(rng, 1, 2048)
                groups = rng.choice((1, 1, rng.randint(1, min(tokens, 12))))
                case |= {"tokens": tokens, "groups": groups, "prefix_lo": rng.choice((prefix, rng.randint(0, prefix))),
                         "prefix_hi": prefix, "suffix_lo": rng.randint(1, suffix), "suffix_hi": suffix,
                         "dim": rng.choice((16, 32, 64, 64, 128, 128, 128))}
        w = work(case)
        if w["bytes"] + w["flops"] / 200 <= most[op]:
            return case


def work(case):
    if case["op"] == "logits":
        values = case["rows"] * case["vocab"]
        tokens = sum(_spread(case["history_lo"], case["history_hi"], case["rows"]))
        return {"bytes": 8 * values + (values // 8 if case["mask"] else 0) + 4 * tokens + 8 * case["rows"] * case["biases"],
                "flops": 4 * values}
    q, kv = case["heads"] * case["dim"], case["kv_heads"] * case["dim"]
    if case["op"] == "qkv":
        n = sum(_chunks(case))
        return {"bytes": n * (4 * (q + 2 * kv) + 4 * q + 4 * kv + 8), "flops": 8 * n * (q + kv)}
    sizes = _group_sizes(case["tokens"], case["groups"])
    prefixes = _spread(case["prefix_lo"], case["prefix_hi"], case["groups"])
    suffixes = _spread(case["suffix_lo"], case["suffix_hi"], case["tokens"])
    keys = sum(prefixes) + sum(suffixes)
    seen = sum(s * p for s, p in zip(sizes, prefixes)) + sum(suffixes)
    return {"bytes": 4 * kv * keys + 6 * q * case["tokens"] + 4 * (keys // case["block"]), "flops": 4 * q * seen}


# ---- inputs -----------------------------------------------------------------------------------


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _prepare_qkv(case, gen):
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    lens = _chunks(case)
    room = max(0, case["max_pos"] - case["chunk_hi"])
    starts = _spread(room // 3, room, case["seqs"])
    pos, seq, off, tables, used = [], [], [], [], 0
    for s, (start, n) in enumerate(zip(starts, lens)):
        # only the blocks that the chunk touches are this pool's; the context before them lies elsewhere
        first, last = start // block, (start + n - 1) // block
        off.append(len(tables))
        tables += [0] * first + list(range(used, used + last - first + 1))
        used += last - first + 1
        pos += range(start, start + n)
        seq += [s] * n
    order = torch.randperm(used, generator=gen, device="cuda").int()
    tokens, width = len(pos), (heads + 2 * kv_heads) * dim
    exponent = torch.arange(0, case["rot"], 2, dtype=torch.float64, device="cuda") / case["rot"]
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    return {"qkv": normal(tokens, width) * 2.0, "bias": normal(width) * 0.1 if case["bias"] else None,
            "q_norm": 1 + 0.1 * normal(dim), "k_norm": 1 + 0.1 * normal(dim), "inv_freq": (THETA ** -exponent).float(),
            "pos": _ints(pos), "seq": _ints(seq), "table_off": _ints(off), "tables": order[_ints(tables).long()],
            "q_out": torch.zeros(tokens, heads * dim, device="cuda"),
            "k_pool": torch.zeros(used, kv_heads, block, dim, dtype=torch.float16, device="cuda"),
            "v_pool": torch.zeros(used, kv_heads, block, dim, dtype=torch.float16, device="cuda")}


def _prepare_prefix(case, gen):
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    sizes = _group_sizes(case["tokens"], case["groups"])
    prefixes = _spread(case["prefix_lo"], case["prefix_hi"], case["groups"])
    suffixes = _spread(case["suffix_lo"], case["suffix_hi"], case["tokens"])
    # A sequence's table starts with its group's blocks. The block in which an odd prefix ends holds
    # keys of its own behind it, so it is a copy in each sequence, as a server makes on the first write.
    pos, off, tables, copies, used, i = [], [], [], [], 0, 0
    for size, prefix in zip(sizes, prefixes):
        whole = prefix // block
        shared, source = list(range(used, used + whole)), None
        used += whole
        for _ in range(size):
            ctx = prefix + suffixes[i]
            mine = list(range(used, used + -(-ctx // block) - whole))
            used += len(mine)
            if prefix % block:
                if source is None:
                    source = mine[0]
                else:
                    copies.append((source, mine[0], prefix % block))
            tables += [0] * (-len(tables) % 4)
            off.append(len(tables))
            tables += shared + mine
            pos.append(ctx - 1)
            i += 1
    order = torch.randperm(used, generator=gen, device="cuda")
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")  # noqa: E731
    k_pool, v_pool = (torch.randn(used, kv_heads, block, dim, generator=gen, dtype=torch.float16, device="cuda") for _ in range(2))
    for src, dst, n in copies:
        for pool in (k_pool, v_pool):
            pool[order[dst], :, :n] = pool[order[src], :, :n]
    group_off = [0]
    for size in sizes:
        group_off.append(group_off[-1] + size)
    return {"q": normal(case["tokens"], (heads + 2 * kv_heads) * dim), "pos": _ints(pos), "seq": _ints(list(range(case["tokens"]))),
            "table_off": _ints(off), "tables": order[_ints(tables).long()].int(), "decode_tokens": _ints(list(range(case["tokens"]))),
            "group_off": _ints(group_off), "prefix_len": _ints(prefixes), "k_pool": k_pool, "v_pool": v_pool,
            "out": torch.zeros(case["tokens"], heads * dim, dtype=torch.float16, device="cuda"),
            "max_group": max(sizes), "max_prefix": max(prefixes), "max_suffix": max(suffixes)}


def _prepare_logits(case, gen):
    rows, vocab = case["rows"], case["vocab"]
    lens = _spread(case["history_lo"], case["history_hi"], rows)
    cap = max(1, case["history_hi"])
    uniform = lambda *shape: torch.rand(*shape, generator=gen, device="cuda")  # noqa: E731
    # text repeats itself: small ids are frequent, large ones rare
    history = (uniform(rows, cap) ** 4 * vocab).int().clamp_(0, vocab - 1)
    params = torch.stack([1.0 + 0.5 * uniform(rows), uniform(rows), 0.5 * uniform(rows), torch.zeros(rows, device="cuda")], 1)
    state = {"logits": torch.randn(rows, vocab, generator=gen, device="cuda") * 4.0, "out": torch.zeros(rows, vocab, device="cuda"),
             "params": params.contiguous(), "history": history, "history_len": _ints(lens), "prompt_len": _ints([n // 2 for n in lens]),
             "bias_ids": None, "bias_values": None, "bias_len": None, "mask": None}
    if case["biases"]:
        state["bias_ids"] = torch.randint(0, vocab, (rows, case["biases"]), generator=gen, device="cuda", dtype=torch.int32)
        state["bias_values"] = torch.randn(rows, case["biases"], generator=gen, device="cuda") * 5.0
        state["bias_len"] = _ints([case["biases"]] * rows)
    if case["mask"]:
        words = -(-vocab // 32)
        # a grammar leaves anything between a handful of tokens and nearly all of them
        some = torch.randint(-2**31, 2**31 - 1, (rows, words), generator=gen, device="cuda", dtype=torch.int32)
        few = uniform(rows, words) < 0.02
        keep = torch.arange(rows, device="cuda")[:, None] % 2 == 0
        state["mask"] = torch.where(keep | few, some, torch.zeros_like(some))
    return state


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    state = {"qkv": _prepare_qkv, "prefix": _prepare_prefix, "logits": _prepare_logits}[case["op"]](case, gen)
    state["case"] = case
    return state


# ---- the framework's calls --------------------------------------------------------------------


def _own(state):
    from relay_b200 import ops
    case = state["case"]
    if case["op"] == "logits":
        return ops.adjust_logits(state["logits"], state["out"], state["params"], state["history"], state["history_len"],
                                 state["prompt_len"], state["bias_ids"], state["bias_values"], state["bias_len"], state["mask"])
    meta = ops.TokenMeta(state["pos"], state["seq"], state["table_off"], state["tables"])
    if case["op"] == "qkv":
        ops.qkv_norm_post(state["qkv"], state["bias"], state["q_norm"], state["k_norm"], EPS, state["inv_freq"], meta,
                          state["q_out"], state["k_pool"], state["v_pool"], case["heads"], case["kv_heads"], case["dim"], case["block"],
                          rot_dim=case["rot"])
        return {"q": state["q_out"], "k_pool": state["k_pool"], "v_pool": state["v_pool"]}
    shape = ops.attn_shape(case["heads"], case["kv_heads"], case["dim"], case["block"])
    return ops.shared_prefix_attention(shape, state["q"], meta, state["decode_tokens"], state["group_off"], state["prefix_len"],
                                       state["max_prefix"], state["max_suffix"], state["k_pool"], state["v_pool"], state["out"])


# ---- the plain forms --------------------------------------------------------------------------


def _plain_qkv(s):
    case = s["case"]
    heads, kv_heads, dim, block, half = case["heads"], case["kv_heads"], case["dim"], case["block"], case["rot"] // 2
    x = s["qkv"] if s["bias"] is None else s["qkv"] + s["bias"]
    x = x.view(x.shape[0], heads + 2 * kv_heads, dim)
    angle = (s["pos"].double()[:, None] * s["inv_freq"].double()).unsqueeze(1)
    cos, sin = angle.cos().float(), angle.sin().float()

    def normed(y, weight):
        return y * torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS) * weight

    def rotated(y):
        a, b = y[..., :half], y[..., half:2 * half]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., 2 * half:]], -1)

    q, k = rotated(normed(x[:, :heads], s["q_norm"])), rotated(normed(x[:, heads:heads + kv_heads], s["k_norm"]))
    pos = s["pos"].long()
    page = s["tables"][s["table_off"][s["seq"].long()].long() + pos // block].long()
    s["q_out"].copy_(q.reshape(q.shape[0], heads * dim))
    s["k_pool"][page, :, pos % block] = k.half()
    s["v_pool"][page, :, pos % block] = x[:, heads + kv_heads:].half()
    return {"q": s["q_out"], "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _plain_prefix(s):
    case = s["case"]
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    tok = s["decode_tokens"].long()
    n, per = tok.numel(), heads // kv_heads
    start = s["group_off"][:-1].long()
    index = torch.arange(n, device="cuda")
    group_of = torch.bucketize(index, s["group_off"][1:].long(), right=True)
    prefix = s["prefix_len"].long()
    row_off = s["table_off"][s["seq"].long()].long()
    ctx = s["pos"][tok].long() + 1
    q = s["q"][tok, :heads * dim].view(n, kv_heads, per, dim) * dim ** -0.5

    def keys(first_row, at, valid):
        page = s["tables"][torch.where(valid, row_off[first_row][:, None] + at // block, 0)].long()
        return s["k_pool"][page, :, at % block].float(), s["v_pool"][page, :, at % block].float()

    # the shared keys, once for each group: queries padded to the largest group
    at = torch.arange(s["max_prefix"], device="cuda")[None].expand(start.numel(), -1)
    valid = at < prefix[:, None]
    k, v = keys(tok[start], at, valid)
    slot = index - start[group_of]
    padded = torch.zeros(start.numel(), s["max_group"], kv_heads, per, dim, device="cuda")
    padded[group_of, slot] = q
    shared = torch.einsum("gmkhd,gpkd->gmkhp", padded, k)
    shared = shared.masked_fill(~valid[:, None, None, None], -math.inf)
    # each sequence's own keys
    own_at = prefix[group_of][:, None] + torch.arange(s["max_suffix"], device="cuda")
    own_valid = own_at < ctx[:, None]
    own_k, own_v = keys(tok, own_at, own_valid)
    mine = torch.einsum("nkhd,npkd->nkhp", q, own_k).masked_fill(~own_valid[:, None, None], -math.inf)
    # one softmax over both
    top = torch.cat([shared[group_of, slot].amax(-1, keepdim=True), mine.amax(-1, keepdim=True)], -1).amax(-1, keepdim=True)
    tops = torch.zeros(start.numel(), s["max_group"], kv_heads, per, 1, device="cuda")
    tops[group_of, slot] = top
    shared, mine = torch.exp(shared - tops), torch.exp(mine - top)
    total = shared.sum(-1, keepdim=True)[group_of, slot] + mine.sum(-1, keepdim=True)
    out = torch.einsum("gmkhp,gpkd->gmkhd", shared, v)[group_of, slot] + torch.einsum("nkhp,npkd->nkhd", mine, own_v)
    s["out"][tok] = (out / total).reshape(n, heads * dim).half()
    return s["out"]


def _plain_logits(s):
    x = s["logits"]
    rows, vocab = x.shape
    ids = s["history"].long()
    at = torch.arange(ids.shape[1], device="cuda")
    known = (at < s["history_len"][:, None]) & (ids >= 0) & (ids < vocab)
    drawn = known & (at >= s["prompt_len"][:, None])
    # what does not count goes to a column behind the vocabulary
    seen = torch.zeros(rows, vocab + 1, dtype=torch.bool, device="cuda")
    seen.scatter_(1, torch.where(known, ids, vocab), True)
    count = torch.zeros(rows, vocab + 1, dtype=torch.int32, device="cuda")
    count.scatter_add_(1, torch.where(drawn, ids, vocab), torch.ones_like(ids, dtype=torch.int32))
    seen, count = seen[:, :vocab], count[:, :vocab]
    repetition, presence, frequency = s["params"][:, 0:1], s["params"][:, 1:2], s["params"][:, 2:3]
    x = torch.where(seen, torch.where(x > 0, x / repetition, x * repetition), x)
    x = torch.where(count > 0, x - (count.float() * frequency + presence), x)
    if s["bias_ids"] is not None:
        at = torch.arange(s["bias_ids"].shape[1], device="cuda")
        valid = (at < s["bias_len"][:, None]) & (s["bias_ids"] >= 0) & (s["bias_ids"] < vocab)
        last = torch.full((rows, vocab + 1), -1, dtype=torch.int64, device="cuda")
        last.scatter_reduce_(1, torch.where(valid, s["bias_ids"].long(), vocab), at.expand(rows, -1).contiguous(), "amax")
        last = last[:, :vocab]
        x = torch.where(last >= 0, x + s["bias_values"].gather(1, last.clamp(min=0)), x)
    if s["mask"] is not None:
        token = torch.arange(vocab, device="cuda")
        x = torch.where((s["mask"][:, token // 32] >> (token % 32).int()) & 1 == 1, x, -math.inf)
    return s["out"].copy_(x)


def run(state):
    if own:
        return _own(state)
    return {"qkv": _plain_qkv, "prefix": _plain_prefix, "logits": _plain_logits}[state["case"]["op"]](state)


# ---- in 64 bits -------------------------------------------------------------------------------


def _exact_qkv(s):
    case = s["case"]
    heads, kv_heads, dim, block, half = case["heads"], case["kv_heads"], case["dim"], case["block"], case["rot"] // 2
    x = s["qkv"].double()
    if s["bias"] is not None:
        x = x + s["bias"].double()
    q, k, v = x.split([heads * dim, kv_heads * dim, kv_heads * dim], 1)
    angle = torch.outer(s["pos"].double(), s["inv_freq"].double())
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    results = []
    for part, count, weight in ((q, heads, s["q_norm"]), (k, kv_heads, s["k_norm"])):
        y = part.reshape(-1, count, dim)
        y = y / (y.square().sum(-1, keepdim=True) / dim + EPS).sqrt() * weight.double()
        z = torch.complex(y[..., :half].contiguous(), y[..., half:2 * half].contiguous()) * turn
        results.append(torch.cat([z.real, z.imag, y[..., 2 * half:]], -1))
    k_pool, v_pool = torch.zeros_like(s["k_pool"], dtype=torch.float64), torch.zeros_like(s["v_pool"], dtype=torch.float64)
    pos = s["pos"].long()
    entry = s["tables"].long()[s["table_off"].long()[s["seq"].long()] + torch.div(pos, block, rounding_mode="floor")]
    rows = entry[:, None] * kv_heads + torch.arange(kv_heads, device="cuda")
    rows = rows * block + (pos % block)[:, None]
    k_pool.view(-1, dim)[rows] = results[1]
    v_pool.view(-1, dim)[rows] = v.reshape(-1, kv_heads, dim)
    return {"q": results[0].reshape(-1, heads * dim), "k_pool": k_pool, "v_pool": v_pool}


def _exact_prefix(s):
    case = s["case"]
    heads, kv_heads, dim, block = case["heads"], case["kv_heads"], case["dim"], case["block"]
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    pos, off = s["pos"].tolist(), s["table_off"].tolist()
    for t, seq in zip(s["decode_tokens"].tolist(), s["seq"].tolist()):
        ctx = pos[t] + 1
        pages = s["tables"][off[seq]:off[seq] + -(-ctx // block)].long()
        k, v = (pool[pages].double().transpose(1, 2).reshape(-1, kv_heads, dim)[:ctx] for pool in (s["k_pool"], s["v_pool"]))
        q = s["q"][t, :heads * dim].double().view(kv_heads, -1, dim)
        weight = torch.softmax(q @ k.permute(1, 2, 0) / math.sqrt(dim), -1)
        out[t] = (weight @ v.transpose(0, 1)).reshape(-1)
    return out


def _exact_logits(s):
    out = s["logits"].double().clone()
    vocab = out.shape[1]
    for r in range(out.shape[0]):
        row, n, prompt = out[r], int(s["history_len"][r]), int(s["prompt_len"][r])
        repetition, presence, frequency, _ = s["params"][r].double()
        ids = s["history"][r, :n].long()
        seen = torch.bincount(ids, minlength=vocab) > 0
        count = torch.bincount(ids[prompt:], minlength=vocab).double()
        row[seen & (row > 0)] /= repetition
        row[seen & (s["logits"][r] <= 0)] *= repetition
        row -= (count > 0) * presence + count * frequency
        if s["bias_ids"] is not None:
            listed_ids = dict(zip(s["bias_ids"][r].tolist(), s["bias_values"][r].double().tolist()))
            row[torch.tensor(list(listed_ids), device="cuda")] += torch.tensor(list(listed_ids.values()), dtype=torch.float64, device="cuda")
        if s["mask"] is not None:
            bits = torch.arange(32, device="cuda")
            allowed = ((s["mask"][r].long()[:, None] >> bits) & 1).reshape(-1)[:vocab]
            row[allowed == 0] = -math.inf
    return out


def exact(case, seed):
    return {"qkv": _exact_qkv, "prefix": _exact_prefix, "logits": _exact_logits}[case["op"]](prepare(case, seed))
