"""The operators of a serving step over the paged cache, as cases that can be timed and compared: the step's layout (positions, cache rows,
pages taken and given back) from the requests' lengths, rotary positions with the store into the pages, attention of ragged batches, and the
rules for logits in front of the sampler.

`run` computes them in plain torch operations, or where `own` is set through `qwen_inference_engine_b200.layers`.
"""
import math

import numpy as np
import torch

own = False

# heads, kv heads, head size: the architectures of qwen_inference_engine_b200/engine.py, and head counts of none of them
HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128), "plain64": (4, 4, 64), "wide": (16, 1, 128), "odd": (15, 3, 64)}
VOCABS = (151936, 152064, 4096)
LAYERS, LAYER = 2, 1  # the pool has two layers and the calls work on the second one


def listed():
    return [
        # a decode step of 64 sequences of ordinary length: latency counts
        {"name": "layout_decode_64", "op": "layout", "decode": 64, "portions": 0, "tokens": 0, "done": 0, "context": 2048, "page": 16},
        # a mixed step: 300 sequences that decode, ragged portions of prompts, requests that are over
        {"name": "layout_mixed_8192", "op": "layout", "decode": 300, "portions": 23, "tokens": 7892, "done": 17, "context": 4096, "page": 16},
        # a full load of long prompts, with the reference's pages of four positions
        {"name": "layout_prompts_131072", "op": "layout", "decode": 1000, "portions": 200, "tokens": 130072, "done": 100, "context": 8192, "page": 4},
        # positions and store of a decode step of 64 sequences
        {"name": "rope_decode_64", "op": "rope", "heads": "7b", "tokens": 64, "pairs": "half", "rotated": 128, "scaling": "none", "far": 8192, "page": 16},
        # a portion of prompts at positions that YaRN's frequencies are for
        {"name": "rope_yarn_8192", "op": "rope", "heads": "1.5b", "tokens": 8192, "pairs": "half", "rotated": 128, "scaling": "yarn", "far": 131072, "page": 16},
        # half of each head rotated, neighbours as pairs, linear scaling, an odd number of tokens at far positions
        {"name": "rope_partial_20011", "op": "rope", "heads": "0.5b", "tokens": 20011, "pairs": "neighbours", "rotated": 32, "scaling": "linear", "far": 1000000, "page": 16},
        # one sequence's single token: the smallest call
        {"name": "attention_single_700", "op": "attention", "heads": "0.5b", "decode": 1, "portions": 0, "portion": 0, "context": 700, "window": 0, "page": 16},
        # a decode step of 64 ragged sequences
        {"name": "attention_decode_64x2048", "op": "attention", "heads": "7b", "decode": 64, "portions": 0, "portion": 0, "context": 2048, "window": 0, "page": 16},
        # a mixed step: sequences that decode beside ragged portions of prompts behind cached positions
        {"name": "attention_mixed_52", "op": "attention", "heads": "1.5b", "decode": 48, "portions": 4, "portion": 500, "context": 4000, "window": 0, "page": 16},
        # a long prompt in one portion: the largest
        {"name": "attention_prompt_8192", "op": "attention", "heads": "7b", "decode": 0, "portions": 1, "portion": 8192, "context": 0, "window": 0, "page": 16},
        # one row of 32-bit logits, a conversation's penalties, no mask
        {"name": "logits_single_fp32", "op": "logits", "rows": 1, "vocab": 151936, "dtype": "float32", "history": 2000, "bias": 10, "masked": 0},
        # a batch of 64 rows with long histories, biases, and a grammar's mask for each second row
        {"name": "logits_batch_64", "op": "logits", "rows": 64, "vocab": 151936, "dtype": "bfloat16", "history": 4000, "bias": 300, "masked": 32},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layout", "rope", "attention", "attention", "attention", "logits"])
    if op == "layout":
        portions = rng.choice([0, _log(rng, 1, 200)])
        tokens = _log(rng, portions, 130000) if portions else 0
        return {"op": op, "decode": _log(rng, 1, 1000), "portions": portions, "tokens": tokens, "done": rng.choice([0, _log(rng, 1, 100)]),
                "context": _log(rng, 1, 8192), "page": rng.choice([4, 8, 16, 16, 64])}
    if op == "rope":
        heads = rng.choice(list(HEADS))
        n_q, _, hd = HEADS[heads]
        return {"op": op, "heads": heads, "tokens": _log(rng, 1, 20000 * 14 * 64 // (n_q * hd)), "pairs": rng.choice(["half", "neighbours"]),
                "rotated": rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]), "scaling": rng.choice(["none", "linear", "yarn"]),
                "far": _log(rng, 100, 1000000), "page": rng.choice([4, 16, 16, 24])}
    if op == "attention":
        heads, decode, portions = rng.choice(list(HEADS)), rng.choice([0, _log(rng, 1, 64)]), rng.choice([0, rng.randint(1, 6)])
        if decode + portions == 0:
            decode = _log(rng, 1, 64)
        portion = _log(rng, 2, 2000) if portions else 0
        # the padded form of the batch costs no more than the long prompt's
        most = int(1.8e9 / ((decode + portions) * max(1, portion) * HEADS[heads][0])) - portion
        context = _log(rng, 1, max(2, min(8000, most)))
        return {"op": op, "heads": heads, "decode": decode, "portions": portions, "portion": portion, "context": context,
                "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]), "page": rng.choice([4, 16, 16, 16, 24, 64])}
    rows = _log(rng, 1, 64)
    return {"op": op, "rows": rows, "vocab": rng.choice(list(VOCABS) + [rng.randint(500, 150000)]), "dtype": rng.choice(["bfloat16", "float32"] if rows <= 32 else ["bfloat16"]),
            "history": rng.choice([0, _log(rng, 1, 4000)]), "bias": rng.choice([0, _log(rng, 1, 300)]), "masked": rng.choice([0, rows, rng.randint(0, rows)])}


# ---------------------------------------------------------------- inputs
def _spread(rs, lo, hi, n):
    """n lengths from lo to hi, evenly spaced, in an order of the seed"""
    return rs.permutation(np.linspace(lo, hi, n).round().astype(np.int64)) if n else np.zeros(0, np.int64)


def _shares(tokens, n):
    """`tokens` in n ragged portions, none of them empty"""
    w = np.arange(1, n + 1, dtype=np.float64) ** 1.5
    return 1 + np.floor((tokens - n) * w / w.sum()).astype(np.int64)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


def _tables(rs, pages, slots, wide, spare):
    """(block table, page ids that no request has): request i has pages[i] pages in its row"""
    owned = int(pages.sum())
    ids = rs.permutation(owned + spare)
    table = np.full((len(pages), wide), 0, np.int64)
    at = np.concatenate([[0], np.cumsum(pages)])
    table[np.repeat(slots, pages), np.arange(owned) - np.repeat(at[:-1], pages)] = ids[:owned]
    return table, ids[owned:]


def _lengths(case):
    """(cached, new) of the attention cases, as ranges that do not hang on the seed"""
    d, p = case["decode"], case["portions"]
    cached = np.concatenate([np.linspace(case["context"] * 0.4, case["context"], d).round(), np.linspace(0, case["context"], p + 2).round()[1:-1]])
    new = np.concatenate([np.ones(d), np.linspace((case["portion"] + 1) // 2, case["portion"], p + 1).round()[1:]])
    return np.maximum(0, cached - (new == 1) * (cached > 0)).astype(np.int64), new.astype(np.int64)


def _frequencies(rotated, scaling):
    """(radians a position, factor of the cosines and sines)"""
    i = np.arange(rotated // 2, dtype=np.float64)
    base = 1000000.0
    w = base ** (-2 * i / rotated)
    if scaling == "linear":
        return w / 8, 1.0
    if scaling == "yarn":  # long wavelengths divided by four, short ones kept, a ramp between
        at = lambda turns: rotated * math.log(32768 / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
        lo, hi = max(0, math.floor(at(32))), min(rotated - 1, math.ceil(at(1)))
        keep = 1 - np.clip((i - lo) / max(hi - lo, 1e-3), 0, 1)
        return w * keep + w / 4 * (1 - keep), 0.1 * math.log(4) + 1
    return w, 1.0


def prepare(case, seed):
    rs, g = np.random.RandomState(seed % (1 << 32)), torch.Generator("cuda").manual_seed(seed)
    s = {"case": case}

    def rand(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    if case["op"] == "layout":
        ps = case["page"]
        new = np.concatenate([np.ones(case["decode"], np.int64), _shares(case["tokens"], case["portions"]), np.full(case["done"], -1)])
        cached = np.concatenate([_spread(rs, case["context"] // 2, case["context"], case["decode"]), _spread(rs, 0, case["context"], case["portions"]),
                                 _spread(rs, 1, case["context"], case["done"])])
        order, n = rs.permutation(len(new)), len(new)
        new, cached, slots = new[order].astype(np.int64), cached[order].astype(np.int64), rs.permutation(n)
        had = -(-cached // ps)
        wide = -(-(case["context"] + int(new.max())) // ps) + 3
        table, spare = _tables(rs, had, slots, wide, int((np.maximum(new, 0) // ps + 1).sum()) + 7)  # as many as it can take, and some
        pages = int(had.sum()) + len(spare)
        ring, first = np.zeros(pages, np.int64), int(rs.randint(pages))
        ring[(first + np.arange(len(spare))) % pages] = spare
        s.update(cached=_i32(cached), new=_i32(new), slots=_i32(slots), table=_i32(table), ring=_i32(ring), ring_in=_i32([first, len(spare)]),
                 max_tokens=int(np.maximum(new, 0).sum()) + 5, pages=pages, most_pages=wide)
        return s
    if case["op"] == "logits":
        rows, vocab, dtype = case["rows"], case["vocab"], getattr(torch, case["dtype"])
        s["logits"] = (rand(rows, vocab) * 4).to(dtype)
        s["out"] = torch.empty_like(s["logits"])
        have = _spread(rs, case["history"] // 2, case["history"], rows)
        start = np.concatenate([[0], np.cumsum(have)])
        s["tokens"] = _i32(np.minimum((vocab * rs.rand(start[-1]) ** 3).astype(np.int64), vocab - 1))  # frequent tokens come often
        s["tok_start"], s["gen_start"] = _i32(start), _i32(start[:-1] + have // 3)
        s["repetition"], s["presence"], s["frequency"] = (torch.from_numpy(a.astype(np.float32)).cuda() for a in (rs.uniform(1, 1.5, rows), rs.uniform(0, 1, rows), rs.uniform(0, .5, rows)))
        s["bias_start"] = _i32(np.arange(rows + 1) * case["bias"])
        s["bias_ids"] = _i32(rs.randint(0, vocab, rows * case["bias"]))
        s["bias"] = torch.from_numpy(rs.uniform(-5, 5, rows * case["bias"]).astype(np.float32)).cuda()
        words = (vocab + 31) // 32
        s["mask"] = _i32(rs.randint(-2 ** 31, 2 ** 31, (max(1, case["masked"]), words), np.int64))
        which = np.full(rows, -1)
        which[rs.permutation(rows)[:case["masked"]]] = np.arange(case["masked"])
        s["mask_row"] = _i32(which)
        s["row_of_token"] = torch.repeat_interleave(torch.arange(rows, device="cuda"), torch.from_numpy(have).cuda())
        s["row_of_bias"] = torch.arange(rows, device="cuda").repeat_interleave(case["bias"])
        return s
    n_q, n_kv, hd = HEADS[case["heads"]]
    ps = case["page"]
    if case["op"] == "rope":
        n = case["tokens"]
        pages = -(-n // ps) + 3
        s["qkv"] = rand(n, (n_q + 2 * n_kv) * hd).bfloat16()  # rows as one product of the projections gives them
        s["q_out"] = torch.empty(n, n_q * hd, dtype=torch.bfloat16, device="cuda")
        s["pool"] = rand(pages, LAYERS, 2, n_kv, ps, hd).bfloat16()
        s["pos"] = _i32(rs.randint(0, case["far"], n))
        s["row"] = _i32(rs.permutation(pages * ps)[:n])
        w, s["factor"] = _frequencies(case["rotated"], case["scaling"])
        s["frequencies"] = torch.from_numpy(w).cuda()
        return s
    cached, new = _lengths(case)
    order = rs.permutation(len(new))
    cached, new, n = cached[order], new[order], len(new)
    total, slots = cached + new, rs.permutation(len(new))
    pages = -(-total // ps)
    table, _ = _tables(rs, pages, slots, int(pages.max()) + 2, 5)
    start = np.concatenate([[0], np.cumsum(new)])
    s["pool"] = rand(int(pages.sum()) + 5, LAYERS, 2, n_kv, ps, hd).bfloat16()
    s["q"] = (rand(int(start[-1]), n_q * hd) * 1.5).bfloat16()
    s["out"] = torch.empty_like(s["q"])
    s.update(table=_i32(table), slots=_i32(slots), q_start=_i32(start), kv_len=_i32(total), most_new=int(new.max()), most_len=int(total.max()))
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)(s)


def _plain(s):
    return {"layout": _plain_layout, "rope": _plain_rope, "attention": _plain_attention, "logits": _plain_logits}[s["case"]["op"]](s)


def _plain_layout(s):
    ps, pages, most, dev = s["case"]["page"], s["pages"], s["max_tokens"], "cuda"
    cached, new, slots, table, ring = s["cached"], s["new"], s["slots"].long(), s["table"], s["ring"]
    first, count = s["ring_in"][0], s["ring_in"][1]
    n = new.clamp(min=0)
    had = (cached + ps - 1) // ps
    need, back = (cached + n + ps - 1) // ps - had, torch.where(new < 0, had, 0)

    def sums(x):
        return torch.cat([torch.zeros(1, dtype=torch.int64, device=dev), x.cumsum(0)])

    q_start, taken, given = sums(n), sums(need), sums(back)
    room = n.numel() * s["most_pages"]
    # pages taken out of the ring, into the requests' rows
    j = torch.arange(room, device=dev)
    req = torch.searchsorted(taken[1:], j, right=True).clamp(max=n.numel() - 1)
    col = had[req] + j - taken[req]
    page = ring[(first + j) % pages]
    live = j < taken[-1]
    flat = torch.cat([table.flatten(), table.new_zeros(1)])
    flat[torch.where(live, slots[req] * table.shape[1] + col, table.numel())] = page
    table.copy_(flat[:-1].view_as(table))
    # pages of requests that are over, back into the ring
    req = torch.searchsorted(given[1:], j, right=True).clamp(max=n.numel() - 1)
    old = flat[(slots[req] * table.shape[1] + j - given[req]).clamp(max=table.numel())]
    grown = torch.cat([ring, ring.new_zeros(1)])
    grown[torch.where(j < given[-1], (first + count + j) % pages, pages)] = old
    ring.copy_(grown[:-1])
    # every token's position and cache row
    t = torch.arange(most, device=dev)
    req = torch.searchsorted(q_start[1:], t, right=True).clamp(max=n.numel() - 1)
    live = t < q_start[-1]
    pos = torch.where(live, cached[req] + t - q_start[req], -1)
    at = pos.clamp(min=0)
    row = table[slots[req], (at // ps).clamp(max=table.shape[1] - 1)] * ps + at % ps
    ints = lambda x: x.to(torch.int32)  # noqa: E731
    state = torch.stack([(first + taken[-1]) % pages, count - taken[-1] + given[-1]])
    return {"q_start": ints(q_start), "kv_len": ints(torch.where(new < 0, 0, cached + n)), "pos": ints(pos), "slot": ints(torch.where(live, slots[req], -1)),
            "row": ints(torch.where(live, row, -1)), "table": table, "ring": ring, "ring_out": ints(state)}


def _plain_rope(s):
    case = s["case"]
    n_q, n_kv, hd = HEADS[case["heads"]]
    rot = case["rotated"]
    angle = s["pos"].double()[:, None] * s["frequencies"]
    cos, sin = ((f(angle) * s["factor"]).float()[:, None] for f in (torch.cos, torch.sin))

    def turned(x):
        x = x.float()
        if case["pairs"] == "half":
            a, b = x[..., :rot // 2], x[..., rot // 2:rot]
            r = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
        else:
            a, b = x[..., 0:rot:2], x[..., 1:rot:2]
            r = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
        return torch.cat([r, x[..., rot:]], -1).bfloat16()

    x = s["qkv"].view(-1, n_q + 2 * n_kv, hd)
    s["q_out"].copy_(turned(x[:, :n_q]).flatten(1))
    page, at = s["row"].long() // case["page"], s["row"].long() % case["page"]
    s["pool"][page, LAYER, 0, :, at] = turned(x[:, n_q:n_q + n_kv])
    s["pool"][page, LAYER, 1, :, at] = x[:, n_q + n_kv:]
    return {"q": s["q_out"], "pool": s["pool"]}


def _plain_attention(s):
    case = s["case"]
    n_q, n_kv, hd = HEADS[case["heads"]]
    ps, m, dev = case["page"], s["most_new"], "cuda"
    n_pages = -(-s["most_len"] // ps)
    new = s["q_start"][1:] - s["q_start"][:-1]
    # requests side by side, padded to the longest
    at = s["q_start"][:-1, None].long() + torch.arange(m, device=dev)
    live = torch.arange(m, device=dev) < new[:, None]
    total = s["q"].shape[0]
    q = s["q"][at.clamp(max=total - 1)].view(-1, m, n_kv, n_q // n_kv, hd).permute(0, 2, 1, 3, 4).flatten(2, 3).float()
    pages = s["table"][s["slots"].long(), :n_pages].long()
    k, v = (s["pool"][:, LAYER, i][pages].permute(0, 2, 1, 3, 4).flatten(2, 3).float() for i in (0, 1))
    score = torch.matmul(q, k.transpose(-1, -2)) * hd ** -0.5
    pos = (s["kv_len"] - new)[:, None] + torch.arange(m, device=dev)
    key = torch.arange(n_pages * ps, device=dev)
    seen = key <= pos[..., None]
    if case["window"]:
        seen &= key > pos[..., None] - case["window"]
    seen = seen[:, None, :, None].expand(-1, 1, -1, n_q // n_kv, -1).flatten(2, 3)
    score.masked_fill_(~seen, float("-inf"))
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    o = torch.matmul(score, v) / score.sum(-1, keepdim=True)
    o = o.view(-1, n_kv, m, n_q // n_kv, hd).permute(0, 2, 1, 3, 4).reshape(-1, m, n_q * hd).bfloat16()
    wide = torch.empty(total + 1, n_q * hd, dtype=torch.bfloat16, device=dev)
    wide[torch.where(live, at, total)] = o
    s["out"].copy_(wide[:total])
    return s["out"]


def _plain_logits(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    tokens, who = s["tokens"].long(), s["row_of_token"]
    made = (torch.arange(tokens.numel(), device="cuda") >= s["gen_start"].long()[who]).float()
    flat = who * vocab + tokens
    seen = torch.zeros(rows * vocab, dtype=torch.bool, device="cuda").index_fill_(0, flat, True).view(rows, vocab)
    count = torch.zeros(rows * vocab, device="cuda").index_add_(0, flat, made).view(rows, vocab)
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - s["frequency"][:, None] * count - s["presence"][:, None] * (count > 0)
    bias = torch.zeros(rows * vocab, dtype=torch.float64, device="cuda").index_add_(0, s["row_of_bias"] * vocab + s["bias_ids"].long(), s["bias"].double())
    x = x + bias.float().view(rows, vocab)
    token = torch.arange(vocab, device="cuda")
    allowed = (s["mask"][s["mask_row"].long().clamp(min=0)][:, token // 32] >> (token % 32).int()) & 1
    s["out"].copy_(torch.where((allowed == 0) & (s["mask_row"] >= 0)[:, None], float("-inf"), x))
    return s["out"]


def _own(s):
    from qwen_inference_engine_b200 import layers as L
    case = s["case"]
    if "handles" not in s:  # made once, as a program that serves keeps them beside its buffers
        s["handles"] = _handles(L, s)
    h = s["handles"]
    if case["op"] == "layout":
        b = h["batch"]
        L.launch_batch_layout(b)
        return {"q_start": b.q_start, "kv_len": b.kv_len, "pos": b.pos, "slot": b.slot, "row": b.row, "table": s["table"], "ring": s["ring"], "ring_out": b.ring_out}
    if case["op"] == "logits":
        L.launch_logits(s["logits"], s["out"], h["rules"])
        return s["out"]
    n_q, n_kv, hd = HEADS[case["heads"]]
    if case["op"] == "rope":
        q, k, v = s["qkv"].split([n_q * hd, n_kv * hd, n_kv * hd], 1)
        L.launch_rope_store(q, k, v, s["q_out"], h["pool"], LAYER, s["pos"], s["row"], h["rope"], n_q)
        return {"q": s["q_out"], "pool": s["pool"]}
    L.launch_attn_batch(s["q"], s["out"], h["pool"], LAYER, h["batch"], n_q, window=case["window"])
    return s["out"]


def _handles(L, s):
    case = s["case"]
    if case["op"] == "layout":
        return {"batch": L.Batch(s["table"], case["page"], s["pages"], s["new"].numel(), s["max_tokens"], cached=s["cached"], n_new=s["new"], slots=s["slots"],
                                 free_ring=s["ring"], ring_in=s["ring_in"])}
    if case["op"] == "logits":
        return {"rules": L.LogitRules(s["tok_start"], s["tokens"], gen_start=s["gen_start"], repetition=s["repetition"], presence=s["presence"], frequency=s["frequency"],
                                      bias_start=s["bias_start"], bias_ids=s["bias_ids"], bias=s["bias"], mask=s["mask"], mask_row=s["mask_row"])}
    if case["op"] == "rope":
        return {"pool": L.KvPool.over(s["pool"]), "rope": L.Rope(s["frequencies"], factor=s["factor"], neighbours=case["pairs"] == "neighbours")}
    return {"pool": L.KvPool.over(s["pool"]), "batch": L.Batch(s["table"], case["page"], s["pool"].shape[0], s["slots"].numel(), s["q"].shape[0], slots=s["slots"],
                                                               q_start=s["q_start"], kv_len=s["kv_len"])}


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    if case["op"] == "layout":
        n, t = case["decode"] + case["portions"] + case["done"], case["decode"] + case["tokens"]
        taken, given = t // case["page"], case["done"] * (case["context"] // (2 * case["page"]))
        return {"bytes": 20 * n + 12 * t + 8 * taken + 8 * given + 4 * case["decode"], "flops": 0}
    if case["op"] == "logits":
        size = 4 if case["dtype"] == "float32" else 2
        return {"bytes": case["rows"] * (2 * size * case["vocab"] + 3 * case["history"] + 8 * case["bias"]) + case["masked"] * case["vocab"] // 8,
                "flops": case["rows"] * case["vocab"]}
    n_q, n_kv, hd = HEADS[case["heads"]]
    if case["op"] == "rope":
        return {"bytes": case["tokens"] * (4 * (n_q + 2 * n_kv) * hd + 8), "flops": case["tokens"] * 3 * (n_q + n_kv) * case["rotated"]}
    cached, new = _lengths(case)
    pairs = keys = 0
    for c, n in zip(cached, new):
        p = np.arange(c, c + n)
        low = np.maximum(0, p - case["window"] + 1) if case["window"] else 0 * p
        pairs, keys = pairs + int((p + 1 - low).sum()), keys + int(c + n - low[0])
    return {"bytes": 4 * int(new.sum()) * n_q * hd + 4 * keys * n_kv * hd, "flops": 4 * hd * n_q * pairs}


# ---------------------------------------------------------------- the definitions, in 64 bits
def exact(case, seed):
    if case["op"] == "layout":  # whole numbers only
        return None
    s = prepare(case, seed)
    if case["op"] == "logits":
        out = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
        at, cut, bias_at = s["tok_start"].tolist(), s["gen_start"].tolist(), s["bias_start"].tolist()
        for i in range(case["rows"]):
            x, list_ = s["logits"][i].double(), s["tokens"][at[i]:at[i + 1]].long()
            r, p, f = (float(s[k][i]) for k in ("repetition", "presence", "frequency"))
            distinct = list_.unique()
            v = x[distinct]
            x[distinct] = torch.where(v > 0, v / r, v * r)
            made, times = s["tokens"][cut[i]:at[i + 1]].long().unique(return_counts=True)
            x[made] -= times.double() * f + p
            b = slice(bias_at[i], bias_at[i + 1])
            x.index_add_(0, s["bias_ids"][b].long(), s["bias"][b].double())
            m = int(s["mask_row"][i])
            if m >= 0:
                bits = np.unpackbits(s["mask"][m].cpu().numpy().view(np.uint8), bitorder="little")[:case["vocab"]]
                x[torch.from_numpy(bits == 0).cuda()] = float("-inf")
            out[i] = x
        return out
    n_q, n_kv, hd = HEADS[case["heads"]]
    if case["op"] == "rope":
        rot = case["rotated"]
        i = torch.arange(rot // 2, device="cuda")
        a, b = (i, i + rot // 2) if case["pairs"] == "half" else (2 * i, 2 * i + 1)
        turn = torch.polar(torch.full((), s["factor"], dtype=torch.float64, device="cuda"), torch.outer(s["pos"].double(), s["frequencies"]))[:, None]

        def turned(x):
            z = torch.complex(x[..., a], x[..., b]) * turn
            y = x.clone()
            y[..., a], y[..., b] = z.real, z.imag
            return y

        q, k, v = (t.reshape(case["tokens"], -1, hd).double() for t in s["qkv"].split([n_q * hd, n_kv * hd, n_kv * hd], 1))
        pool = s["pool"].double()
        rows = pool[:, LAYER].permute(1, 0, 3, 2, 4).reshape(2, -1, n_kv, hd)  # [k|v][cache row][head]
        rows[0, s["row"].long()], rows[1, s["row"].long()] = turned(k), v
        pool[:, LAYER] = rows.view(2, -1, case["page"], n_kv, hd).permute(1, 0, 3, 2, 4)
        return {"q": turned(q).flatten(1), "pool": pool}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    start, lens, slots = s["q_start"].tolist(), s["kv_len"].tolist(), s["slots"].tolist()
    for r in range(len(lens)):
        t0, t1, n = start[r], start[r + 1], lens[r]
        pages = s["table"][slots[r], :-(-n // case["page"])].long()
        kv = s["pool"][pages, LAYER].double().permute(1, 2, 0, 3, 4).reshape(2, n_kv, -1, hd)[:, :, :n]
        p = torch.arange(n - (t1 - t0), n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        hidden = (j > p) | (j <= p - (case["window"] or n + 1))
        for h in range(n_q):
            g = h * n_kv // n_q
            x = s["q"][t0:t1, h * hd:(h + 1) * hd].double() @ kv[0, g].T / math.sqrt(hd)
            out[t0:t1, h * hd:(h + 1) * hd] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ kv[1, g]
    return out
