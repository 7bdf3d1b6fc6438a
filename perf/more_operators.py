"""The operators of a serving step over a cache held in 8 bits, as cases that can be timed and compared: rotary positions with the store that quantises keys
and values as they are written, cache rows read back, and attention of ragged batches over such a cache.

The cache: of each token and kv head one vector of codes (e4m3, or int8) and one power of two for keys, and the same for values.  `run` computes the operators in
plain torch operations, or where `own` is set through `qwen_inference_engine_b200.layers`.
"""
import math

import numpy as np
import torch

own = False

# heads, kv heads, head size: the architectures of qwen_inference_engine_b200/engine.py, and head counts of none of them
HEADS = {"0.5b": (14, 2, 64), "1.5b": (12, 2, 128), "7b": (28, 4, 128), "plain64": (4, 4, 64), "wide": (16, 1, 128), "odd": (15, 3, 64)}
LAYERS, LAYER = 2, 1  # the pool has two layers and the calls work on the second one
MOST = {"e4m3": 448, "int8": 127}  # the largest code


def listed():
    return [
        # a decode step of 64 sequences: latency counts
        {"name": "store_decode_64", "op": "store", "heads": "7b", "code": "e4m3", "tokens": 64, "pairs": "half", "rotated": 128, "scaling": "none", "far": 8192, "page": 16},
        # a portion of prompts at positions that YaRN's frequencies are for
        {"name": "store_yarn_8192", "op": "store", "heads": "1.5b", "code": "e4m3", "tokens": 8192, "pairs": "half", "rotated": 128, "scaling": "yarn", "far": 131072, "page": 16},
        # half of each head rotated, neighbours as pairs, linear scaling, an odd number of tokens, in int8, and the rows read back as the values that the cache stands for
        {"name": "store_read_partial_20011", "op": "store", "heads": "0.5b", "code": "int8", "tokens": 20011, "pairs": "neighbours", "rotated": 32, "scaling": "linear", "far": 1000000, "page": 16},
        # one request's rows, out of pages in any order: the smallest call
        {"name": "read_request_701", "op": "read", "heads": "0.5b", "code": "e4m3", "tokens": 701, "page": 16},
        # a long prefix
        {"name": "read_prefix_32768", "op": "read", "heads": "7b", "code": "int8", "tokens": 32768, "page": 16},
        # one sequence's single token
        {"name": "attention_single_700", "op": "attention", "heads": "0.5b", "code": "e4m3", "decode": 1, "portions": 0, "portion": 0, "context": 700, "window": 0, "page": 16},
        # a decode step of 64 ragged sequences
        {"name": "attention_decode_64x2048", "op": "attention", "heads": "7b", "code": "e4m3", "decode": 64, "portions": 0, "portion": 0, "context": 2048, "window": 0, "page": 16},
        # a few long documents: what a cache in 8 bits makes room for
        {"name": "attention_decode_4x100000", "op": "attention", "heads": "1.5b", "code": "int8", "decode": 4, "portions": 0, "portion": 0, "context": 100000, "window": 0, "page": 16},
        # a window, and pages that end inside a tile
        {"name": "attention_window_200", "op": "attention", "heads": "odd", "code": "int8", "decode": 200, "portions": 0, "portion": 0, "context": 4000, "window": 1000, "page": 24},
        # a mixed step: sequences that decode beside ragged portions of prompts behind cached positions
        {"name": "attention_mixed_52", "op": "attention", "heads": "1.5b", "code": "int8", "decode": 48, "portions": 4, "portion": 500, "context": 4000, "window": 0, "page": 16},
        # short portions of many prompts
        {"name": "attention_portions_16", "op": "attention", "heads": "0.5b", "code": "e4m3", "decode": 0, "portions": 16, "portion": 701, "context": 1500, "window": 0, "page": 16},
        # a long prompt in one portion: the largest
        {"name": "attention_prompt_8192", "op": "attention", "heads": "7b", "code": "e4m3", "decode": 0, "portions": 1, "portion": 8192, "context": 0, "window": 0, "page": 16},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op, heads, code = rng.choice(["store", "read", "attention", "attention", "attention"]), rng.choice(list(HEADS)), rng.choice(list(MOST))
    n_q, n_kv, hd = HEADS[heads]
    if op == "store":
        return {"op": op, "heads": heads, "code": code, "tokens": _log(rng, 1, 20000 * 14 * 64 // (n_q * hd)), "pairs": rng.choice(["half", "neighbours"]),
                "rotated": rng.choice([hd, hd, hd // 2, 2 * rng.randint(1, hd // 2)]), "scaling": rng.choice(["none", "linear", "yarn"]),
                "far": _log(rng, 100, 1000000), "page": rng.choice([4, 16, 16, 24])}
    if op == "read":
        return {"op": op, "heads": heads, "code": code, "tokens": _log(rng, 1, 32768 * 4 * 128 // (n_kv * hd)), "page": rng.choice([4, 16, 16, 24])}
    decode, portions = rng.choice([0, _log(rng, 1, 200)]), rng.choice([0, rng.randint(1, 16)])
    if decode + portions == 0:
        decode = _log(rng, 1, 200)
    portion = _log(rng, 2, 2000) if portions else 0
    # the padded form of the batch costs no more than the long prompt's, and the rows of its keys and values no more than the long documents'
    most = min(int(1.8e9 / ((decode + portions) * max(1, portion) * n_q)) - portion, 400000 // (decode + portions))
    context = _log(rng, 1, max(2, min(100000, most)))
    return {"op": op, "heads": heads, "code": code, "decode": decode, "portions": portions, "portion": portion, "context": context,
            "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)]), "page": rng.choice([4, 16, 16, 16, 24, 64])}


# ---------------------------------------------------------------- the cache, in plain torch operations
def _pow2(b):
    """the scales of bytes b, in 32 bits: 2^(b - 127)"""
    return (b.int() << 23).view(torch.float32)


def _coded(x, code):
    """vectors x [..., head size] in 32 bits -> (codes as bytes, the scales' bytes): the smallest power of two with which the largest element is no more than the largest code"""
    m, e = torch.frexp(x.abs().amax(-1))
    b = e + 127 - (9 if code == "e4m3" else 7) + (m > MOST[code] / (512 if code == "e4m3" else 128))
    b = torch.where(m == 0, 0, b.clamp(min=1))
    y = x * _pow2(254 - b)[..., None]
    return (y.to(torch.float8_e4m3fn) if code == "e4m3" else y.round().to(torch.int8)).view(torch.uint8), b.to(torch.uint8)


def _values(codes, scale, code):
    """what codes and scales stand for, in 32 bits"""
    return codes.view(torch.float8_e4m3fn if code == "e4m3" else torch.int8).float() * _pow2(scale)[..., None]


# ---------------------------------------------------------------- inputs
def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).cuda()


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

    n_q, n_kv, hd = HEADS[case["heads"]]
    ps = case["page"]

    def pool(pages):
        """keys and values of tokens whose sizes differ, as a cache holds them"""
        x = rand(pages, LAYERS, 2, n_kv, ps, hd) * torch.exp2(rand(pages, LAYERS, 2, n_kv, ps, 1).mul_(0.7).round_())
        s["codes"], s["scale"] = _coded(x, case["code"])
        s["codes"] = s["codes"].view(torch.float8_e4m3fn if case["code"] == "e4m3" else torch.int8)

    if case["op"] in ("store", "read"):
        n = case["tokens"]
        pages = -(-n // ps) + 3
        pool(pages)
        s["row"] = _i32(rs.permutation(pages)[np.arange(n) // ps] * ps + np.arange(n) % ps if case["op"] == "read" else rs.permutation(pages * ps)[:n])
        s["k"], s["v"] = (torch.empty(n, n_kv * hd, dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
        if case["op"] == "store":
            s["qkv"] = rand(n, (n_q + 2 * n_kv) * hd).bfloat16()  # rows as one product of the projections gives them
            s["q_out"] = torch.empty(n, n_q * hd, dtype=torch.bfloat16, device="cuda")
            s["pos"] = _i32(rs.randint(0, case["far"], n))
            w, s["factor"] = _frequencies(case["rotated"], case["scaling"])
            s["frequencies"] = torch.from_numpy(w).cuda()
        return s
    cached, new = _lengths(case)
    order = rs.permutation(len(new))
    cached, new, n = cached[order], new[order], len(new)
    total, slots = cached + new, rs.permutation(n)
    pages = -(-total // ps)
    owned = int(pages.sum())
    table = np.zeros((n, int(pages.max()) + 2), np.int64)
    first = np.concatenate([[0], np.cumsum(pages)])
    table[np.repeat(slots, pages), np.arange(owned) - np.repeat(first[:-1], pages)] = rs.permutation(owned + 5)[:owned]
    pool(owned + 5)
    start = np.concatenate([[0], np.cumsum(new)])
    s["q"] = (rand(int(start[-1]), n_q * hd) * 1.5).bfloat16()
    s["out"] = torch.empty_like(s["q"])
    s.update(table=_i32(table), slots=_i32(slots), q_start=_i32(start), kv_len=_i32(total), most_new=int(new.max()), most_len=int(total.max()))
    return s


# ---------------------------------------------------------------- one pass
def run(s):
    return (_own if own else _plain)(s)


def _stored(s):
    """what a store leaves: the queries, and the cache as the values of its two types (e4m3), or the rows' values read back"""
    if s["case"]["code"] == "e4m3":
        return {"q": s["q_out"], "codes": s["codes"], "scale": s["scale"].view(torch.float8_e8m0fnu)}
    return {"q": s["q_out"], "k": s["k"], "v": s["v"]}


def _plain(s):
    return {"store": _plain_store, "read": _plain_read, "attention": _plain_attention}[s["case"]["op"]](s)


def _plain_read(s):
    case = s["case"]
    page, at = s["row"].long() // case["page"], s["row"].long() % case["page"]
    for i, out in ((0, s["k"]), (1, s["v"])):
        codes = s["codes"].view(torch.uint8)[page, LAYER, i, :, at]
        out.copy_(_values(codes, s["scale"][page, LAYER, i, :, at], case["code"]).flatten(1))
    return {"k": s["k"], "v": s["v"]}


def _plain_store(s):
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
        return torch.cat([r, x[..., rot:]], -1)

    x = s["qkv"].view(-1, n_q + 2 * n_kv, hd)
    s["q_out"].copy_(turned(x[:, :n_q]).flatten(1))
    page, at = s["row"].long() // case["page"], s["row"].long() % case["page"]
    for i, y in ((0, turned(x[:, n_q:n_q + n_kv])), (1, x[:, n_q + n_kv:].float())):
        codes, scale = _coded(y, case["code"])
        s["codes"].view(torch.uint8)[page, LAYER, i, :, at] = codes
        s["scale"][page, LAYER, i, :, at] = scale
    if case["code"] == "int8":
        _plain_read(s)
    return _stored(s)


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
    codes = s["codes"].view(torch.uint8)
    k, v = (_values(codes[:, LAYER, i][pages], s["scale"][:, LAYER, i][pages], case["code"]).permute(0, 2, 1, 3, 4).flatten(2, 3) for i in (0, 1))
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


def _own(s):
    from qwen_inference_engine_b200 import layers as L
    case = s["case"]
    n_q, n_kv, hd = HEADS[case["heads"]]
    if "pool" not in s:  # made once, as a program that serves keeps them beside its buffers
        s["pool"] = L.KvPool8.over(s["codes"], s["scale"])
        if case["op"] == "store":
            s["rope"] = L.Rope(s["frequencies"], factor=s["factor"], neighbours=case["pairs"] == "neighbours")
        if case["op"] == "attention":
            s["batch"] = L.Batch(s["table"], case["page"], s["codes"].shape[0], s["slots"].numel(), s["q"].shape[0], slots=s["slots"], q_start=s["q_start"], kv_len=s["kv_len"])
    if case["op"] == "store":
        q, k, v = s["qkv"].split([n_q * hd, n_kv * hd, n_kv * hd], 1)
        L.launch_rope_store8(q, k, v, s["q_out"], s["pool"], LAYER, s["pos"], s["row"], s["rope"], n_q)
        if case["code"] == "int8":
            L.launch_kv8_read(s["pool"], LAYER, s["row"], s["k"], s["v"])
        return _stored(s)
    if case["op"] == "read":
        L.launch_kv8_read(s["pool"], LAYER, s["row"], s["k"], s["v"])
        return {"k": s["k"], "v": s["v"]}
    L.launch_attn_batch8(s["q"], s["out"], s["pool"], LAYER, s["batch"], n_q, window=case["window"])
    return s["out"]


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    n_q, n_kv, hd = HEADS[case["heads"]]
    vector = hd + 1  # codes and a scale
    if case["op"] == "store":
        read = 2 * n_kv * 2 * hd if case["code"] == "int8" else 0  # (what was just written need not be fetched again)
        return {"bytes": case["tokens"] * ((4 * n_q + 4 * n_kv) * hd + 2 * n_kv * vector + read + 8), "flops": case["tokens"] * 3 * (n_q + n_kv) * case["rotated"]}
    if case["op"] == "read":
        return {"bytes": case["tokens"] * (2 * n_kv * (vector + 2 * hd) + 4), "flops": case["tokens"] * 2 * n_kv * hd}
    cached, new = _lengths(case)
    pairs = keys = 0
    for c, n in zip(cached, new):
        p = np.arange(c, c + n)
        low = np.maximum(0, p - case["window"] + 1) if case["window"] else 0 * p
        pairs, keys = pairs + int((p + 1 - low).sum()), keys + int(c + n - low[0])
    return {"bytes": 4 * int(new.sum()) * n_q * hd + 2 * keys * n_kv * vector, "flops": 4 * hd * n_q * pairs}


# ---------------------------------------------------------------- the definitions, in 64 bits
def _exact_values(codes, scale):
    """codes (as values of their type) and scale bytes"""
    return codes.double() * torch.exp2(scale.double() - 127)[..., None]


def _exact_codes(x, code):
    """(codes as values, powers of two) of vectors in 64 bits"""
    most = x.abs().amax(-1)
    p = torch.exp2(torch.ceil(torch.log2(most / MOST[code])))
    p = torch.where(most > MOST[code] * p, 2 * p, torch.where(most <= MOST[code] * p / 2, p / 2, p))  # (a logarithm next to a whole number)
    y = x / p[..., None]
    if code == "int8":
        return torch.round(y), p
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)  # of three bits behind the first, and of the smallest numbers
    return torch.round(y / step) * step, p


def exact(case, seed):
    s = prepare(case, seed)
    n_q, n_kv, hd = HEADS[case["heads"]]
    ps = case["page"]

    def rows(x):
        """a layer's [k|v][cache row][kv head][...] of the pool's order"""
        return x[:, LAYER].permute(1, 0, 3, 2, *range(4, x.dim() - 1)).reshape(2, -1, n_kv, *x.shape[5:])

    if case["op"] == "read":
        k, v = _exact_values(rows(s["codes"].double())[:, s["row"].long()], rows(s["scale"].double())[:, s["row"].long()])
        return {"k": k.flatten(1), "v": v.flatten(1)}
    if case["op"] == "store":
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
        new = [_exact_codes(x, case["code"]) for x in (turned(k), v)]
        if case["code"] == "int8":
            return {"q": turned(q).flatten(1), "k": (new[0][0] * new[0][1][..., None]).flatten(1), "v": (new[1][0] * new[1][1][..., None]).flatten(1)}
        codes, scale = s["codes"].double(), torch.exp2(s["scale"].double() - 127)
        for i in (0, 1):
            c, p = rows(codes), rows(scale)
            c[i, s["row"].long()], p[i, s["row"].long()] = new[i]
            codes[:, LAYER] = c.view(2, -1, ps, n_kv, hd).permute(1, 0, 3, 2, 4)
            scale[:, LAYER] = p.view(2, -1, ps, n_kv).permute(1, 0, 3, 2)
        return {"q": turned(q).flatten(1), "codes": codes, "scale": scale}
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    start, lens, slots = s["q_start"].tolist(), s["kv_len"].tolist(), s["slots"].tolist()
    for r in range(len(lens)):
        t0, t1, n = start[r], start[r + 1], lens[r]
        pages = s["table"][slots[r], :-(-n // ps)].long()
        kv = _exact_values(s["codes"].view(torch.uint8)[pages, LAYER].view(s["codes"].dtype), s["scale"][pages, LAYER]).permute(1, 2, 0, 3, 4).reshape(2, n_kv, -1, hd)[:, :, :n]
        p = torch.arange(n - (t1 - t0), n, device="cuda")[:, None]
        j = torch.arange(n, device="cuda")
        hidden = (j > p) | (j <= p - (case["window"] or n + 1))
        for h in range(n_q):
            g = h * n_kv // n_q
            x = s["q"][t0:t1, h * hd:(h + 1) * hd].double() @ kv[0, g].T / math.sqrt(hd)
            out[t0:t1, h * hd:(h + 1) * hd] = torch.softmax(x.masked_fill(hidden, float("-inf")), -1) @ kv[1, g]
    return out
