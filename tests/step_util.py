"""Plain forms in 64 bits of the operators of a serving step (qie_batch in include/qie_b200.h), for their tests."""
import math

import numpy as np
import torch


def layout(cached, new, slots, table, ring, first, count, ps, max_tokens):
    """(q_start, kv_len, pos, slot, row, table, ring, {first, count}, status) of one step, one page and token after the other"""
    table, ring, n_pages = table.copy(), ring.copy(), len(ring)
    flags = missing = 0
    had, need, back = [], 0, 0
    for c, n, s in zip(cached, new, slots):
        if c < 0 or n < -1 or not 0 <= s < table.shape[0]:
            flags |= 8
            continue
        if c + max(n, 0) > table.shape[1] * ps:
            flags |= 2
            continue
        h = -(-c // ps)
        need += -(-(c + n) // ps) - h if n > 0 else 0
        back += h if n < 0 else 0
    ok = [c >= 0 and n >= -1 and 0 <= s < table.shape[0] and c + max(n, 0) <= table.shape[1] * ps for c, n, s in zip(cached, new, slots)]
    total = sum(max(n, 0) for n, o in zip(new, ok) if o)
    if not (0 <= first < n_pages and 0 <= count <= n_pages):
        flags |= 8
    elif need > count:
        flags, missing = flags | 1, need - count
    elif count + back > n_pages:
        flags |= 8
    if total > max_tokens:
        flags |= 4
    q_start, kv_len = np.zeros(len(cached) + 1, np.int64), np.zeros(len(cached), np.int64)
    pos, slot, row = (np.full(max_tokens, -1, np.int64) for _ in range(3))
    if flags:
        return q_start, kv_len, pos, slot, row, table, ring, (first, count), (flags, missing)
    taken = given = t = 0
    for i, (c, n, s) in enumerate(zip(cached, new, slots)):
        h = -(-c // ps)
        if n < 0:
            for j in range(h):
                ring[(first + count + given) % n_pages] = table[s, j]
                given += 1
        for p in range(c, c + max(n, 0)):
            if p % ps == 0:
                table[s, p // ps] = ring[(first + taken) % n_pages]
                taken += 1
            pos[t], slot[t], row[t] = p, s, table[s, p // ps] * ps + p % ps
            t += 1
        kv_len[i] = 0 if n < 0 else c + n
        q_start[i + 1] = t
    return q_start, kv_len, pos, slot, row, table, ring, ((first + taken) % n_pages, count - taken + given), (0, 0)


def rope(x, pos, freq, factor, neighbours):
    """x [n, heads, hd], in float64"""
    x, h = x.double(), len(freq)
    angle = pos.double()[:, None] * freq
    c, s = (factor * torch.cos(angle))[:, None], (factor * torch.sin(angle))[:, None]
    a, b = (x[..., 0:2 * h:2], x[..., 1:2 * h:2]) if neighbours else (x[..., :h], x[..., h:2 * h])
    u, w = a * c - b * s, b * c + a * s
    return torch.cat([torch.stack([u, w], -1).flatten(-2) if neighbours else torch.cat([u, w], -1), x[..., 2 * h:]], -1)


def attention(q, k, v, cached, window=0, scale=0.0):
    """rows q [n, nq, hd] at positions cached + i over k, v [len, nkv, hd] -> (out, the mean of |v| under the weights), in float64"""
    n, nq, hd = q.shape
    g = nq // k.shape[1]
    k, v = (x.double().repeat_interleave(g, 1).transpose(0, 1) for x in (k, v))
    s = q.double().transpose(0, 1) @ k.transpose(1, 2) * (scale or 1 / math.sqrt(hd))
    p = torch.arange(cached, cached + n, device=q.device)[:, None]
    j = torch.arange(k.shape[1], device=q.device)
    s = s.masked_fill((j > p) | (j <= p - (window or cached + n + 1)), float("-inf")).softmax(-1)
    return (s @ v).transpose(0, 1), (s @ v.abs()).transpose(0, 1)


def logits(x, tokens=(), generated=0, repetition=None, presence=None, frequency=None, bias=(), mask=None):
    """one row x [vocab] in float64; `generated`: the index from which tokens are generated ones; bias: (id, value) pairs; mask: bool [vocab]"""
    x, n = x.double().cpu().clone(), x.numel()
    for t in {t for t in tokens if 0 <= t < n}:
        if repetition is not None:
            x[t] = x[t] / repetition if x[t] > 0 else x[t] * repetition
        times = sum(1 for j, u in enumerate(tokens) if u == t and j >= generated)
        if times:
            x[t] -= (frequency or 0) * times + (presence or 0)
    for t, b in bias:
        if 0 <= t < n:
            x[t] += b
    if mask is not None:
        x[~mask] = float("-inf")
    return x
