"""A cache in 8 bits in its plain form, in 64 bits (qie_kv8_view in include/qie_b200.h), for the tests of its operators."""
import numpy as np
import torch

import step_util as ref

DTYPES = {"e4m3": torch.float8_e4m3fn, "int8": torch.int8}
MOST = {"e4m3": 448.0, "int8": 127.0}


def coded(x, kind):
    """vectors x [..., hd] of numbers -> (their codes as numbers, scale bytes), both in float64 / int64"""
    x = x.double()
    most = x.abs().amax(-1)
    e = torch.ceil(torch.log2(most / MOST[kind]))
    e = torch.where(most > MOST[kind] * torch.exp2(e), e + 1, torch.where(most <= MOST[kind] * torch.exp2(e - 1), e - 1, e))  # (a logarithm next to a whole number)
    byte = torch.where(most == 0, 0, (e + 127).clamp(min=1)).long()
    y = torch.where(most[..., None] == 0, 0.0, x / torch.exp2(byte.double() - 127)[..., None])
    if kind == "int8":
        return y.round(), byte
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return (y / step).round() * step, byte


def as_bytes(codes, kind):
    return codes.float().to(DTYPES[kind]).view(torch.uint8)  # (the codes are numbers of the type)


def values(codes, byte, kind):
    """bytes of codes [..., hd] and of scales -> float64"""
    v = codes.view(DTYPES[kind]).double() * torch.where(byte == 0, 0.0, torch.exp2(byte.double() - 127))[..., None]
    return torch.where((byte == 255)[..., None], float("nan"), v)


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def rand(seed, *shape, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * scale


class Requests8:
    """requests of given (cached, new) lengths with keys and values in the pages of a pool whose other places hold any bytes, codes and scales that are no numbers among them"""

    def __init__(self, L, lens, nq, nkv, hd, ps, kind, seed=0, max_tokens=None, slots=True, spare=3, n_layers=2, spread=1.0):
        rs = np.random.default_rng(seed)
        self.lens, self.nq, self.hd, self.kind, n = lens, nq, hd, kind, len(lens)
        had = [-(-(c + m) // ps) for c, m in lens]
        ids = rs.permutation(sum(had) + spare)
        rows = rs.permutation(n + spare)[:n] if slots else np.arange(n)
        table = np.full((n + spare, max(had + [1]) + 2), 10 ** 6)
        shape = (len(ids), n_layers, 2, nkv, ps)
        g = torch.Generator("cuda").manual_seed(seed + 5)
        self.codes = torch.randint(0, 256, (*shape, hd), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
        self.scale = torch.randint(0, 256, shape, generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
        self.codes[..., ::7] = 0x7f
        self.scale[..., ::3] = 255
        self.kv_at, self.k, self.v, at = [], [], [], 0
        for i, (c, m) in enumerate(lens):
            mine = ids[at:at + had[i]]
            table[rows[i], :had[i]] = mine
            at += had[i]
            p = torch.arange(c + m, device="cuda")
            pg = torch.from_numpy(mine).cuda()[p // ps]
            self.kv_at.append((pg, p % ps))
            for j, to in ((0, self.k), (1, self.v)):
                x = rand(seed * 1000 + 2 * i + j, c + m, nkv, hd) * torch.exp2((rand(seed * 1000 + 2 * i + j + 500, c + m, nkv, 1) * spread).round().clamp(-2, 2) if spread <= 1 else
                                                                             (rand(seed * 1000 + 2 * i + j + 500, c + m, nkv, 1) * spread).round())
                codes, byte = coded(x, kind)
                b, s = as_bytes(codes, kind), byte.to(torch.uint8)
                self.codes[pg, n_layers - 1, j, :, p % ps], self.scale[pg, n_layers - 1, j, :, p % ps] = b, s
                to.append(values(b, byte, kind))
        self.start = np.concatenate([[0], np.cumsum([m for _, m in lens])]).astype(int)
        self.rows = int(self.start[-1]) if max_tokens is None else max_tokens
        self.q = rand(seed + 77, self.rows, nq * hd, scale=1.5).bfloat16()
        self.kv = L.KvPool8.over(self.codes.view(DTYPES[kind]), self.scale)
        self.layer = n_layers - 1
        self.batch = L.Batch(i32(table), ps, len(ids), n, self.rows, slots=i32(rows) if slots else None, q_start=i32(self.start), kv_len=i32([c + m for c, m in lens]))

    def attend(self, L, window=0, scale=0.0, fill=9.0):
        out = torch.full_like(self.q, fill)
        L.launch_attn_batch8(self.q, out, self.kv, self.layer, self.batch, self.nq, window=window, scale=scale)
        torch.cuda.synchronize()
        return out

    def check(self, out, window=0, scale=0.0, left=None, more=0.0):
        """`more`: of the mean of |v| under the weights, beside the bound of the file"""
        assert torch.isfinite(out[:self.start[-1]]).all()
        for i, (c, m) in enumerate(self.lens):
            if m:
                s = slice(self.start[i], self.start[i + 1])
                want, size = ref.attention(self.q[s].view(m, self.nq, self.hd), self.k[i], self.v[i], c, window, scale)
                tiny = 2.0 ** -31 * (c + m) * self.v[i].abs().max()
                d = (out[s].reshape(m, self.nq, self.hd).double() - want).abs() - 2.0 ** -8 * want.abs() - (2.0 ** -11 + 2.0 ** -9 + more) * size - tiny
                assert (d <= 0).all(), (i, c, m, float((d / size).max()))
        if left is not None:
            assert (out[self.start[-1]:] == left).all()


def attend(L, lens, nq, nkv, hd, ps, kind, window=0, scale=0.0, extra=0, **k):
    r = Requests8(L, lens, nq, nkv, hd, ps, kind, max_tokens=sum(m for _, m in lens) + extra, **k)
    out = r.attend(L, window, scale)
    r.check(out, window, scale, 9.0)
    return r, out
