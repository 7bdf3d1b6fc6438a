"""The operators of a serving step (csrc/batch_layout.cu, rope_store.cu, attn_batch.cu, logit_rules.cu) against their plain forms in 64 bits
(step_util.py), one by one and as a step in a captured graph whose lengths change.

Bounds: a rounding to bf16 is off by at most 2^-8 of the value, to fp32 by 2^-24.
Rotary positions: the turns' fraction, in 64-bit fixed point, is off by 2^-23.6 of a turn at 2^31 positions, 2^-21 of a radian; as fp32, in [-pi, pi], by three roundings of 2^-22.3 more; the
hardware's sine and cosine by 2^-21.2, the three fp32 operations by 2^-23 of |a| + |b|: 2^-18 of |a| + |b| holds them together.
Attention: weights are rounded to bf16 in the product with the values: 2^-8 of the mean of |v| under the weights.  Scores in fp32 are off by at most 128 * 2^-23 of
sum |q k| / sqrt(hd), below 2^6 here, so weights by 2^-10 of themselves, exponentials and sums by less: 2^-9 of that mean for all of it.
Logits: seven fp32 operations and as many additions as biases, each off by 2^-24 of at most |x| r + f n + p + sum |b|."""
import numpy as np
import pytest
import torch

import step_util as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from qwen_inference_engine_b200 import layers
    return layers


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def rand(seed, *shape, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator("cuda").manual_seed(seed), device="cuda") * scale


# ---------------------------------------------------------------- layout
def make_layout(rs, n, ps, most_len, most_new, over, spare_rows=3, slack=0):
    """requests of random lengths, `over` of them finished, and pages that are theirs or in a ring that starts anywhere"""
    cached = rs.integers(0, most_len + 1, n)
    new = rs.integers(0, most_new + 1, n)
    new[rs.permutation(n)[:over]] = -1
    slots = rs.permutation(n + spare_rows)[:n]
    had = -(-cached // ps)
    need = int((-(-(cached + np.maximum(new, 0)) // ps) - had).sum())
    ids = rs.permutation(int(had.sum()) + need + slack + 1)
    table = np.full((n + spare_rows, -(-(most_len + most_new) // ps) + 1), -7)
    at = 0
    for s, h in zip(slots, had):
        table[s, :h] = ids[at:at + h]
        at += h
    free = ids[at:at + need + slack]
    n_pages = len(ids)
    first = int(rs.integers(n_pages))
    ring = np.full(n_pages, -9)
    ring[(first + np.arange(len(free))) % n_pages] = free
    return dict(cached=cached, new=new, slots=slots, table=table, ring=ring, first=first, count=len(free))


def run_layout(L, d, ps, max_tokens, in_place=False, slots=True, steps=1):
    b = L.Batch(i32(d["table"]), ps, len(d["ring"]), len(d["cached"]), max_tokens, slots=i32(d["slots"]) if slots else None, cached=i32(d["cached"]), n_new=i32(d["new"]),
                free_ring=i32(d["ring"]), ring_in=i32([d["first"], d["count"]]),
                q_start=torch.full((len(d["cached"]) + 4,), 55, dtype=torch.int32, device="cuda"), pos=torch.full((max_tokens + 4,), 55, dtype=torch.int32, device="cuda"))
    if in_place:
        b.ring_out = b.ring_in
        b.view.ring_out = b.ring_in.data_ptr()
    for _ in range(steps):
        L.launch_batch_layout(b)
    torch.cuda.synchronize()
    assert (b.q_start[len(d["cached"]) + 1:] == 55).all() and (b.pos[max_tokens:] == 55).all()
    return b


def check_layout(b, d, want, max_tokens):
    n = len(d["cached"])
    names = ("q_start", "kv_len", "pos", "slot", "row", "block_table", "free_ring", "ring_out", "status")
    for name, w in zip(names, want):
        got = getattr(b, name)[:{"q_start": n + 1, "pos": max_tokens}.get(name, None)].cpu().numpy()
        assert np.array_equal(got, np.asarray(w)), name


@pytest.mark.parametrize("n,ps,most_len,most_new,over", [(1, 16, 700, 1, 0), (1, 1, 0, 1, 0), (3, 16, 100, 0, 1), (64, 16, 2048, 1, 0), (64, 16, 2048, 1, 64), (31, 4, 90, 40, 5),
                                                         (33, 3, 50, 7, 2), (300, 16, 4000, 100, 20), (1025, 64, 500, 3, 9), (200, 5, 3, 700, 1), (2, 16, 30000, 40000, 0),
                                                         (8192, 16, 40, 5, 400)])
@pytest.mark.parametrize("in_place", [False, True])
def test_layout(L, n, ps, most_len, most_new, over, in_place):
    d = make_layout(np.random.default_rng(n * 7 + ps), n, ps, most_len, most_new, over, slack=n % 3)
    for max_tokens in sorted({int(np.maximum(d["new"], 0).sum()), int(np.maximum(d["new"], 0).sum()) + 37}):
        want = ref.layout(d["cached"], d["new"], d["slots"], d["table"], d["ring"], d["first"], d["count"], ps, max_tokens)
        assert want[-1] == (0, 0)
        check_layout(run_layout(L, d, ps, max_tokens, in_place), d, want, max_tokens)


def test_layout_without_requests_and_slots(L):
    d = dict(cached=np.zeros(0, int), new=np.zeros(0, int), slots=np.zeros(0, int), table=np.zeros((1, 1), int), ring=np.arange(5), first=4, count=3)
    check_layout(run_layout(L, d, 16, 9), d, ref.layout(d["cached"], d["new"], d["slots"], d["table"], d["ring"], 4, 3, 16, 9), 9)
    d = make_layout(np.random.default_rng(0), 20, 16, 200, 30, 2)
    d["table"] = d["table"][d["slots"]]
    d["slots"] = np.arange(20)
    want = ref.layout(d["cached"], d["new"], d["slots"], d["table"], d["ring"], d["first"], d["count"], 16, 700)
    check_layout(run_layout(L, d, 16, 700, slots=False), d, want, 700)


def broken(name, d):
    top = d["table"].shape[1] * 16
    if name == "pages":
        d["count"] -= 1
    elif name == "no pages":
        d["count"] = 0
    elif name == "tokens":
        return -1
    elif name == "row":
        d["cached"][3], d["new"][3] = top, 1
    elif name == "row, far":
        d["cached"][3], d["new"][3] = 2 ** 31 - 1, 2 ** 31 - 1
    elif name == "slot":
        d["slots"][5] = len(d["table"])
    elif name == "slot below":
        d["slots"][5] = -1
    elif name == "cached":
        d["cached"][0] = -1
    elif name == "new":
        d["new"][7] = -2
    elif name == "first":
        d["first"] = len(d["ring"])
    elif name == "first below":
        d["first"] = -1
    elif name == "count":
        d["count"] = len(d["ring"]) + 1
    elif name == "count below":
        d["count"] = -1
    elif name == "ring overfull":
        d["count"] = len(d["ring"])
    return 0


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("name", ["pages", "no pages", "tokens", "row", "row, far", "slot", "slot below", "cached", "new", "first", "first below", "count", "count below", "ring overfull"])
def test_layout_all_or_nothing(L, name, in_place):
    d = make_layout(np.random.default_rng(5), 40, 16, 300, 20, 4)
    max_tokens = int(np.maximum(d["new"], 0).sum()) + broken(name, d)
    want = ref.layout(d["cached"], d["new"], d["slots"], d["table"], d["ring"], d["first"], d["count"], 16, max_tokens)
    flag = {"pages": 1, "no pages": 1, "tokens": 4, "row": 2, "row, far": 2}.get(name, 8)
    assert want[-1][0] & flag
    b = run_layout(L, d, 16, max_tokens, in_place)
    check_layout(b, d, want, max_tokens)


# ---------------------------------------------------------------- rotary positions
def placed(t, off, stride):
    """rows of t, `stride` apart, `off` elements behind a 256-byte boundary, with 77 between them"""
    buf = torch.full((off + t.shape[0] * stride + 8,), 77.0, dtype=t.dtype, device="cuda")
    v = buf[off:off + t.shape[0] * stride].view(t.shape[0], stride)[:, :t.shape[1]]
    v.copy_(t)
    return v, buf


def near(got, want, size):
    assert torch.isfinite(got).all()
    d = (got.double() - want).abs() - 2.0 ** -8 * want.abs()
    assert (d <= 2.0 ** -18 * size).all(), float((d / size).max())


ROPE = [(2, 1, 64, 64), (14, 2, 64, 32), (28, 4, 128, 128), (12, 2, 128, 50), (3, 3, 64, 2), (1, 1, 128, 64), (5, 1, 96, 80), (4, 2, 40, 16), (2, 2, 10, 6), (0, 2, 64, 64), (2, 1, 256, 256)]


@pytest.mark.parametrize("nq,nkv,hd,rot", ROPE)
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("n,off,more,far", [(1, 0, 0, 1), (7, 0, 8, 2 ** 31 - 1), (65, 3, 1, 5000), (300, 8, 16, 40000)])
def test_rope_store(L, nq, nkv, hd, rot, neighbours, n, off, more, far):
    rs = np.random.default_rng(nq * 100 + hd + rot + n)
    pages, ps = (n + 4) // 5 + 2, 5
    w, factor = L.Rope.frequencies(rot, 10000.0, "yarn", 2.0, 4096)
    freq = torch.from_numpy(w).cuda()
    pos = rs.integers(max(0, far - 60000), far + 1, n)
    row = rs.permutation(pages * ps)[:n]
    no_q, no_kv = rs.random(n) < 0.1, rs.random(n) < 0.1
    pos[no_q] = -1 - rs.integers(0, 5, int(no_q.sum()))
    row[no_kv] = rs.choice([-1, pages * ps, 2 ** 31 - 1], int(no_kv.sum()))
    pos_k = torch.from_numpy(pos).cuda()
    x = rand(n + hd, n, (nq + 2 * nkv) * hd).bfloat16()
    qkv, buf = placed(x, off, (nq + 2 * nkv) * hd + more)
    q, k, v = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
    out, out_buf = placed(torch.full((n, nq * hd), 5.0, dtype=torch.bfloat16, device="cuda"), off, nq * hd + more + 1 if nq else 1)
    pool = rand(1, pages, 2, 2, nkv, ps, hd).bfloat16()
    before, kept = pool.clone(), buf.clone()
    L.launch_rope_store(q, k, v, out, L.KvPool.over(pool), 1, i32(pos), i32(row), L.Rope(freq, factor, neighbours), nq)
    torch.cuda.synchronize()
    assert torch.equal(buf, kept)
    heads = x.view(n, -1, hd)
    want = ref.rope(heads, pos_k.clamp(min=0), freq, factor, neighbours)
    size = (heads.double().abs().amax((1, 2)) * 2 * factor)[:, None, None]
    yes = torch.from_numpy(~no_q).cuda()
    if nq:
        near(out.reshape(n, nq, hd)[yes], want[yes, :nq], size[yes])
        assert (out[~yes] == 5).all()
        assert (out_buf == 77).sum() >= out_buf.numel() - out.numel()
        assert torch.equal(out.reshape(n, nq, hd)[yes][..., rot:], heads[yes, :nq, rot:])
    put = torch.from_numpy(~no_kv).cuda()
    r = torch.from_numpy(row).cuda()[put]
    both = pool[r // ps, 1, :, :, r % ps]
    # (a token without a position stores what position that its angle's turns are: not defined)
    sure = put & yes
    near(pool[:, 1, 0].transpose(1, 2).reshape(-1, nkv, hd)[torch.from_numpy(row).cuda()[sure]], want[sure, nq:nq + nkv], size[sure])
    assert torch.equal(both[:, 1], heads[put, nq + nkv:])
    left = torch.ones(pages * ps, dtype=torch.bool, device="cuda")
    left[r] = False
    for i in (0, 1):
        assert torch.equal(pool[:, 1, i].transpose(1, 2).reshape(-1, nkv, hd)[left], before[:, 1, i].transpose(1, 2).reshape(-1, nkv, hd)[left])
    assert torch.equal(pool[:, 0], before[:, 0])


@pytest.mark.parametrize("heads,hd,rot", [(14, 64, 64), (3, 128, 30), (1, 72, 72), (2, 512, 512)])
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("off", [0, 1])
def test_rope_rows_in_place(L, heads, hd, rot, neighbours, off):
    n = 70
    freq = torch.from_numpy(L.Rope.frequencies(rot)[0]).cuda()
    x = rand(heads, n, heads * hd).bfloat16()
    y, buf = placed(x, off, heads * hd + 16)
    pos = torch.arange(n, device="cuda") * 977
    L.launch_rope_rows(y, y, pos.int(), L.Rope(freq, 1.0, neighbours), heads, hd)
    near(y.reshape(n, heads, hd), ref.rope(x.view(n, heads, hd), pos, freq, 1.0, neighbours), 2 * x.double().abs().max())
    assert (buf == 77).sum() >= buf.numel() - y.numel()


def test_rope_as_the_present_operator(L):
    """neighbours as pairs over the whole head: what qie_rope does with its table, as far as its fp32 angles go"""
    n, heads, hd = 40, 4, 64
    x = rand(3, n, heads * hd).bfloat16()
    cos, sin = L.precompute_cos_sin(n, hd)
    y, z = x.clone(), torch.empty_like(x)
    L.launch_rope(torch.from_numpy(cos).cuda(), torch.from_numpy(sin).cuda(), y, n, hd, heads * hd, heads)
    L.launch_rope_rows(x, z, torch.arange(n, dtype=torch.int32, device="cuda"), L.Rope(torch.from_numpy(L.Rope.frequencies(hd, 1e6)[0]).cuda(), 1.0, True), heads, hd)
    # the table's frequencies (powf) and angles are off by 2^-21 of up to 40 radians, and both results are rounded
    assert ((y.double() - z.double()).abs() <= 2.0 ** -7 * y.double().abs() + 2.0 ** -14 * x.double().abs().max()).all()


# ---------------------------------------------------------------- attention
class Requests:
    """requests of given (cached, new) lengths with keys and values in the pages of a pool that is NaN elsewhere"""

    def __init__(self, L, lens, nq, nkv, hd, ps, seed=0, max_tokens=None, slots=True, spare=3, n_layers=2):
        rs = np.random.default_rng(seed)
        self.lens, self.nq, self.hd, n = lens, nq, hd, len(lens)
        had = [-(-(c + m) // ps) for c, m in lens]
        ids = rs.permutation(sum(had) + spare)
        rows = rs.permutation(n + spare)[:n] if slots else np.arange(n)
        table = np.full((n + spare, max(had + [1]) + 2), 10 ** 6)
        self.pool = torch.full((len(ids), n_layers, 2, nkv, ps, hd), float("nan"), dtype=torch.bfloat16, device="cuda")
        self.k, self.v, at = [], [], 0
        for i, (c, m) in enumerate(lens):
            mine = ids[at:at + had[i]]
            table[rows[i], :had[i]] = mine
            at += had[i]
            k, v = (rand(seed * 1000 + 2 * i + j, c + m, nkv, hd).bfloat16() for j in (0, 1))
            self.k.append(k), self.v.append(v)
            p = torch.arange(c + m, device="cuda")
            pg = torch.from_numpy(mine).cuda()[p // ps]
            self.pool[pg, n_layers - 1, 0, :, p % ps], self.pool[pg, n_layers - 1, 1, :, p % ps] = k, v
        self.start = np.concatenate([[0], np.cumsum([m for _, m in lens])]).astype(int)
        self.rows = int(self.start[-1]) if max_tokens is None else max_tokens
        self.q = rand(seed + 77, self.rows, nq * hd, scale=1.5).bfloat16()
        self.kv = L.KvPool.over(self.pool)
        self.layer = n_layers - 1
        self.batch = L.Batch(i32(table), ps, len(ids), n, self.rows, slots=i32(rows) if slots else None, q_start=i32(self.start), kv_len=i32([c + m for c, m in lens]))

    def check(self, out, window=0, scale=0.0, left=None):
        assert torch.isfinite(out[:self.start[-1]]).all()
        for i, (c, m) in enumerate(self.lens):
            if m:
                s = slice(self.start[i], self.start[i + 1])
                want, size = ref.attention(self.q[s].view(m, self.nq, self.hd), self.k[i], self.v[i], c, window, scale)
                d = (out[s].reshape(m, self.nq, self.hd).double() - want).abs() - 2.0 ** -8 * want.abs() - (2.0 ** -8 + 2.0 ** -9) * size
                assert (d <= 0).all(), (i, c, m, float((d / size).max()))
        if left is not None:
            assert (out[self.start[-1]:] == left).all()


def attend(L, lens, nq, nkv, hd, ps, window=0, scale=0.0, extra=0, **k):
    r = Requests(L, lens, nq, nkv, hd, ps, max_tokens=sum(m for _, m in lens) + extra, **k)
    out = torch.full_like(r.q, 9.0)
    L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, nq, window=window, scale=scale)
    torch.cuda.synchronize()
    r.check(out, window, scale, 9.0)
    return r, out


HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (3, 3, 64), (1, 1, 128)]


@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("lens", [[(0, 1)], [(699, 1)], [(0, 63)], [(0, 64), (64, 64)], [(63, 2), (1, 0), (64, 1)], [(0, 300)], [(1000, 130)], [(129, 19), (5, 18), (127, 1)],
                                  [(i * 37 % 500, 1) for i in range(40)], [(2000, 1), (0, 500), (100, 3), (0, 1), (50, 0), (9, 77)], [(5000, 1), (1, 1)]])
def test_attention(L, nq, nkv, hd, lens):
    attend(L, lens, nq, nkv, hd, 16, extra=3, seed=len(lens))


@pytest.mark.parametrize("nq,nkv,hd", HEADS + [(16, 1, 128), (17, 1, 64), (16, 16, 64), (5, 1, 128), (9, 3, 128)])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("lens", [[(i * 97 % 1500, 1) for i in range(64)], [(0, 1)] * 3, [(500, 1), (77, 0), (0, 1), (64, 0), (63, 1)], [(300, 5), (10, 0), (9, 0), (8, 0), (6, 0)],
                                  [(4000, 3), (100, 0), (200, 0), (1, 1)], [(20000, 1)]])
def test_attention_no_more_rows_than_requests(L, nq, nkv, hd, window, lens):
    """decode steps, and steps with a few more rows for some requests and none for others"""
    attend(L, lens, nq, nkv, hd, 16, window=window, seed=len(lens) + nq)


@pytest.mark.parametrize("ps", [1, 2, 3, 4, 5, 8, 16, 24, 32, 48, 64, 100, 128, 256])
@pytest.mark.parametrize("nq,nkv,hd", [(14, 2, 64), (4, 1, 128)])
def test_attention_page_sizes(L, ps, nq, nkv, hd):
    attend(L, [(70, 40), (0, 1), (333, 1), (128, 70), (0, 0), (511, 1)], nq, nkv, hd, ps, seed=ps)


@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 200, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("nq,nkv,hd,ps", [(14, 2, 64, 16), (6, 2, 128, 4), (6, 2, 128, 64)])
def test_attention_window(L, window, nq, nkv, hd, ps):
    attend(L, [(0, 300), (700, 1), (64, 64), (513, 130), (0, 1), (2100, 1)], nq, nkv, hd, ps, window=window, seed=window % 1000)


@pytest.mark.parametrize("nq,nkv,hd", [(128, 1, 64), (100, 1, 128), (65, 1, 64), (64, 1, 128), (32, 2, 64), (43, 1, 128), (16, 16, 64)])
def test_attention_heads_of_a_group(L, nq, nkv, hd):
    attend(L, [(0, 5), (200, 1), (65, 33), (0, 130)], nq, nkv, hd, 16, seed=nq, extra=1)


@pytest.mark.parametrize("scale", [0.01, 0.3])
def test_attention_scale(L, scale):
    attend(L, [(10, 90), (300, 1)], 14, 2, 64, 16, scale=scale)


def test_attention_strides_and_plain_slots(L):
    lens = [(100, 30), (0, 1), (64, 65)]
    r = Requests(L, lens, 14, 2, 64, 16, slots=False, seed=3)
    wide = torch.full((r.rows, 14 * 64 + 40), float("nan"), dtype=torch.bfloat16, device="cuda")
    q, out = wide[:, 8:8 + 14 * 64], torch.full((r.rows, 14 * 64 + 16), 9.0, dtype=torch.bfloat16, device="cuda")
    q.copy_(r.q)
    L.launch_attn_batch(q, out[:, :14 * 64], r.kv, r.layer, r.batch, 14)
    r.check(out[:, :14 * 64])
    assert (out[:, 14 * 64:] == 9).all()


def test_attention_many_requests(L):
    rs = np.random.default_rng(1)
    attend(L, [(int(c), int(m)) for c, m in zip(rs.integers(0, 200, 700), rs.integers(0, 4, 700))], 4, 2, 64, 16, seed=9)


def test_attention_long(L):
    """one row behind many positions beside short ones, and a long prompt: the split over the positions"""
    attend(L, [(40000, 1), (3, 2)], 14, 2, 64, 16, seed=2)
    attend(L, [(0, 2500), (7000, 600)], 7, 1, 128, 16, seed=4)


def test_attention_values_behind_the_weights(L):
    """large scores: the largest weight is one and the others vanish; and rows whose keys are all alike"""
    r = Requests(L, [(300, 70), (900, 1)], 4, 2, 128, 16, seed=5)
    r.q.mul_(30)
    out = torch.empty_like(r.q)
    L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 4)
    # scores are 30 times as large and their fp32 errors with them: weights off by 2^-5 of themselves, the mean of |v| by the bound's 2^-9 plus that
    for i, (c, m) in enumerate(r.lens):
        s = slice(r.start[i], r.start[i + 1])
        want, size = ref.attention(r.q[s].view(m, 4, 128), r.k[i], r.v[i], c)
        assert ((out[s].reshape(m, 4, 128).double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -4 * size).all()
    r.q.zero_()
    L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 4)
    r.check(out)


def test_attention_infinite_values(L):
    """an infinity among the values comes out where a row sees it, and nowhere else"""
    r = Requests(L, [(0, 100), (70, 1)], 2, 1, 64, 16, seed=6)
    page = int(r.batch.block_table[r.batch.slots[0], 3])
    r.pool[page, r.layer, 1, 0, 2, 5] = float("inf")  # position 50 of the first request
    out = torch.empty_like(r.q)
    L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 2)
    o = out.view(101, 2, 64)
    assert torch.isinf(o[50:100, :, 5]).all()
    o = o.clone()
    o[50:100, :, 5] = 0
    assert torch.isfinite(o).all()


def test_attention_same_bits_again(L):
    r, out = attend(L, [(3000, 1), (0, 700), (10, 5)], 14, 2, 64, 16, seed=8)
    for _ in range(3):
        r.batch.work.random_(0, 255)  # whatever an earlier call left in the work area
        again = torch.full_like(out, 9.0)
        L.launch_attn_batch(r.q, again, r.kv, r.layer, r.batch, 14)
        assert torch.equal(again, out)


def test_attention_two_streams(L):
    """two calls at once, each with a work area of its own"""
    a = [Requests(L, [(1500 + 100 * i, 1), (0, 400), (33, 2)], 14, 2, 64, 16, seed=20 + i) for i in range(2)]
    outs = [torch.full_like(r.q, 9.0) for r in a]
    streams = [torch.cuda.Stream() for _ in a]
    for r in a:
        r.batch.reserve(r.kv, 14)
    torch.cuda.synchronize()
    for _ in range(5):
        for r, o, s in zip(a, outs, streams):
            with torch.cuda.stream(s):
                L.launch_attn_batch(r.q, o, r.kv, r.layer, r.batch, 14)
    torch.cuda.synchronize()
    for r, o in zip(a, outs):
        r.check(o)


def test_attention_nonsense_stays_inside(L):
    """offsets, lengths, slots and pages that make no sense: nothing is read or written outside, and requests beside them keep their results"""
    r = Requests(L, [(100, 10), (50, 20), (300, 1), (7, 5)], 14, 2, 64, 16, seed=11)
    out = torch.full_like(r.q, 9.0)
    kv_len, slots, table = r.batch.kv_len.clone(), r.batch.slots.clone(), r.batch.block_table.clone()
    r.batch.kv_len[1] = 2 ** 31 - 1
    r.batch.block_table[slots[1]] = i32([-5])
    r.batch.block_table[slots[1], 1] = 2 ** 31 - 1
    L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 14)
    good = torch.ones(36, dtype=torch.bool, device="cuda")
    good[10:30] = False
    want = torch.full_like(r.q, 9.0)
    r.batch.kv_len.copy_(kv_len), r.batch.block_table.copy_(table)
    L.launch_attn_batch(r.q, want, r.kv, r.layer, r.batch, 14)
    r.check(want)
    # the split over the positions may fall elsewhere: two results within their bounds
    assert ((out[good].double() - want[good].double()).abs() <= 2.0 ** -6 * 5).all()
    for bad in (-1, 10 ** 6, -2 ** 31):
        r.batch.slots[1] = bad
        out.fill_(9.0)
        L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 14)
        assert (out[10:30] == 9).all() and torch.isfinite(out).all()
    r.batch.slots.copy_(slots)
    for start in ([0, 10, 30, 31, 2 ** 31 - 1], [0, -50, 30, 31, 36], [36, 31, 30, 10, 0], [2 ** 31 - 1] * 5, [-2 ** 31, 2 ** 31 - 1, 0, 0, 0]):
        r.batch.q_start.copy_(i32(start))
        L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 14)
    for n in (-2 ** 31, -1, 0):
        r.batch.q_start.copy_(i32(r.start))
        r.batch.kv_len.fill_(n)
        L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 14)
    torch.cuda.synchronize()
    r.batch.kv_len.copy_(kv_len)
    L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 14)
    r.check(out)


@pytest.mark.parametrize("ps", [16, 4])
def test_offsets_beyond_32_bits(L, ps):
    """a pool of more than 2^31 elements: store and attention at its end"""
    pages = (2 ** 31 // (2 * ps * 128)) + 300
    pool = torch.empty(pages, 1, 2, 1, ps, 128, dtype=torch.bfloat16, device="cuda")
    n, g = 200, 4
    mine = torch.arange(pages - 1, pages - 1 - (n + ps - 1) // ps, -1, dtype=torch.int32, device="cuda")
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    row = mine[(pos // ps).long()] * ps + pos % ps
    qkv = rand(1, n, (g + 2) * 128).bfloat16()
    q, k, v = qkv.split([g * 128, 128, 128], 1)
    q_out, out, freq = torch.empty_like(q.contiguous()), torch.empty_like(q.contiguous()), torch.from_numpy(L.Rope.frequencies(128)[0]).cuda()
    kv = L.KvPool.over(pool)
    L.launch_rope_store(q, k, v, q_out, kv, 0, pos, row, L.Rope(freq), g)
    batch = L.Batch(mine[None].contiguous(), ps, pages, 1, n, q_start=i32([0, n]), kv_len=i32([n]))
    L.launch_attn_batch(q_out, out, kv, 0, batch, g)
    turned = ref.rope(qkv.view(n, g + 2, 128), pos.long(), freq, 1.0, False)
    near(q_out.view(n, g, 128), turned[:, :g], 2 * qkv.double().abs().max())
    stored = pool[:, 0, 0, 0][mine.long()].reshape(-1, 128)[:n]
    assert torch.equal(pool[:, 0, 1, 0][mine.long()].reshape(-1, 128)[:n], v)
    want, size = ref.attention(q_out.view(n, g, 128), stored[:, None], v[:, None], 0)
    assert ((out.view(n, g, 128).double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -8 + 2.0 ** -9) * size).all()


def test_attention_refuses_a_small_work_area(L):
    from qwen_inference_engine_b200._lib import QieError
    r = Requests(L, [(10, 1)], 2, 1, 64, 16)
    r.batch.reserve(r.kv, 2)
    n, r.batch.view.work_bytes = r.batch.view.work_bytes, r.batch.view.work_bytes - 1
    with pytest.raises(QieError) as e:
        L.launch_attn_batch(r.q, torch.empty_like(r.q), r.kv, r.layer, r.batch, 2)
    assert e.value.code == -1 and "work area" in str(e.value)
    r.batch.view.work_bytes = n
    out = torch.empty_like(r.q)
    L.launch_attn_batch(r.q, out, r.kv, r.layer, r.batch, 2)
    r.check(out)


def test_python_forms_refuse(L):
    """types, shapes, strides and devices that the Python forms turn away"""
    x, pos, freq = rand(1, 4, 128).bfloat16(), i32([0, 1, 2, 3]), torch.ones(32, dtype=torch.float64, device="cuda")
    rope, pool = L.Rope(freq), L.KvPool.over(torch.zeros(3, 1, 2, 1, 16, 64, dtype=torch.bfloat16, device="cuda"))
    table, k = i32([[0, 1, 2]]), rand(2, 4, 64).bfloat16()
    batch = L.Batch(table, 16, 3, 1, 4, q_start=i32([0, 4]), kv_len=i32([4]))
    for call in (lambda: L.launch_rope_rows(x.float(), x.float(), pos, rope, 2, 64), lambda: L.launch_rope_rows(x, x, pos[:3], rope, 2, 64),
                 lambda: L.launch_rope_rows(x, x, pos, rope, 3, 64), lambda: L.launch_rope_rows(x.T.contiguous().T, x, pos, rope, 2, 64),
                 lambda: L.launch_rope_rows(x.cpu(), x.cpu(), pos, rope, 2, 64), lambda: L.launch_rope_rows(x, x, pos.long(), rope, 2, 64),
                 lambda: L.launch_rope_store(x, k, k[:3], x, pool, 0, pos, pos, rope, 2), lambda: L.launch_rope_store(x, k, k.cpu(), x, pool, 0, pos, pos, rope, 2),
                 lambda: L.launch_rope_store(x, k, k, x, pool, 0, pos, pos.cpu(), rope, 2), lambda: L.launch_rope_store(x, x, k, x, pool, 0, pos, pos, rope, 2),
                 lambda: L.launch_attn_batch(x[:3], x[:3].clone(), pool, 0, batch, 2), lambda: L.launch_attn_batch(x, x.float(), pool, 0, batch, 2),
                 lambda: L.launch_attn_batch(x, x.cpu(), pool, 0, batch, 2), lambda: L.Rope(freq.float()), lambda: L.Batch(table.long(), 16, 3, 1, 4),
                 lambda: L.Batch(table, 16, 3, 2, 4, kv_len=i32([1])), lambda: L.Batch(table, 16, 3, 1, 4, cached=i32([1]).cpu()), lambda: L.KvPool.over(k),
                 lambda: L.launch_logits(x, x.float(), L.LogitRules()), lambda: L.launch_logits(x.half(), x.half(), L.LogitRules()),
                 lambda: L.launch_logits(x, x, L.LogitRules(i32([0, 0]), pos)), lambda: L.LogitRules(i32([0, 1]).long(), pos), lambda: L.LogitRules(bias_start=i32([0, 1]), bias=freq.float()),
                 lambda: L.LogitRules(mask=pos)):
        with pytest.raises((AssertionError, ValueError)):
            call()


# ---------------------------------------------------------------- logits
def ragged(rs, rows, most, vocab, wild=True):
    lens = rs.integers(0, most + 1, rows)
    start = np.concatenate([[0], np.cumsum(lens)])
    t = (vocab * rs.random(int(start[-1])) ** 3).astype(np.int64)
    if wild and len(t):
        at = rs.random(len(t)) < 0.03
        t[at] = rs.choice([-1, vocab, -2 ** 31, 2 ** 31 - 1, vocab + 31], int(at.sum()))
    return start, t


RULES = ("repetition", "presence", "frequency", "bias", "mask")


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,most,off,more", [(1, 7, 3, 0, 0), (3, 512, 40, 1, 5), (2, 4096, 0, 0, 0), (5, 4097, 300, 0, 7), (2, 151936, 3000, 0, 0), (4, 33333, 700, 3, 2), (70, 2048, 60, 0, 0)])
@pytest.mark.parametrize("rules", [RULES, ("repetition",), ("presence",), ("frequency", "mask"), ("bias",), ("mask",), ()])
@pytest.mark.parametrize("in_place", [False, True])
def test_logits(L, dtype, rows, vocab, most, off, more, rules, in_place):
    rs = np.random.default_rng(rows * 1000 + vocab + len(rules))
    x = rand(vocab, rows, vocab, scale=4.0).to(dtype)
    at = torch.from_numpy(rs.random((rows, vocab)) < 0.01).cuda()
    x[at] = torch.tensor(rs.choice([0.0, -0.0, float("inf"), float("-inf"), float("nan"), 1e-38, -1e30], int(at.sum())), dtype=dtype, device="cuda")
    logits, buf = placed(x, off, vocab + more)
    start, tokens = ragged(rs, rows, most, vocab)
    gen = start[:-1] + ((start[1:] - start[:-1]) * rs.random(rows)).astype(int)
    bias_start, bias_ids = ragged(rs, rows, 60, vocab)
    bias = rs.uniform(-6, 6, len(bias_ids)).astype(np.float32)
    p = {k: rs.uniform(lo, hi, rows).astype(np.float32) for k, lo, hi in (("repetition", 0.7, 1.6), ("presence", -1, 1), ("frequency", 0, 0.5))}
    mask_rows = rs.choice([-1, 0, 1, 2, 3, 99], rows)
    words = (vocab + 31) // 32 + rows % 2
    mask = rs.integers(0, 2 ** 32, (4, words), dtype=np.uint64).astype(np.uint32)
    mask[3] = 0  # a row of which nothing is left
    lists = dict(tok_start=i32(start), tokens=i32(tokens), gen_start=i32(gen)) if any(k in rules for k in p) else {}
    k = {**lists, **{n: torch.from_numpy(p[n]).cuda() for n in p if n in rules}}
    if "bias" in rules:
        k.update(bias_start=i32(bias_start), bias_ids=i32(bias_ids), bias=torch.from_numpy(bias).cuda())
    if "mask" in rules:
        k.update(mask=torch.from_numpy(mask.view(np.int32)).cuda(), mask_row=i32(mask_rows))
    out, out_buf = (logits, buf) if in_place else placed(torch.zeros_like(x), off + 2, vocab + more + 3)
    L.launch_logits(logits, out, L.LogitRules(**k))
    torch.cuda.synchronize()
    assert (out_buf == 77).sum() >= out_buf.numel() - out.numel()
    if not in_place:
        assert torch.equal(logits.nan_to_num(123), x.nan_to_num(123))
    eps = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -24
    for i in range(rows):
        t, b = tokens[start[i]:start[i + 1]].tolist(), slice(bias_start[i], bias_start[i + 1])
        allowed = None
        if "mask" in rules and 0 <= mask_rows[i] < 4:
            allowed = torch.from_numpy(np.unpackbits(mask[mask_rows[i]].view(np.uint8), bitorder="little")[:vocab].astype(bool))
        args = {n: float(p[n][i]) for n in p if n in rules}
        pairs = list(zip(bias_ids[b].tolist(), bias[b].tolist())) if "bias" in rules else []
        want = ref.logits(x[i], t if lists else (), int(gen[i] - start[i]), **args, bias=pairs, mask=allowed)
        got = out[i].double().cpu()
        fine = torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got[~fine].nan_to_num(5), want[~fine].nan_to_num(5)), i
        size = x[i].double().cpu().abs() * 1.6 + 0.5 * len(t) + 1 + sum(abs(v) for _, v in pairs)
        d = (got - want).abs()[fine] - eps * want.abs()[fine]
        assert (d <= (7 + len(pairs)) * 2.0 ** -24 * size[fine]).all(), (i, float(d.max()))


def test_logits_as_the_present_operator(L):
    """the repetition penalty alone: the bits of qie_repetition_penalty"""
    x = rand(4, 1, 5000, scale=4.0).bfloat16()
    tokens = torch.randint(-3, 5100, (900,), dtype=torch.int32, device="cuda")
    y, z = x.clone(), x.clone()
    L.apply_repetition_penalty(y, tokens, 5000, 1.3)
    L.launch_logits(z, z, L.LogitRules(i32([0, 900]), tokens, repetition=torch.tensor([1.3], device="cuda")))
    assert torch.equal(y, z)


def test_logits_many_biases_of_one_token(L):
    """entries of one token add up in the order of the list, every time"""
    rs = np.random.default_rng(2)
    ids, b = np.full(500, 77), rs.uniform(-1e3, 1e3, 500).astype(np.float32)
    ids[::7] = rs.integers(0, 200, len(ids[::7]))
    x = rand(1, 1, 200)
    rules = L.LogitRules(bias_start=i32([0, 500]), bias_ids=i32(ids), bias=torch.from_numpy(b).cuda())
    want = np.float32(0)
    for i, v in zip(ids, b):
        if i == 77:
            want = np.float32(want + v)
    for _ in range(4):
        out = torch.empty_like(x)
        L.launch_logits(x, out, rules)
        assert out[0, 77].item() == np.float32(x[0, 77].item() + want)


def test_logits_nonsense_stays_inside(L):
    x = rand(1, 3, 1000)
    for start in ([0, 2 ** 31 - 1, -5, 50], [-2 ** 31, -1, 2 ** 31 - 1, 0], [40, 30, 20, 10]):
        t = torch.randint(0, 1000, (50,), dtype=torch.int32, device="cuda")
        one = torch.ones(3, device="cuda")
        out = torch.empty_like(x)
        L.launch_logits(x, out, L.LogitRules(i32(start), t, gen_start=i32([-2 ** 31, 5, 2 ** 31 - 1]), repetition=one, presence=one, bias_start=i32(start), bias_ids=t,
                                             bias=torch.ones(50, device="cuda")))
        assert torch.isfinite(out).all()


def test_logits_mask_of_each_row(L):
    x = rand(1, 3, 100)
    mask = i32([[1, 0, 0, 0], [0, 2, 0, 0], [0, 0, 0, 8]])
    out = torch.empty_like(x)
    L.launch_logits(x, out, L.LogitRules(mask=mask))
    want = torch.full_like(x, float("-inf"))
    for r, t in ((0, 0), (1, 33), (2, 99)):
        want[r, t] = x[r, t]
    assert torch.equal(out, want)


# ---------------------------------------------------------------- a step
def test_a_step_in_a_graph(L):
    """layout, positions and store, attention, rules and the sampler, captured once and replayed for steps of other lengths: prompts in portions beside sequences that
    decode, one that is over and its pages with another request"""
    nq, nkv, hd, ps, n, rows, vocab = 6, 2, 64, 16, 5, 48, 500
    rs = np.random.default_rng(0)
    n_pages, max_pages = 40, 20
    g = dict(dtype=torch.int32, device="cuda")
    first = 17
    ring = (rs.permutation(n_pages))
    state = torch.tensor([first, n_pages], **g)
    batch = L.Batch(torch.full((n, max_pages), -3, **g), ps, n_pages, n, rows, cached=torch.zeros(n, **g), n_new=torch.zeros(n, **g), free_ring=i32(ring), ring_in=state, ring_out=state)
    pool = L.KvPool.over(torch.full((n_pages, 2, 2, nkv, ps, hd), float("nan"), dtype=torch.bfloat16, device="cuda"), batch.block_table)
    batch.reserve(pool, nq)
    w, f = L.Rope.frequencies(hd, 10000.0, "parts", 8.0, 64)
    freq = torch.from_numpy(w).cuda()
    rope = L.Rope(freq, f)
    qkv = torch.zeros(rows, (nq + 2 * nkv) * hd, dtype=torch.bfloat16, device="cuda")
    q, k, v = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
    q_out, out = torch.zeros(rows, nq * hd, dtype=torch.bfloat16, device="cuda"), torch.full((rows, nq * hd), 9.0, dtype=torch.bfloat16, device="cuda")
    logits, tokens = rand(3, n, vocab, scale=3.0).bfloat16(), torch.zeros(n, **g)
    mask = torch.zeros(n, 16, **g)
    for i in range(n):
        mask[i, i] = 1 << (3 * i)  # one token is left
    rules = L.LogitRules(mask=mask)
    ruled = torch.empty_like(logits)
    from qwen_inference_engine_b200 import _lib

    def step():
        L.launch_batch_layout(batch)
        L.launch_rope_store(q, k, v, q_out, pool, 1, batch.pos, batch.row, rope, nq)
        L.launch_attn_batch(q_out, out, pool, 1, batch, nq)
        L.launch_logits(logits, ruled, rules)
        _lib.check(_lib.lib().qie_sample_topk(ruled.data_ptr(), tokens.data_ptr(), n, vocab, 1.0, 1, 1, 0, L._st()))

    step()  # nothing to do: every request has no token
    torch.cuda.synchronize()
    assert (out == 9).all()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    cached, keys, values = [0] * n, [None] * n, [None] * n
    plan = [[30, 0, 10, 0, 1], [1, 1, 20, 0, 1], [1, 40, 1, 5, 1], [-1, 1, 1, 1, 40], [0, 1, 17, 17, 1], [45, 1, 1, 0, -1], [1, 1, -1, 1, 0], [1, 1, 44, 1, 0]]
    for s, new in enumerate(plan):
        x = rand(100 + s, rows, (nq + 2 * nkv) * hd).bfloat16()
        qkv.copy_(x)
        out.fill_(9.0)
        batch.cached.copy_(i32(cached)), batch.n_new.copy_(i32(new))
        graph.replay()
        torch.cuda.synchronize()
        assert batch.status.tolist() == [0, 0] and tokens.tolist() == [32 * i + 3 * i for i in range(n)]
        at = 0
        heads = x.view(rows, -1, hd)
        for i, m in enumerate(new):
            if m < 0:
                cached[i], keys[i], values[i] = 0, None, None
                continue
            if not m:
                continue
            part, pos = heads[at:at + m], torch.arange(cached[i], cached[i] + m, device="cuda")
            turned = ref.rope(part, pos, freq, f, False).bfloat16()
            # (the cache's own rounding of the keys is the operator's; where it falls on the other side of a border both are within its bound)
            keys[i] = turned[:, nq:nq + nkv] if keys[i] is None else torch.cat([keys[i], turned[:, nq:nq + nkv]])
            values[i] = part[:, nq + nkv:] if values[i] is None else torch.cat([values[i], part[:, nq + nkv:]])
            want, size = ref.attention(turned[:, :nq], keys[i], values[i], cached[i])
            d = (out[at:at + m].view(m, nq, hd).double() - want).abs() - 2.0 ** -8 * want.abs() - (2.0 ** -8 + 2.0 ** -8) * size
            assert (d <= 0).all(), (s, i, float(d.max()))
            cached[i] += m
            at += m
        assert (out[at:] == 9).all()
        held = sum(-(-c // ps) for c in cached)
        assert state[1].item() == n_pages - held
        ids = torch.cat([batch.block_table[i, :-(-c // ps)] for i, c in enumerate(cached)] + [batch.free_ring[(state[0] + torch.arange(n_pages - held, device="cuda")) % n_pages]])
        assert sorted(ids.tolist()) == list(range(n_pages))  # no page lost, none twice


def test_operators_take_the_current_stream(L):
    """each on a stream of its own, behind work that is still running there"""
    s = torch.cuda.Stream()
    x = torch.zeros(64, 64, dtype=torch.bfloat16, device="cuda")
    freq = torch.zeros(32, dtype=torch.float64, device="cuda")
    rope, pos, logits, out = L.Rope(freq, 2.0), torch.zeros(64, dtype=torch.int32, device="cuda"), torch.zeros(4, 900, device="cuda"), torch.empty(4, 900, device="cuda")
    y = torch.empty_like(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        torch.cuda._sleep(20_000_000)
        x.fill_(1.0), logits.fill_(3.0)
        L.launch_rope_rows(x, y, pos, rope, 1, 64)
        L.launch_logits(logits, out, L.LogitRules())
    s.synchronize()
    assert (y == 2).all() and (out == 3).all()
