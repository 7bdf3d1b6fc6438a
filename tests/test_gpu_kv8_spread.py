"""Attention over a cache in 8 bits where scales lie far apart: a row's result hangs on the keys and values that it sees, each by its own scale, and on nothing beside them.

Bound, of each column of a row's result.  Weights and their sums are fp32 of scores in fp32: 2^-9 of sum w |v| for scores below 2^6 (derived in test_gpu_kv8.py); a weight is rounded to fp16 in the
product, 2^-11 of itself.  It is there by 2^7 and its value's scale s beside the row's largest w s, of which the reference is at most twice as much (blocks of few rows) or 2^9 times (larger
blocks: a tile's largest weight and largest scale, which are one another's within 2^8, and a whole number): below 2^-14 it is off by 2^-25, so by 2^-32 of the reference, times the code beside it, at
most 448: of n keys n * 448 * 2^-31 (2^-23) of the largest w s.  The result is rounded to bf16, 2^-8 of itself."""
import numpy as np
import pytest
import torch

from kv8_util import DTYPES, Requests8, i32, values

pytestmark = pytest.mark.gpu
KINDS = ["e4m3", "int8"]
# (cached, new) of requests, query heads, kv heads; room for more rows than requests: blocks of few rows, and larger ones
FEW = [([(300, 3), (70, 8), (40, 1)], 2, 2), ([(200, 2), (9, 1)], 14, 2), ([(90, 1), (50, 1)], 16, 1)]
MANY = [([(300, 100), (9, 1)], 4, 2), ([(100, 333)], 14, 2)]


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from qwen_inference_engine_b200 import layers
    return layers


@pytest.fixture(scope="module", autouse=True)
def no_wait_ran_out(L):
    from qwen_inference_engine_b200 import _lib
    _lib.lib().qie_kernel_status()
    yield
    torch.cuda.synchronize()
    assert _lib.lib().qie_kernel_status() == 0


def scaled(r, i, pos, j, byte):
    """scale bytes into position pos of request i's keys (j 0) or values (1), all kv heads, and what they stand for"""
    pg, at = int(r.kv_at[i][0][pos]), int(r.kv_at[i][1][pos])
    r.scale[pg, r.layer, j, :, at] = torch.as_tensor(byte, device="cuda").to(torch.uint8)
    (r.k, r.v)[j][i][pos] = values(r.codes[pg, r.layer, j, :, at], r.scale[pg, r.layer, j, :, at].int(), r.kind)


def raised(r, i, pos, j, d):
    pg, at = int(r.kv_at[i][0][pos]), int(r.kv_at[i][1][pos])
    scaled(r, i, pos, j, r.scale[pg, r.layer, j, :, at].int() + d)


def scales_of(r, i, j):
    pg, at = r.kv_at[i]
    b = r.scale[pg, r.layer, j, :, at].double()
    return torch.where((b == 0) | (b == 255), 0.0, torch.exp2(b - 127))


def check(r, i, out, few, window=0, rows=None):
    """request i's rows (those of `rows`) against the formula in 64 bits over the positions that each of them sees"""
    c, m = r.lens[i]
    n, g = c + m, r.nq // r.kv_heads
    q = r.q[r.start[i]:r.start[i + 1]].view(m, r.nq, r.hd).double()
    got = out[r.start[i]:r.start[i + 1]].view(m, r.nq, r.hd).double()
    k, v, s = (t.repeat_interleave(g, 1) for t in (r.k[i], r.v[i], scales_of(r, i, 1)))  # [position][query head]...
    x = torch.einsum("mhd,nhd->hmn", q, torch.nan_to_num(k, nan=0.0)) * r.hd ** -0.5
    p, j = torch.arange(c, n, device="cuda")[:, None], torch.arange(n, device="cuda")
    hidden = (j > p) | ((j <= p - window) if window else (j < 0))
    x = x.masked_fill(hidden, float("-inf"))
    rows = torch.ones(m, dtype=torch.bool, device="cuda") if rows is None else rows
    assert rows.any() and (x[:, rows].amax(-1) < 64).all()  # (scores far below: weights of zero)
    w = torch.softmax(x, -1)
    clean = torch.nan_to_num(v, nan=0.0)
    want, size = torch.einsum("hmn,nhd->mhd", w, clean), torch.einsum("hmn,nhd->mhd", w, clean.abs())
    most = (w * s.T[:, None]).amax(-1).T[..., None]  # [row][head][1]
    tiny = n * 448 * 2.0 ** (-31 if few else -23) * most
    d = (got - want).abs() - 2.0 ** -8 * want.abs() - (2.0 ** -11 + 2.0 ** -9) * size - tiny
    assert torch.isfinite(got[rows]).all() and (d[rows] <= 0).all(), (i, float((d / size)[rows].max()))


def requests(L, lens, nq, nkv, hd, kind, room=4, ps=16, **k):
    r = Requests8(L, lens, nq, nkv, hd, ps, kind, max_tokens=sum(m for _, m in lens) + room, **k)
    r.kv_heads = nkv
    return r


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("j", [0, 1])
@pytest.mark.parametrize("d", [9, 15, 16, 20, 24, 25, 40])
@pytest.mark.parametrize("few,case", [(True, c) for c in FEW[:2]] + [(False, c) for c in MANY])
def test_tokens_that_a_row_does_not_see(L, kind, hd, j, d, few, case):
    """a later token's key or value 2^d times as large: the rows before it are those of the formula over what they see"""
    lens, nq, nkv = case
    r = requests(L, lens, nq, nkv, hd, kind, seed=d)
    for at in (sum(lens[0]) - 1, lens[0][0] + 1):  # (the last one, and one in the middle of the larger blocks' diagonal)
        if at > lens[0][0]:
            raised(r, 0, at, j, d)
    out = r.attend(L)
    rows = torch.arange(lens[0][1], device="cuda") < 1
    check(r, 0, out, few, rows=rows)
    for i in range(1, len(lens)):
        check(r, i, out, few)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("j", [0, 1])
@pytest.mark.parametrize("d", [15, 25, 40])
@pytest.mark.parametrize("few,lens,nq,nkv,window,at", [(True, [(200, 8), (9, 1)], 2, 2, 50, 152), (False, [(200, 200)], 4, 2, 70, 140), (False, [(0, 300)], 14, 2, 30, 100)])
def test_tokens_behind_the_window(L, kind, j, d, few, lens, nq, nkv, window, at):
    r = requests(L, lens, nq, nkv, 64, kind, seed=d + 1)
    raised(r, 0, at, j, d)
    p = torch.arange(lens[0][0], sum(lens[0]), device="cuda")
    check(r, 0, r.attend(L, window), few, window, (at > p) | (at <= p - window))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("d", [9, 15, 20, 24, 25, 33, 40])
@pytest.mark.parametrize("few,case", [(True, c) for c in FEW] + [(False, c) for c in MANY])
def test_values_of_weights_that_vanish(L, kind, hd, d, few, case):
    """a value 2^d times as large under a weight of 2^-80 or so: its part of the result is nothing, and takes nothing from the others"""
    lens, nq, nkv = case
    r = requests(L, lens, nq, nkv, hd, kind, seed=d + 2)
    r.q.view(-1, nq, hd)[..., 0] = 8.0
    at = lens[0][0] // 2
    pg, slot = int(r.kv_at[0][0][at]), int(r.kv_at[0][1][at])
    codes = torch.zeros(hd, device="cuda")
    codes[0] = -112.0  # the key: 8 * 112 * 2^-1 / sqrt(hd) is 56 or 40, below the others' 0
    r.codes[pg, r.layer, 0, :, slot] = codes.to(DTYPES[kind]).view(torch.uint8)
    scaled(r, 0, at, 0, torch.full((nkv,), 126))
    raised(r, 0, at, 1, d)
    out = r.attend(L)
    for i in range(len(lens)):
        check(r, i, out, few)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("d", [9, 15, 16, 20, 24, 25, 40])
@pytest.mark.parametrize("few,case", [(True, c) for c in FEW] + [(False, c) for c in MANY])
def test_keys_beside_a_far_larger_one(L, kind, hd, d, few, case):
    """queries that lie on keys of small scales, beside one that all rows see, 2^d times as large, with a score far below theirs"""
    lens, nq, nkv = case
    r = requests(L, lens, nq, nkv, hd, kind, seed=d + 3)
    at = lens[0][0] // 2
    r.q.view(-1, nq, hd)[..., 0] = 2.0
    pg, slot = int(r.kv_at[0][0][at]), int(r.kv_at[0][1][at])
    codes = torch.zeros(hd, device="cuda")
    codes[0] = -112.0
    r.codes[pg, r.layer, 0, :, slot] = codes.to(DTYPES[kind]).view(torch.uint8)
    scaled(r, 0, at, 0, torch.full((nkv,), 121 + d))
    out = r.attend(L)
    for i in range(len(lens)):
        check(r, i, out, few)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("d", [12, 18, 20, 24, 40, 60])
@pytest.mark.parametrize("few,case", [(True, c) for c in FEW] + [(False, c) for c in MANY])
def test_scores_beyond_their_differences(L, kind, hd, d, few, case):
    """two keys alike, far above the others, with scores of 2^d and more, and values 2^3 apart: their mean, however few bits a score has behind its point"""
    lens, nq, nkv = case
    r = requests(L, lens, nq, nkv, hd, kind, seed=d + 4)
    r.q.view(-1, nq, hd)[..., 0] = 4.0
    codes = torch.zeros(hd, device="cuda")
    codes[0] = 112.0
    at = (5, lens[0][0] - 2)
    for a in at:
        pg, slot = int(r.kv_at[0][0][a]), int(r.kv_at[0][1][a])
        r.codes[pg, r.layer, 0, :, slot] = codes.to(DTYPES[kind]).view(torch.uint8)
        scaled(r, 0, a, 0, torch.full((nkv,), 127 + d))
    raised(r, 0, at[1], 1, 3)
    out = r.attend(L)[:lens[0][1]].view(-1, nq, hd).double()
    v = [r.v[0][a].repeat_interleave(nq // nkv, 0) for a in at]
    want, size = (v[0] + v[1]) / 2, (v[0].abs() + v[1].abs()) / 2
    assert ((out - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -9) * size).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd,ps", [(64, 16), (128, 24), (128, 16)])
@pytest.mark.parametrize("few,case", [(True, c) for c in FEW] + [(False, c) for c in MANY] + [(False, ([(0, 700)], 7, 1))])
@pytest.mark.parametrize("window", [0, 90])
def test_scales_of_any_distance(L, kind, hd, ps, few, case, window):
    """each key's scale is any of 2^-60 .. 1 of the usual one's and each value's any of 2^-40 .. 2^40, zeros and vectors of no numbers that no row sees among them: every key counts once, by its own scale"""
    lens, nq, nkv = case
    r = requests(L, lens, nq, nkv, hd, kind, seed=7, ps=ps)
    rs = np.random.default_rng(3)
    for i, (c, m) in enumerate(lens):
        for j, lo, hi in ((0, -60, 1), (1, -40, 41)):
            pg, at = r.kv_at[i]
            b = r.scale[pg, r.layer, j, :, at].int() + torch.from_numpy(rs.integers(lo, hi, (c + m, nkv))).cuda()
            b[torch.from_numpy(rs.random((c + m, nkv)) < 0.1).cuda()] = 0
            r.scale[pg, r.layer, j, :, at] = b.to(torch.uint8)
            (r.k, r.v)[j][i] = values(r.codes[pg, r.layer, j, :, at], r.scale[pg, r.layer, j, :, at].int(), kind)
    out = r.attend(L, window)
    for i in range(len(lens)):
        check(r, i, out, few, window)
    again = r.attend(L, window)
    assert torch.equal(out[:r.start[-1]], again[:r.start[-1]])


@pytest.mark.parametrize("j", [0, 1])
@pytest.mark.parametrize("few,lens,at", [(True, [(100, 5), (9, 1)], 102), (False, [(100, 60), (9, 1)], 130), (False, [(0, 200)], 3)])
def test_no_numbers_beside_scales_far_apart(L, j, few, lens, at):
    """a vector of no numbers: the rows that see it are none, the others are as without it, though scales are of any distance"""
    r = requests(L, lens, 4, 2, 64, "e4m3", seed=11)
    for p in range(0, sum(lens[0]), 3):
        raised(r, 0, p, 1, -30 + p % 60)
    scaled(r, 0, at, j, torch.full((2,), 255))
    out = r.attend(L)
    p = torch.arange(lens[0][0], sum(lens[0]), device="cuda")
    seen = p >= at
    assert out[:lens[0][1]][seen].isnan().all()
    check(r, 0, out, few, rows=~seen)


def test_a_step_of_rows_that_end_apart(L):
    """wide tiles at the cuts between CTAs: one long prompt and long decode rows, single and in the same call"""
    for lens, few in (([(5000, 1), (3000, 1)], True), ([(2000, 600), (4000, 1)], False)):
        r = requests(L, lens, 8, 1, 128, "e4m3", seed=13, room=0)
        for i, (c, m) in enumerate(lens):
            for j, step in ((0, 5), (1, 7)):
                pg, at = r.kv_at[i]
                b = r.scale[pg, r.layer, j, :, at].int()
                b[::step] -= 18
                r.scale[pg, r.layer, j, :, at] = b.to(torch.uint8)
                (r.k, r.v)[j][i] = values(r.codes[pg, r.layer, j, :, at], r.scale[pg, r.layer, j, :, at].int(), "e4m3")
        out = r.attend(L)
        for i in range(len(lens)):
            check(r, i, out, few or lens[i][1] == 1)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("few,case", [(True, c) for c in FEW] + [(False, c) for c in MANY])
@pytest.mark.parametrize("zeros", [40, 10 ** 6])
def test_values_that_are_zeros(L, kind, hd, few, case, zeros):
    """many values in a row that are zeros, at the beginning or all of them, with keys that are none"""
    lens, nq, nkv = case
    r = requests(L, lens, nq, nkv, hd, kind, seed=15)
    for i, (c, m) in enumerate(lens):
        for p in range(0 if zeros > c + m else max(0, c - zeros) // 2, min(zeros + c // 2, c + m)):
            scaled(r, i, p, 1, torch.zeros(nkv))
    out = r.attend(L)
    for i in range(len(lens)):
        check(r, i, out, few)
        if zeros > sum(lens[i]):
            assert (out[r.start[i]:r.start[i + 1]] == 0).all()


@pytest.mark.parametrize("lens,nq,nkv,few", [([(9000, 1)] * 4, 8, 4, True), ([(100, 333)], 14, 2, False), ([(600, 300)], 4, 2, False)])
@pytest.mark.parametrize("first", [150, 4000])
@pytest.mark.parametrize("j", [0, 1])
def test_first_keys_of_zeros(L, j, first, lens, nq, nkv, few):
    """the first positions' keys, or values, are zeros: whole units and tiles of them ahead of others of the same stretch"""
    r = requests(L, lens, nq, nkv, 128, "e4m3", seed=16, room=0 if few else 4)
    for i, (c, m) in enumerate(lens):
        pg, at = r.kv_at[i]
        n = min(first, c - 10)
        r.scale[pg[:n], r.layer, j, :, at[:n]] = 0
        (r.k, r.v)[j][i][:n] = 0
    out = r.attend(L)
    for i in range(len(lens)):
        check(r, i, out, few)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("few,case", [(True, c) for c in FEW] + [(False, c) for c in MANY])
def test_a_value_of_zeros_that_takes_the_weight(L, hd, few, case):
    """a key that every row lies on, e^40 above the others, with a value of zeros: the result is the others', small as it is"""
    lens, nq, nkv = case
    r = requests(L, lens, nq, nkv, hd, "e4m3", seed=17)
    r.q.view(-1, nq, hd)[..., 0] = 4.0
    at = lens[0][0] // 2
    pg, slot = int(r.kv_at[0][0][at]), int(r.kv_at[0][1][at])
    codes = torch.zeros(hd, device="cuda")
    codes[0] = 112.0 if hd == 128 else 80.0  # 4 * 112 / sqrt(128), 4 * 80 / 8: about 40
    r.codes[pg, r.layer, 0, :, slot] = codes.to(DTYPES["e4m3"]).view(torch.uint8)
    scaled(r, 0, at, 0, torch.full((nkv,), 127))
    scaled(r, 0, at, 1, torch.zeros(nkv))
    check(r, 0, r.attend(L), few)
