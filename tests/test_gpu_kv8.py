"""The operators over a cache in 8 bits (csrc/kv8_store.cu, attn_batch8.cu) against their plain forms in 64 bits (kv8_util.py, step_util.py), one by one and as a step.

Bounds.  Read back: exact.  Values stored: exact codes.  Keys: the rotation in fp32 is off by 2^-18 of |a| + |b| (derived in test_gpu_serving_step.py), and rounding a number that is off by d
gives one that is off by d and half a step of the code: 2^-4 of itself or half of 2^-9 scales for e4m3, half a scale for int8; 2^-24 more of each for the comparison's own arithmetic.
Attention: weights are rounded to fp16 in the product with the values, 2^-11 of the mean of |v| under the weights.  They are there by 2^7, so one below 2^-14 of fp16's is off by 2^-25 of 2^7
of a row's reference, which the largest weight is not below: 2^-32 of it, for each key, times the largest |v|; 2^-31 with what the values' powers of two add.
Codes and queries are exact in fp16; scores in fp32 are off by at most 128 * 2^-23 of sum |q k| / sqrt(hd), below 2^6 here, so weights by 2^-10 of themselves, exponentials and sums by
less: 2^-9 of that mean for all of it."""
import numpy as np
import pytest
import torch

import step_util as ref
from kv8_util import DTYPES, MOST, Requests8, as_bytes, attend, coded, i32, rand, values

pytestmark = pytest.mark.gpu
KINDS = ["e4m3", "int8"]


@pytest.fixture(scope="module")
def L():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    from qwen_inference_engine_b200 import layers
    return layers


def placed(t, off, stride):
    """rows of t, `stride` apart, `off` elements behind a 256-byte boundary, with 77 between them"""
    buf = torch.full((off + t.shape[0] * stride + 8,), 77.0, dtype=t.dtype, device="cuda")
    v = buf[off:off + t.shape[0] * stride].view(t.shape[0], stride)[:, :t.shape[1]]
    v.copy_(t)
    return v, buf


def any_pool(seed, kind, pages, layers, nkv, ps, hd):
    g = torch.Generator("cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (pages, layers, 2, nkv, ps, hd), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    scale = torch.randint(0, 256, (pages, layers, 2, nkv, ps), generator=g, device="cuda", dtype=torch.int32).to(torch.uint8)
    return codes, scale


def same(a, b):
    return torch.equal(a.nan_to_num(nan=123.0), b.nan_to_num(nan=123.0)) and torch.equal(a.isnan(), b.isnan())


# ---------------------------------------------------------------- rows read back
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nkv,hd,ps", [(1, 64, 16), (2, 128, 5), (4, 128, 16), (3, 64, 1)])
@pytest.mark.parametrize("n,off,more", [(1, 0, 0), (7, 0, 8), (300, 3, 1), (5000, 8, 16)])
def test_read(L, kind, nkv, hd, ps, n, off, more):
    rs, pages = np.random.default_rng(n + hd), 40
    codes, scale = any_pool(n, kind, pages, 2, nkv, ps, hd)
    row = rs.integers(0, pages * ps, n)
    bad = rs.random(n) < 0.1
    row[bad] = rs.choice([-1, pages * ps, 2 ** 31 - 1, -2 ** 31], int(bad.sum()))
    k, kb = placed(torch.full((n, nkv * hd), 5.0, dtype=torch.bfloat16, device="cuda"), off, nkv * hd + more)
    v, vb = placed(torch.full((n, nkv * hd), 5.0, dtype=torch.bfloat16, device="cuda"), off, nkv * hd + 2 * more)
    L.launch_kv8_read(L.KvPool8.over(codes.view(DTYPES[kind]), scale), 1, i32(row), k, v)
    torch.cuda.synchronize()
    at, ok = torch.from_numpy(np.where(bad, 0, row)).cuda(), torch.from_numpy(~bad).cuda()
    for i, (got, buf) in enumerate(((k, kb), (v, vb))):
        want = values(codes[at // ps, 1, i, :, at % ps], scale[at // ps, 1, i, :, at % ps].long(), kind).flatten(1).bfloat16()
        assert same(got[ok].float(), want[ok].float())
        assert (got[~ok] == 5).all() and (buf == 77).sum() >= buf.numel() - got.numel()
        only = torch.zeros_like(got, memory_format=torch.contiguous_format)
        L.launch_kv8_read(L.KvPool8.over(codes.view(DTYPES[kind]), scale), 1, i32(row), *((only, None) if i == 0 else (None, only)))
        assert same(only[ok].float(), want[ok].float())


@pytest.mark.parametrize("kind", KINDS)
def test_read_every_code_and_scale(L, kind):
    codes = torch.stack([torch.arange(256, device="cuda").to(torch.uint8).view(4, 1, 64)] * 2).expand(256, 1, 2, 4, 1, 64).contiguous()
    scale = torch.arange(256, device="cuda").to(torch.uint8).view(256, 1, 1, 1, 1).expand(256, 1, 2, 4, 1).contiguous()
    k, v = (torch.empty(256, 256, dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
    L.launch_kv8_read(L.KvPool8.over(codes.view(DTYPES[kind]), scale), 0, i32(np.arange(256)), k, v)
    want = values(codes[:, 0, 0, :, 0], scale[:, 0, 0, :, 0].long(), kind).flatten(1)
    assert same(k.float(), want.bfloat16().float()) and same(v.float(), want.bfloat16().float())
    exact = (want.abs() >= 2.0 ** -126) & (want.abs() < 2.0 ** 128) | (want == 0)  # (scales of 2^120 and more, which a store has no use for, have codes beyond bf16's numbers)
    assert torch.equal(k.double()[exact], want[exact])


# ---------------------------------------------------------------- the store
def near_codes(kind, got, byte, want, size):
    """values `got` with scale bytes `byte` of vectors that are `want` but for 2^-18 of `size`"""
    s = torch.exp2(byte.double() - 127)
    most, d = want.abs().amax(-1), 2.0 ** -18 * size
    assert (most - d.amax(-1) <= MOST[kind] * s).all() and (most + d.amax(-1) > MOST[kind] / 2 * s).all()
    half = torch.maximum(2.0 ** -4 * (want.abs() + d), 2.0 ** -10 * s[..., None]) if kind == "e4m3" else 0.5 * s[..., None]
    assert ((got - want).abs() <= half * (1 + 2.0 ** -20) + d).all()


ROPE = [(2, 1, 64, 64), (14, 2, 64, 32), (28, 4, 128, 128), (12, 2, 128, 50), (3, 3, 64, 2), (1, 1, 128, 64), (0, 2, 64, 64), (5, 5, 128, 96), (2, 1, 64, 48), (4, 2, 64, 62)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nq,nkv,hd,rot", ROPE)
@pytest.mark.parametrize("neighbours", [False, True])
@pytest.mark.parametrize("n,off,more,far", [(1, 0, 0, 1), (7, 0, 8, 2 ** 31 - 1), (65, 3, 1, 5000), (3000, 8, 16, 40000)])
def test_rope_store(L, kind, nq, nkv, hd, rot, neighbours, n, off, more, far):
    rs = np.random.default_rng(nq * 100 + hd + rot + n)
    pages, ps = (n + 4) // 5 + 2, 5
    w, factor = L.Rope.frequencies(rot, 10000.0, "yarn", 2.0, 4096)
    freq = torch.from_numpy(w).cuda()
    pos = rs.integers(max(0, far - 60000), far + 1, n)
    row = rs.permutation(pages * ps)[:n]
    no_q, no_kv = rs.random(n) < 0.1, rs.random(n) < 0.1
    pos[no_q] = -1 - rs.integers(0, 5, int(no_q.sum()))
    row[no_kv] = rs.choice([-1, pages * ps, 2 ** 31 - 1], int(no_kv.sum()))
    x = rand(n + hd, n, (nq + 2 * nkv) * hd).bfloat16()
    qkv, buf = placed(x, off, (nq + 2 * nkv) * hd + more)
    q, k, v = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
    out, out_buf = placed(torch.full((n, nq * hd), 5.0, dtype=torch.bfloat16, device="cuda"), off, nq * hd + more + 1 if nq else 1)
    codes, scale = any_pool(1, kind, pages, 2, nkv, ps, hd)
    before, kept = (codes.clone(), scale.clone()), buf.clone()
    L.launch_rope_store8(q, k, v, out, L.KvPool8.over(codes.view(DTYPES[kind]), scale), 1, i32(pos), i32(row), L.Rope(freq, factor, neighbours), nq)
    torch.cuda.synchronize()
    assert torch.equal(buf, kept)
    heads = x.view(n, -1, hd)
    want = ref.rope(heads, torch.from_numpy(pos).cuda().clamp(min=0), freq, factor, neighbours)
    size = (heads.double().abs().amax((1, 2)) * 2 * factor)[:, None, None]
    yes, put = torch.from_numpy(~no_q).cuda(), torch.from_numpy(~no_kv).cuda()
    if nq:
        got = out.reshape(n, nq, hd)
        assert ((got[yes].double() - want[yes, :nq]).abs() <= 2.0 ** -8 * want[yes, :nq].abs() + 2.0 ** -18 * size[yes]).all()
        assert (got[~yes] == 5).all() and (out_buf == 77).sum() >= out_buf.numel() - out.numel()
        assert torch.equal(got[yes][..., rot:], heads[yes, :nq, rot:])
    r = torch.from_numpy(row).cuda()
    got_v, got_s = codes[r[put] // ps, 1, 1, :, r[put] % ps], scale[r[put] // ps, 1, 1, :, r[put] % ps]
    c, b = coded(heads[put, nq + nkv:], kind)
    assert torch.equal(got_s.long(), b) and torch.equal(got_v.view(DTYPES[kind]).double(), c)
    sure = put & yes
    at = r[sure]
    byte = scale[at // ps, 1, 0, :, at % ps].long()
    near_codes(kind, values(codes[at // ps, 1, 0, :, at % ps], byte, kind), byte, want[sure, nq:nq + nkv], size[sure].expand(-1, nkv, 1))
    left = torch.ones(pages * ps, dtype=torch.bool, device="cuda")
    left[r[put]] = False
    for now, was in zip((codes, scale), before):
        assert torch.equal(now[:, 0], was[:, 0])
        for i in (0, 1):
            assert torch.equal(now[:, 1, i].transpose(1, 2).reshape(pages * ps, -1)[left], was[:, 1, i].transpose(1, 2).reshape(pages * ps, -1)[left])


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("hd", [64, 128])
def test_store_without_a_rotation(L, kind, hd):
    """vectors at the borders of what a scale holds: zeros, the smallest and the largest numbers, a largest element at and next to the largest code, ties, no numbers"""
    top = MOST[kind]
    nxt = {"e4m3": 450.0, "int8": 127.5}[kind]  # bf16's next number
    special = torch.zeros(16, hd)
    special[1, 3] = 2.0 ** -133
    special[2, 5], special[2, 6] = 3.3e38, -2.0 ** -20
    special[3, 0], special[4, 0], special[5, 0], special[6, hd - 1] = top, nxt, top * 2.0 ** -60, -nxt * 2.0 ** 40
    special[7] = torch.arange(hd) + 0.5                     # ties
    special[8] = (torch.arange(hd) - hd / 2) * 2.0 ** -8
    special[9, 1], special[10, 2], special[11, 7] = float("inf"), float("nan"), -float("inf")
    special[12] = -0.0
    special[13] = torch.linspace(-100, 100, hd)
    special[14] = 2.0 ** -120
    special[15] = torch.exp2(torch.linspace(-20, 8, hd))
    x = special.bfloat16().cuda().repeat_interleave(3, 0)  # three kv heads
    k = x.view(16, 3 * hd)
    v = k.flip(0).contiguous()
    codes, scale = any_pool(2, kind, 4, 1, 3, 7, hd)
    pool, row = L.KvPool8.over(codes.view(DTYPES[kind]), scale), np.random.default_rng(0).permutation(28)[:16]
    L.launch_rope_store8(None, k, v, None, pool, 0, None, i32(row), None, 0)
    ko, vo = torch.empty_like(k), torch.empty_like(v)
    L.launch_kv8_read(pool, 0, i32(row), ko, vo)
    r = torch.from_numpy(row).cuda()
    for i, (src, got) in enumerate(((k, ko), (v, vo))):
        heads = src.view(16, 3, hd)
        fine = torch.isfinite(heads.float()).all(-1)
        c, b = coded(torch.where(fine[..., None], heads.double(), 0.0), kind)
        byte = scale[r // 7, 0, i, :, r % 7].long()
        assert (byte[~fine] == 255).all() and torch.equal(byte[fine], b[fine])
        assert torch.equal(codes[r // 7, 0, i, :, r % 7].view(DTYPES[kind]).double()[fine], c[fine])
        g = got.view(16, 3, hd)
        assert g[~fine].isnan().all() and torch.equal(g[fine], (c * torch.exp2(b.double() - 127)[..., None]).bfloat16()[fine])


@pytest.mark.parametrize("kind", KINDS)
def test_store_in_place(L, kind):
    n, nq, hd = 50, 14, 64
    x = rand(4, n, nq * hd).bfloat16()
    kv = rand(5, n, 2 * hd).bfloat16()
    freq, pos = torch.from_numpy(L.Rope.frequencies(hd)[0]).cuda(), i32(np.arange(n) * 331)
    outs = []
    for here in (False, True):
        codes, scale = any_pool(2, kind, 4, 1, 1, 16, hd)
        q = x.clone()
        out = q if here else torch.empty_like(q)
        L.launch_rope_store8(q, kv[:, :hd], kv[:, hd:], out, L.KvPool8.over(codes.view(DTYPES[kind]), scale), 0, pos, i32(np.arange(n)), L.Rope(freq), nq)
        outs.append((out, codes, scale))
    assert all(torch.equal(a, b) for a, b in zip(*outs))


# ---------------------------------------------------------------- attention
HEADS = [(14, 2, 64), (12, 2, 128), (28, 4, 128), (3, 3, 64), (1, 1, 128)]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nq,nkv,hd", HEADS)
@pytest.mark.parametrize("lens", [[(0, 1)], [(699, 1)], [(0, 63)], [(0, 64), (64, 64)], [(63, 2), (1, 0), (64, 1)], [(0, 300)], [(1000, 130)], [(129, 19), (5, 18), (127, 1)],
                                  [(i * 37 % 500, 1) for i in range(40)], [(2000, 1), (0, 500), (100, 3), (0, 1), (50, 0), (9, 77)], [(5000, 1), (1, 1)]])
def test_attention(L, kind, nq, nkv, hd, lens):
    attend(L, lens, nq, nkv, hd, 16, kind, extra=3, seed=len(lens))


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nq,nkv,hd", HEADS + [(16, 1, 128), (17, 1, 64), (16, 16, 64), (5, 1, 128), (9, 3, 128), (8, 1, 64)])
@pytest.mark.parametrize("window", [0, 70])
@pytest.mark.parametrize("lens", [[(i * 97 % 1500, 1) for i in range(64)], [(0, 1)] * 3, [(500, 1), (77, 0), (0, 1), (64, 0), (63, 1)], [(300, 5), (10, 0), (9, 0), (8, 0), (6, 0)],
                                  [(4000, 3), (100, 0), (200, 0), (1, 1)], [(20000, 1)]])
def test_attention_no_more_rows_than_requests(L, kind, nq, nkv, hd, window, lens):
    """decode steps, and steps with a few more rows for some requests and none for others"""
    attend(L, lens, nq, nkv, hd, 16, kind, window=window, seed=len(lens) + nq)


@pytest.mark.parametrize("ps", [1, 2, 3, 4, 5, 8, 16, 24, 32, 48, 64, 100, 128, 256])
@pytest.mark.parametrize("nq,nkv,hd,kind", [(14, 2, 64, "e4m3"), (4, 1, 128, "int8")])
@pytest.mark.parametrize("decode", [False, True])
def test_attention_page_sizes(L, ps, nq, nkv, hd, kind, decode):
    attend(L, [(300, 1), (0, 1), (333, 1), (1600, 1), (0, 0), (511, 1)] if decode else [(70, 40), (0, 1), (333, 1), (128, 70), (0, 0), (511, 1)], nq, nkv, hd, ps, kind, seed=ps)


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 63, 64, 65, 200, 1000, 2 ** 31 - 1])
@pytest.mark.parametrize("nq,nkv,hd,ps,kind", [(14, 2, 64, 16, "int8"), (6, 2, 128, 4, "e4m3"), (6, 2, 128, 64, "int8")])
def test_attention_window(L, window, nq, nkv, hd, ps, kind):
    attend(L, [(0, 300), (700, 1), (64, 64), (513, 130), (0, 1), (2100, 1)], nq, nkv, hd, ps, kind, window=window, seed=window % 1000)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("nq,nkv,hd", [(128, 1, 64), (100, 1, 128), (65, 1, 64), (64, 1, 128), (32, 2, 64), (43, 1, 128), (16, 16, 64)])
@pytest.mark.parametrize("lens", [[(0, 5), (200, 1), (65, 33), (0, 130)], [(2000, 1), (65, 1), (0, 1)]])
def test_attention_heads_of_a_group(L, kind, nq, nkv, hd, lens):
    attend(L, lens, nq, nkv, hd, 16, kind, seed=nq, extra=1 if len(lens) > 3 else 0)


@pytest.mark.parametrize("scale", [0.01, 0.3])
def test_attention_scale(L, scale):
    attend(L, [(10, 90), (300, 1)], 14, 2, 64, 16, "e4m3", scale=scale)


@pytest.mark.parametrize("lens", [[(100, 30), (0, 1), (64, 65)], [(100, 1), (0, 1), (64, 1)]])
def test_attention_strides_and_plain_slots(L, lens):
    r = Requests8(L, lens, 14, 2, 64, 16, "int8", slots=False, seed=3)
    wide = torch.full((r.rows, 14 * 64 + 40), float("nan"), dtype=torch.bfloat16, device="cuda")
    q, out = wide[:, 8:8 + 14 * 64], torch.full((r.rows, 14 * 64 + 16), 9.0, dtype=torch.bfloat16, device="cuda")
    q.copy_(r.q)
    L.launch_attn_batch8(q, out[:, :14 * 64], r.kv, r.layer, r.batch, 14)
    r.check(out[:, :14 * 64])
    assert (out[:, 14 * 64:] == 9).all()


@pytest.mark.parametrize("kind", KINDS)
def test_attention_many_requests(L, kind):
    rs = np.random.default_rng(1)
    attend(L, [(int(c), int(m)) for c, m in zip(rs.integers(0, 200, 700), rs.integers(0, 4, 700))], 4, 2, 64, 16, kind, seed=9)


@pytest.mark.parametrize("kind", KINDS)
def test_attention_long(L, kind):
    """one row behind many positions beside short ones, and a long prompt: the split over the positions"""
    attend(L, [(40000, 1), (3, 2)], 14, 2, 64, 16, kind, seed=2)
    attend(L, [(0, 2500), (7000, 600)], 7, 1, 128, 16, kind, seed=4)
    attend(L, [(70000, 1), (3, 1)], 6, 1, 128, 16, kind, seed=5)


def test_attention_same_bits_again(L):
    for lens in ([(3000, 1), (0, 700), (10, 5)], [(3000, 1), (700, 1), (10, 1)]):
        r = Requests8(L, lens, 14, 2, 64, 16, "e4m3", seed=8)
        out = r.attend(L)
        for _ in range(3):
            r.batch.work.random_(0, 255)  # whatever an earlier call left in the work area
            assert torch.equal(r.attend(L), out)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("lens", [[(300, 70), (900, 1)], [(300, 1), (900, 1)]])
def test_attention_values_behind_the_weights(L, kind, lens):
    """large scores: the largest weight is one and the others vanish; and rows whose keys are all alike"""
    r = Requests8(L, lens, 4, 2, 128, 16, kind, seed=5)
    r.q.mul_(30)
    # scores are 30 times as large and their fp32 errors with them: weights off by 2^-5 of themselves, the mean of |v| by the bound's 2^-9 plus that
    r.check(r.attend(L), more=2.0 ** -4)
    r.q.zero_()
    r.check(r.attend(L))


@pytest.mark.parametrize("lens", [[(500, 200), (3, 1), (1000, 1)], [(500, 1), (3, 1), (3000, 1)]])
@pytest.mark.parametrize("nq,nkv,hd", [(7, 1, 128), (14, 2, 64), (16, 1, 128)])
def test_attention_scales_far_apart(L, lens, nq, nkv, hd):
    """Keys and values whose scales differ by up to 2^40: what a key or a value beside a far larger one loses is 2^-24 of the larger one's smallest unit's, which its part of the result does not
    show: weights are those of the exact scores, and the result is off by the bound's share of the mean of |v|."""
    r = Requests8(L, lens, nq, nkv, hd, 16, "e4m3", seed=6, spread=5.0)
    r.q.mul_(2.0 ** -18)  # (scores stay below 2^6)
    r.check(r.attend(L), more=2.0 ** -9)


def put(r, i, pos, j, codes=None, scale=None):
    """bytes into position pos of request i's keys (j 0) or values (1), of the first kv head"""
    pg, at = int(r.kv_at[i][0][pos]), int(r.kv_at[i][1][pos])
    if codes is not None:
        r.codes[pg, r.layer, j, 0, at] = codes
    if scale is not None:
        r.scale[pg, r.layer, j, 0, at] = scale


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("j", [0, 1])
@pytest.mark.parametrize("lens,at", [([(0, 100), (70, 1)], 50), ([(300, 300), (9, 2)], 300), ([(64, 1), (40, 1), (33, 1)], 3), ([(200, 3), (0, 0), (5, 1), (6, 0)], 201)])
def test_attention_vectors_of_no_numbers(L, kind, j, lens, at):
    """a key's or value's scale of 255: no number in every column of the rows that see it, and nothing in the others"""
    r = Requests8(L, lens, 4, 2, 64, 16, kind, seed=6)
    before = r.attend(L)
    put(r, 0, at, j, scale=255)
    out = r.attend(L).view(-1, 4, 64)
    c, m = lens[0]
    sees = torch.zeros(len(out), dtype=torch.bool, device="cuda")
    sees[max(0, at - c):m] = True
    assert out[sees][:, :2].isnan().all()
    assert torch.equal(out[~sees], before.view(-1, 4, 64)[~sees]) and torch.equal(out[:, 2:], before.view(-1, 4, 64)[:, 2:])


@pytest.mark.parametrize("lens,at", [([(0, 100), (70, 1)], 50), ([(300, 300), (9, 2)], 300), ([(200, 3), (0, 0), (5, 1), (6, 0)], 201)])
def test_attention_codes_of_no_number(L, lens, at):
    """e4m3's code for no number among the values: in that column at least of the rows that see it, and in no other row"""
    r = Requests8(L, lens, 4, 2, 64, 16, "e4m3", seed=6)
    before = r.attend(L).view(-1, 4, 64)
    for code in (0x7f, 0xff):
        bytes_ = r.codes[int(r.kv_at[0][0][at]), r.layer, 1, 0, int(r.kv_at[0][1][at])].clone()
        bytes_[7] = code
        put(r, 0, at, 1, codes=bytes_)
        out = r.attend(L).view(-1, 4, 64)
        c, m = lens[0]
        sees = torch.zeros(len(out), dtype=torch.bool, device="cuda")
        sees[max(0, at - c):m] = True
        assert out[sees][:, :2, 7].isnan().all() and torch.equal(out[~sees], before[~sees]) and torch.equal(out[:, 2:], before[:, 2:])


def test_attention_queries_of_no_numbers(L):
    for lens in ([(50, 20), (300, 2)], [(50, 1), (300, 1)]):
        r = Requests8(L, lens, 4, 2, 128, 16, "int8", seed=7)
        before = r.attend(L).view(-1, 4, 128)
        r.q.view(-1, 4, 128)[0, 1, 5], r.q.view(-1, 4, 128)[1, 2, 0] = float("inf"), float("nan")
        out = r.attend(L).view(-1, 4, 128)
        assert out[0, 1].isnan().all() and out[1, 2].isnan().all()
        out[0, 1], out[1, 2] = before[0, 1], before[1, 2]
        assert torch.equal(out, before)


@pytest.mark.parametrize("lens", [[(500, 90), (0, 1), (64, 2)], [(500, 1), (0, 1), (64, 1)]])
def test_attention_of_zeros(L, lens):
    """keys of zeros: the mean of the values; values of zeros: zeros; a pool as it is made"""
    r = Requests8(L, lens, 14, 2, 64, 16, "e4m3", seed=7)
    for x in r.k:
        x.zero_()
    r.codes[:, r.layer, 0], r.scale[:, r.layer, 0] = 0, 0
    r.check(r.attend(L))
    r.codes.zero_(), r.scale.zero_()
    assert (r.attend(L)[:r.start[-1]] == 0).all()


@pytest.mark.parametrize("lens", [[(1500, 1), (0, 400), (33, 2)], [(1500, 1), (40, 1), (33, 1)]])
def test_attention_two_streams(L, lens):
    """two calls at once, each with a work area of its own"""
    a = [Requests8(L, lens, 14, 2, 64, 16, "int8", seed=20 + i) for i in range(2)]
    outs, streams = [torch.full_like(r.q, 9.0) for r in a], [torch.cuda.Stream() for _ in a]
    for r in a:
        r.batch.reserve(r.kv, 14)
    torch.cuda.synchronize()
    for _ in range(5):
        for r, o, s in zip(a, outs, streams):
            with torch.cuda.stream(s):
                L.launch_attn_batch8(r.q, o, r.kv, r.layer, r.batch, 14)
    torch.cuda.synchronize()
    for r, o in zip(a, outs):
        r.check(o)


@pytest.mark.parametrize("lens", [[(100, 10), (50, 20), (300, 1), (7, 5)], [(100, 1), (50, 1), (300, 1), (7, 1)]])
@pytest.mark.parametrize("ps", [16, 4, 5])
def test_attention_nonsense_stays_inside(L, lens, ps):
    """offsets, lengths, slots and pages that make no sense: nothing is read or written outside, and requests beside them keep their results"""
    r = Requests8(L, lens, 14, 2, 64, ps, "e4m3", seed=11)
    s, n = r.start, int(r.start[-1])
    kv_len, slots, table = r.batch.kv_len.clone(), r.batch.slots.clone(), r.batch.block_table.clone()
    want = r.attend(L)
    r.check(want)
    r.batch.kv_len[1] = 2 ** 31 - 1
    r.batch.block_table[slots[1]] = i32([-5])
    r.batch.block_table[slots[1], 1] = 2 ** 31 - 1
    out = r.attend(L)
    good = torch.ones(n, dtype=torch.bool, device="cuda")
    good[s[1]:s[2]] = False
    # the split over the positions may fall elsewhere: two results within their bounds
    assert ((out[good].double() - want[good].double()).abs() <= 2.0 ** -6 * 20).all()
    r.batch.kv_len.copy_(kv_len)
    r.attend(L)  # pages that are none
    r.batch.block_table.copy_(table)
    for bad in (-1, 10 ** 6, -2 ** 31):
        r.batch.slots[1] = bad
        out = r.attend(L)
        assert (out[s[1]:s[2]] == 9).all() and torch.isfinite(out).all()
    r.batch.slots.copy_(slots)
    for start in ([0, 10, 30, 31, 2 ** 31 - 1], [0, -50, 30, 31, 36], [36, 31, 30, 10, 0], [2 ** 31 - 1] * 5, [-2 ** 31, 2 ** 31 - 1, 0, 0, 0]):
        r.batch.q_start.copy_(i32(start))
        r.attend(L)
    for k in (-2 ** 31, -1, 0):
        r.batch.q_start.copy_(i32(r.start))
        r.batch.kv_len.fill_(k)
        r.attend(L)
    r.batch.kv_len.copy_(kv_len)
    r.check(r.attend(L))


@pytest.mark.parametrize("ps", [16, 5])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n,room", [(200, 200), (1, 1)])
def test_offsets_beyond_32_bits(L, ps, kind, n, room):
    """a pool of more than 2^32 bytes: store, read and attention at its end"""
    pages, g, cached = 2 ** 32 // (2 * ps * 128) + 300, 4, 199 if n == 1 else 0
    codes = torch.empty(pages, 1, 2, 1, ps, 128, dtype=torch.uint8, device="cuda").view(DTYPES[kind])
    scale = torch.empty(pages, 1, 2, 1, ps, dtype=torch.uint8, device="cuda")
    total = cached + n
    mine = torch.arange(pages - 1, pages - 1 - (total + ps - 1) // ps, -1, dtype=torch.int32, device="cuda")
    pos = torch.arange(total, dtype=torch.int32, device="cuda")
    row = mine[(pos // ps).long()] * ps + pos % ps
    x = rand(1, total, (g + 2) * 128).bfloat16()
    q, k, v = x.split([g * 128, 128, 128], 1)
    q_out, freq = torch.empty_like(q.contiguous()), torch.from_numpy(L.Rope.frequencies(128)[0]).cuda()
    kv = L.KvPool8.over(codes, scale)
    L.launch_rope_store8(q, k, v, q_out, kv, 0, pos, row, L.Rope(freq), g)
    kb, vb = torch.empty_like(k.contiguous()), torch.empty_like(v.contiguous())
    L.launch_kv8_read(kv, 0, row, kb, vb)
    c, b = coded(v.view(total, 1, 128), kind)
    assert torch.equal(vb.double(), (c * torch.exp2(b.double() - 127)[..., None]).flatten(1))
    batch = L.Batch(mine[None].contiguous(), ps, pages, 1, n, q_start=i32([0, n]), kv_len=i32([total]))
    rows = q_out[cached:].contiguous()
    out = torch.empty_like(rows)
    L.launch_attn_batch8(rows, out, kv, 0, batch, g)
    want, size = ref.attention(rows.view(n, g, 128), kb[:, None], vb[:, None], cached)
    assert ((out.view(n, g, 128).double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -9) * size + 2.0 ** -20).all()


def test_attention_refuses_a_small_work_area(L):
    from qwen_inference_engine_b200._lib import QieError
    r = Requests8(L, [(10, 1)], 2, 1, 64, 16, "e4m3")
    r.batch.reserve(r.kv, 2)
    n, r.batch.view.work_bytes = r.batch.view.work_bytes, r.batch.view.work_bytes - 1
    with pytest.raises(QieError, match="work area"):
        r.attend(L)
    r.batch.view.work_bytes = n
    r.check(r.attend(L))


def test_one_batch_over_both_pools(L):
    """a batch whose work area serves the pool in bfloat16 and the one in 8 bits, and a graph from before it grew"""
    lens = [(100, 30), (0, 1), (64, 65)]
    r = Requests8(L, lens, 4, 2, 64, 16, "int8", seed=3)
    out8, out16 = torch.zeros_like(r.q), torch.zeros_like(r.q)
    pool = torch.zeros(r.codes.shape, dtype=torch.bfloat16, device="cuda")
    for i in range(len(lens)):
        pg, at = r.kv_at[i]
        pool[pg, r.layer, 0, :, at], pool[pg, r.layer, 1, :, at] = r.k[i].bfloat16(), r.v[i].bfloat16()
    kv = L.KvPool.over(pool)
    L.launch_attn_batch(r.q, out16, kv, r.layer, r.batch, 4)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.launch_attn_batch(r.q, out16, kv, r.layer, r.batch, 4)
    L.launch_attn_batch8(r.q, out8, r.kv, r.layer, r.batch, 4)
    out16.zero_()
    g.replay()
    torch.cuda.synchronize()
    r.check(out8)
    r.check(out16, more=2.0 ** -8)  # (weights in bf16)


# ---------------------------------------------------------------- a step
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("room", [0, 60])
def test_step_in_a_graph(L, kind, room):
    """a layer's part of serving steps, captured once: layout, rotary positions with the store, attention, over lengths that change between replays; every row against its request's own
    history, as the cache stands for it"""
    n, nq, nkv, hd, ps, pages = 5, 6, 2, 64, 16, 120
    most = n + room
    rope = L.Rope(torch.from_numpy(L.Rope.frequencies(hd)[0]).cuda())
    kv = L.KvPool8(pages, ps, 1, nkv, hd, dtype=DTYPES[kind])
    table, ring = torch.zeros(n, 40, dtype=torch.int32, device="cuda"), torch.randperm(pages, generator=torch.Generator("cuda").manual_seed(1), device="cuda").int()
    cached, new, at = (torch.zeros(n, dtype=torch.int32, device="cuda") for _ in range(3))
    ring_in = i32([0, pages])
    b = L.Batch(table, ps, pages, n, most, cached=cached, n_new=new, free_ring=ring, ring_in=ring_in)
    b.ring_out, b.view.ring_out = ring_in, ring_in.data_ptr()
    qkv = torch.zeros(most, (nq + 2 * nkv) * hd, dtype=torch.bfloat16, device="cuda")
    q, k, v = qkv.split([nq * hd, nkv * hd, nkv * hd], 1)
    q_out, out = torch.zeros(most, nq * hd, dtype=torch.bfloat16, device="cuda"), torch.zeros(most, nq * hd, dtype=torch.bfloat16, device="cuda")

    def step():
        L.launch_batch_layout(b)
        L.launch_rope_store8(q, k, v, q_out, kv, 0, b.pos, b.row, rope, nq)
        L.launch_attn_batch8(q_out, out, kv, 0, b, nq)

    b.reserve(kv, nq)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    rs, have = np.random.default_rng(2), np.zeros(n, int)
    for turn in range(6):
        m = rs.integers(0, 2, n) if room == 0 else rs.integers(0, 14, n) * (rs.random(n) < 0.8)
        cached.copy_(i32(have)), new.copy_(i32(m))
        qkv.copy_(rand(turn, *qkv.shape).bfloat16())
        out.fill_(9.0)
        g.replay()
        torch.cuda.synchronize()
        assert (b.status == 0).all()
        start = np.concatenate([[0], np.cumsum(m)])
        for i in range(n):
            if m[i]:
                p = torch.arange(have[i] + m[i], device="cuda")
                row = table[i, p // ps] * ps + (p % ps).int()
                kb, vb = (torch.empty(len(p), nkv * hd, dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
                L.launch_kv8_read(kv, 0, row.int(), kb, vb)
                s = slice(start[i], start[i + 1])
                want, size = ref.attention(q_out[s].view(-1, nq, hd), kb.view(-1, nkv, hd), vb.view(-1, nkv, hd), have[i])
                assert ((out[s].view(-1, nq, hd).double() - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -9) * size + 2.0 ** -20).all()
                turned = ref.rope(k[s].reshape(-1, nkv, hd), p[have[i]:], rope.freq, 1.0, False)
                near = 2.0 ** -3 if kind == "e4m3" else 2.0 ** -6  # (half a step of the largest element's, twice)
                assert ((kb.view(-1, nkv, hd)[have[i]:].double() - turned).abs() <= near * turned.abs().amax(-1, keepdim=True)).all()
        assert (out[start[-1]:] == 9).all()
        have += m


def test_no_wait_ran_out(L):
    """in the kernels of the tests above"""
    from qwen_inference_engine_b200 import _lib
    assert _lib.lib().qie_kernel_status() == 0


@pytest.mark.parametrize("lens", [[(100, 200), (0, 1), (64, 65)], [(100, 1), (0, 1), (64, 1)]])
@pytest.mark.parametrize("ps", [16, 64])
def test_attention_scales_off_a_boundary(L, lens, ps):
    """scale bytes that begin anywhere: bulk copies of them would need 16-byte boundaries"""
    r = Requests8(L, lens, 14, 2, 64, ps, "e4m3", seed=3)
    want = r.attend(L)
    for off in (1, 8):
        buf = torch.empty(r.scale.numel() + 16, dtype=torch.uint8, device="cuda")
        s = buf[off:off + r.scale.numel()].view(r.scale.shape)
        s.copy_(r.scale)
        r.kv = L.KvPool8.over(r.codes.view(DTYPES["e4m3"]), s)
        out = r.attend(L)
        r.check(out)
        assert torch.equal(out, want)


@pytest.mark.parametrize("lens", [[(100, 200), (64, 65)], [(100, 1), (64, 1)]])
@pytest.mark.parametrize("kind", KINDS)
def test_attention_scale_of_zero(L, lens, kind):
    """a scale byte of 0 stands for zeros, whatever the codes beside it"""
    r = Requests8(L, lens, 4, 2, 64, 16, kind, seed=4)
    for i in range(len(lens)):
        pg, at = r.kv_at[i]
        for p in range(0, lens[i][0], 3):
            r.scale[pg[p], r.layer, 1, :, at[p]] = 0
            r.v[i][p] = 0
        r.scale[pg[1], r.layer, 0, :, at[1]] = 0
        r.k[i][1] = 0
    r.check(r.attend(L))


def test_calls_that_do_not_fit(L):
    """what the Python forms refuse"""
    r = Requests8(L, [(10, 3)], 2, 1, 64, 16, "e4m3")
    kv, row = r.kv, i32([0, 1, 2])
    k, v = (torch.zeros(3, 64, dtype=torch.bfloat16, device="cuda") for _ in (0, 1))
    rope = L.Rope(torch.from_numpy(L.Rope.frequencies(64)[0]).cuda())
    q = torch.zeros(3, 128, dtype=torch.bfloat16, device="cuda")
    for bad in (lambda: L.KvPool8.over(r.codes, r.scale), lambda: L.KvPool8.over(r.codes.view(torch.int8), r.scale[:-1]), lambda: L.KvPool8.over(r.codes.view(torch.int8), r.scale.int()),
                lambda: L.KvPool8.over(r.codes.view(torch.int8).cpu(), r.scale.cpu()), lambda: L.launch_kv8_read(kv, 1, row, k[:2], v), lambda: L.launch_kv8_read(kv, 1, row.long(), k, v),
                lambda: L.launch_kv8_read(kv, 1, row, k.float(), v), lambda: L.launch_kv8_read(kv, 1, row, k, v.cpu()), lambda: L.launch_rope_store8(None, k, v[:2], None, kv, 1, None, row, None, 0),
                lambda: L.launch_rope_store8(q, k, v, q, kv, 1, row, row, None, 2), lambda: L.launch_rope_store8(q[:, :64], k, v, q, kv, 1, row, row, rope, 2),
                lambda: L.launch_rope_store8(q, k, v, q, kv, 1, row[:2], row, rope, 2), lambda: L.launch_rope_store8(q, k.T.contiguous().T, v, q, kv, 1, row, row, rope, 2),
                lambda: L.launch_attn_batch8(r.q[:2], r.q[:2], kv, 1, r.batch, 2), lambda: L.launch_attn_batch8(r.q.float(), r.q.float(), kv, 1, r.batch, 2)):
        with pytest.raises(AssertionError):
            bad()
    torch.cuda.synchronize()


def test_no_wait_ran_out_to_the_end(L):
    """in the kernels of any test of this file"""
    from qwen_inference_engine_b200 import _lib
    torch.cuda.synchronize()
    assert _lib.lib().qie_kernel_status() == 0
