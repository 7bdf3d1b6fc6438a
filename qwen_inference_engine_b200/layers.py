"""Operator-level mirror of the reference's `layers/` API.

Same names and argument meaning as layers/include/helpers.cuh:45-166
(launch_rms, launch_rope, launch_rope_single, launch_matmul, launch_elem, launch_act,
launch_resadd, launch_attn, launch_qknorm, sample_topk_bf16), so a parity test reads like
the reference's call site in llm() (src/qwen_main.cu).  Tensors are torch CUDA tensors
(torch is plumbing for device memory and the stream); the work is done by
libqie_b200.so through its C ABI.  bf16 tensors must be contiguous.
"""
import ctypes as C

import numpy as np
import torch

from . import _lib
from ._lib import BatchView, Kv8View, KvView, LogitRulesView, RopePlan, check


def _p(t):
    assert t.is_cuda and t.is_contiguous(), "device-resident contiguous tensor expected"
    return t.data_ptr()


def _st():
    """cudaStream_t of torch's current stream.  (torch.cuda.current_stream() builds an object around it: 3.4 us of an operator call of 8, by the raw handle
    0.3; the latter's names are torch's own, so a torch without them takes the former.)"""
    try:
        return torch._C._cuda_getCurrentRawStream(torch._C._cuda_getDevice())
    except AttributeError:
        return torch.cuda.current_stream().cuda_stream


def embedding(out, table, ids):
    """embedding_matrix_func (src/embedded_matrix.cu:5-17)"""
    check(_lib.lib().qie_embedding(_p(out), _p(table), _p(ids), table.shape[1], ids.numel(), _st()))


def launch_rms(x, w, y, hidden, seqlen):
    check(_lib.lib().qie_rmsnorm(_p(x), _p(w), _p(y), hidden, seqlen, _st()))


def launch_matmul(A, B, Cout, M, N, K):
    """C[M,K] = A[M,N] @ B[K,N]^T -- N is the inner dimension, as in the reference."""
    check(_lib.lib().qie_matmul(_p(A), _p(B), _p(Cout), M, N, K, _st()))


def launch_qknorm(X, w, head_dim, seqlen, hidden, nheads):
    check(_lib.lib().qie_qknorm(_p(X), _p(w), head_dim, seqlen, hidden, nheads, _st()))


def launch_rope(cos_d, sin_d, x, seqlen, head_dim, hidden_dim, nheads):
    check(_lib.lib().qie_rope(_p(cos_d), _p(sin_d), _p(x), seqlen, 0, head_dim, hidden_dim, nheads, _st()))


def launch_rope_single(cos_d, sin_d, x, pos, head_dim, hidden_dim, nheads):
    check(_lib.lib().qie_rope(_p(cos_d), _p(sin_d), _p(x), 1, pos, head_dim, hidden_dim, nheads, _st()))


def launch_act(x, n):
    check(_lib.lib().qie_silu(_p(x), n, _st()))


def launch_elem(a, b, out, n):
    check(_lib.lib().qie_elem_mul(_p(a), _p(b), _p(out), n, _st()))


def launch_resadd(x, y, n):
    check(_lib.lib().qie_residual_add(_p(x), _p(y), n, _st()))


def precompute_cos_sin(seq_len, head_dim):
    """src/include.cpp:5-18 -- host fp32 tables [seq_len, head_dim/2]"""
    c = np.zeros((seq_len, head_dim // 2), np.float32)
    s = np.zeros((seq_len, head_dim // 2), np.float32)
    check(_lib.lib().qie_precompute_cos_sin(c.ctypes.data, s.ctypes.data, seq_len, head_dim))
    return c, s


class KvPool:
    """B200 KV pool pool[page][layer][k|v][kv_head][slot][head_dim] plus a block table; the
    operator-level stand-in for create_page_list / allocate_page_buffers (iengine.cu:73-96)."""

    def __init__(self, n_pages, page_size, n_layers, n_kv_heads, head_dim, max_seqs=8):
        self.pool = torch.zeros(n_pages, n_layers, 2, n_kv_heads, page_size, head_dim, dtype=torch.bfloat16,
                                device="cuda")
        self.view = KvView(self.pool.data_ptr(), n_pages, page_size, n_layers, n_kv_heads, head_dim)
        self.ref, self.head_dim, self.kv_wide = C.byref(self.view), head_dim, n_kv_heads * head_dim
        self.max_pages = n_pages
        # identity-ish block table: sequence s owns pages s, s+max_seqs, ... (deliberately non-contiguous)
        bt = np.zeros((max_seqs, n_pages), np.int32)
        for s in range(max_seqs):
            ids = list(range(s, n_pages, max_seqs))
            bt[s, :len(ids)] = ids
        self.block_table = torch.from_numpy(bt).cuda()

    @classmethod
    def over(cls, pool, block_table=None):
        """the same over a caller's pool [page][layer][k|v][kv_head][slot][head_dim] and, for the operators that take it from here, block table"""
        assert pool.dim() == 6 and pool.shape[2] == 2 and pool.dtype == torch.bfloat16, "bfloat16 pool [page][layer][k|v][kv_head][slot][head_dim] expected"
        n_pages, n_layers, _, n_kv_heads, page_size, head_dim = pool.shape
        self = cls.__new__(cls)
        self.pool, self.block_table = pool, block_table
        self.view = KvView(_p(pool), n_pages, page_size, n_layers, n_kv_heads, head_dim)
        self.ref, self.head_dim, self.kv_wide = C.byref(self.view), head_dim, n_kv_heads * head_dim
        self.max_pages = n_pages if block_table is None else block_table.shape[1]
        return self

    def store(self, layer, K, V, pos, slot):
        check(_lib.lib().qie_kv_store(C.byref(self.view), layer, _p(K), _p(V), _p(pos), _p(slot),
                                      _p(self.block_table), self.max_pages, pos.numel(), _st()))


def launch_attn(Q, out, pool, layer, pos, slot, n_q_heads):
    """selfattention over the paged cache; row t attends to positions 0..pos[t]."""
    check(_lib.lib().qie_attention(C.byref(pool.view), layer, _p(Q), _p(out), _p(pos), _p(slot),
                                   _p(pool.block_table), pool.max_pages, pos.numel(), n_q_heads, _st()))


def sample_topk_bf16(logits_d, vocab, temperature, topk, seed, step=0):
    """helpers.cuh:157-166 -- returns the sampled token ids (one per row of logits)."""
    rows = logits_d.numel() // vocab
    # The kernel writes the tokens into page-locked memory itself: a device buffer, its clearing and a copy to pageable memory were 20 us of 72 (64 rows).
    out = torch.empty(rows, dtype=torch.int32, pin_memory=True)
    # the reference hands `step` to the kernel as the cuRAND subsequence (helpers.cuh:157-166)
    check(_lib.lib().qie_sample_topk_subseq(_p(logits_d), out.data_ptr(), rows, vocab, float(temperature), topk, seed, 0, step,
                                            _st()))
    torch.cuda.current_stream().synchronize()
    return out.numpy().copy()


def apply_repetition_penalty(logits_d, context_tokens_d, vocab, penalty):
    """layers_include.cuh:33 (declared, never defined in the reference): in place on one row of logits"""
    check(_lib.lib().qie_repetition_penalty(_p(logits_d), _p(context_tokens_d), context_tokens_d.numel(), vocab, float(penalty), _st()))


# ---- fast-numerics operators (tolerance parity, see include/qie_b200.h) ---------------------
def launch_matmul_fast(A, B, Cout, M, N, K):
    """tcgen05/TMEM/TMA GEMM: same contract as launch_matmul, results within 1e-2 (bf16)."""
    check(_lib.lib().qie_matmul_fast(_p(A), _p(B), _p(Cout), M, N, K, _st()))


def launch_attn_decode_fast(Q, out, pool, layer, pos, slot, n_q_heads, n_splits=0):
    """split-KV flash-decoding: one query token per row."""
    check(_lib.lib().qie_attention_decode_fast(C.byref(pool.view), layer, _p(Q), _p(out), _p(pos), _p(slot),
                                               _p(pool.block_table), pool.max_pages, pos.numel(), n_q_heads,
                                               n_splits, _st()))


def launch_attn_prefill_fast(Q, out, pool, layer, pos, slot, n_q_heads):
    """causal tiled attention for prefill rows: consecutive positions pos[0]+t of one sequence."""
    check(_lib.lib().qie_attention_prefill_fast(C.byref(pool.view), layer, _p(Q), _p(out), _p(pos), _p(slot),
                                                _p(pool.block_table), pool.max_pages, pos.numel(), n_q_heads,
                                                _st()))


def launch_attn_prefill_tc(Q, out, pool, layer, pos, slot, n_q_heads, variant=0):
    """the same on tcgen05 / TMEM (head_dim 128)."""
    check(_lib.lib().qie_attention_prefill_tc(C.byref(pool.view), layer, _p(Q), _p(out), _p(pos), _p(slot),
                                              _p(pool.block_table), pool.max_pages, pos.numel(), n_q_heads, variant,
                                              _st()))


# ---- a serving step over the paged cache (see qie_batch in include/qie_b200.h) ----------------
def _here(t):
    """a tensor on the current device (torch's raw name, or the public way where torch does not have it: see _st)"""
    try:
        dev = torch._C._cuda_getDevice()
    except AttributeError:
        dev = torch.cuda.current_device()
    assert t.get_device() == dev, "a tensor of another device than the current one, or of the host"


def _ints(t, n, name):
    """pointer of n int32"""
    assert t.dtype is torch.int32 and t.numel() >= n and t.is_cuda and t.is_contiguous(), f"{name}: {n} contiguous int32 on the device expected"
    return t.data_ptr()


def _rows(t):
    """(pointer, row stride) of rows of contiguous elements"""
    n, wide = t.shape
    stride, one = t.stride()
    assert t.is_cuda and (one == 1 or wide == 1), "device-resident rows of contiguous elements expected"
    return t.data_ptr(), stride if n > 1 else wide


class Batch:
    """A step of n_req requests and up to max_tokens rows: the arrays of qie_batch.  Those of the layout that are not given are made here; the
    object holds what it points to and is used step after step, its arrays changed in place."""

    def __init__(self, block_table, page_size, n_pages, n_req, max_tokens, *, slots=None, cached=None, n_new=None, free_ring=None, ring_in=None,
                 ring_out=None, q_start=None, kv_len=None, pos=None, slot=None, row=None, status=None):
        def ints(t, n):
            return torch.zeros(n, dtype=torch.int32, device=block_table.device) if t is None else t

        assert block_table.dim() == 2
        self.block_table, self.slots, self.cached, self.n_new, self.free_ring, self.ring_in = block_table, slots, cached, n_new, free_ring, ring_in
        self.ring_out, self.q_start, self.kv_len, self.status = ints(ring_out, 2), ints(q_start, n_req + 1), ints(kv_len, n_req), ints(status, 2)
        self.pos, self.slot, self.row = ints(pos, max_tokens), ints(slot, max_tokens), ints(row, max_tokens)
        self.work, self.heads, self.heads8, self.replaced, self.max_tokens = None, 0, 0, [], max_tokens
        b = self.view = BatchView(n_req=n_req, max_tokens=max_tokens, max_seqs=block_table.shape[0], max_pages=block_table.shape[1], n_pages=n_pages,
                                  page_size=page_size)
        for name, n in (("block_table", 0), ("slots", n_req), ("cached", n_req), ("n_new", n_req), ("free_ring", n_pages), ("ring_in", 2), ("ring_out", 2),
                        ("q_start", n_req + 1), ("kv_len", n_req), ("pos", max_tokens), ("slot", max_tokens), ("row", max_tokens), ("status", 2)):
            t = getattr(self, name)
            if t is not None:
                _here(t)
                setattr(b, name, _ints(t, n, name))
        self.ref = C.byref(b)

    def reserve(self, pool, n_q_heads):
        """the work area of launch_attn_batch and launch_attn_batch8; one call at a time uses it.  A smaller one from before is kept beside it: captured graphs and launches
        under way may have it."""
        eight = isinstance(pool, KvPool8)
        n = (_lib.lib().qie_attention_batch8_work if eight else _lib.lib().qie_attention_batch_work)(pool.ref, n_q_heads)
        if n == 0:  # a geometry that the operator refuses
            return
        if self.work is None or self.work.numel() < n:
            self.replaced.append(self.work)
            self.work = torch.empty(n, dtype=torch.uint8, device=self.block_table.device)
            self.view.work, self.view.work_bytes = self.work.data_ptr(), n
        if eight:  # the area's size hangs on the head size alone
            self.heads8 = max(self.heads8, pool.head_dim)
        else:
            self.heads = max(self.heads, pool.head_dim)


def launch_batch_layout(batch):
    _here(batch.block_table)
    check(_lib.lib().qie_batch_layout(batch.ref, _st()))


class Rope:
    """rotary frequencies on the device: freq, float64 radians a position of each pair"""
    KINDS = {"plain": 0, "linear": 1, "ntk": 2, "yarn": 3, "parts": 4}

    def __init__(self, freq, factor=1.0, neighbours=False):
        assert freq.dtype == torch.float64 and freq.dim() == 1
        _here(freq)
        self.freq, self.device = freq, freq.get_device()
        self.plan = RopePlan(_p(freq), 2 * freq.numel(), int(neighbours), float(factor))
        self.ref = C.byref(self.plan)

    @staticmethod
    def frequencies(rotated, base=1000000.0, kind="plain", scale=1.0, original=0, a=0.0, b=0.0):
        """host: (float64 array of rotated / 2, factor), see qie_rope_frequencies"""
        w, f = np.zeros(max(1, rotated // 2)), C.c_float()
        check(_lib.lib().qie_rope_frequencies(w.ctypes.data, C.byref(f), rotated, base, Rope.KINDS[kind], scale, original, a, b))
        return w, f.value


def launch_rope_rows(x, out, pos, rope, n_heads, head_dim):
    """rows [n_tok, n_heads * head_dim] -> out (may be x), token t at position pos[t]"""
    n, wide = x.shape
    assert x.dtype is out.dtype is torch.bfloat16 and x.shape == out.shape and wide == n_heads * head_dim, "bfloat16 rows of n_heads * head_dim expected"
    assert x.get_device() == out.get_device() == pos.get_device() == rope.device, "rows, positions and frequencies on one device expected"
    _here(x)
    check(_lib.lib().qie_rope_rows(*_rows(x), *_rows(out), rope.ref, _ints(pos, n, "pos"), n, n_heads, head_dim, _st()))


def launch_rope_store(q, k, v, q_out, pool, layer, pos, row, rope, n_q_heads):
    """q -> q_out, k and v -> the cache rows row[t] of the pool's layer"""
    (n, wide), (nk, kw), (nv, vw), (no, ow) = q.shape, k.shape, v.shape, q_out.shape
    (qs, q1), (ks, k1), (vs, v1), (os, o1) = q.stride(), k.stride(), v.stride(), q_out.stride()
    assert q.dtype is k.dtype is v.dtype is q_out.dtype is torch.bfloat16, "bfloat16 rows expected"
    assert n == nk == nv == no and wide == ow == n_q_heads * pool.head_dim and kw == vw == pool.kv_wide, "rows of the heads of as many tokens expected"
    assert (q1 == o1 == 1 or wide <= 1) and (k1 == v1 == 1 or kw <= 1), "rows of contiguous elements expected"
    assert q.get_device() == k.get_device() == v.get_device() == q_out.get_device() == pool.pool.get_device() == pos.get_device() == row.get_device() == rope.device, \
        "rows, pool, positions and frequencies on one device expected"
    _here(q)
    if n == 1:
        qs, os, ks, vs = wide, wide, kw, kw
    check(_lib.lib().qie_rope_store(pool.ref, layer, q.data_ptr(), qs, q_out.data_ptr(), os, k.data_ptr(), ks, v.data_ptr(), vs, rope.ref, _ints(pos, n, "pos"),
                                    _ints(row, n, "row"), n, n_q_heads, _st()))


def launch_attn_batch(Q, out, pool, layer, batch, n_q_heads, window=0, scale=0.0):
    """attention of the batch's rows over the pool, ragged over its requests (fast numerics)"""
    assert Q.dtype is out.dtype is torch.bfloat16 and Q.shape == out.shape == (batch.max_tokens, n_q_heads * pool.head_dim), "bfloat16 rows of the batch expected"
    if batch.heads < pool.head_dim:
        batch.reserve(pool, n_q_heads)
    assert Q.get_device() == out.get_device() == pool.pool.get_device() == batch.block_table.get_device(), "rows, pool and batch on one device expected"
    _here(Q)
    check(_lib.lib().qie_attention_batch(pool.ref, layer, batch.ref, *_rows(Q), *_rows(out), n_q_heads, window, scale, _st()))


class KvPool8:
    """the same pool in 8 bits (qie_kv8_view): codes [page][layer][k|v][kv_head][slot][head_dim] of torch.float8_e4m3fn or torch.int8, and scale bytes of the same shape without the last"""
    CODES = {torch.float8_e4m3fn: 0, torch.int8: 1}

    def __init__(self, n_pages, page_size, n_layers, n_kv_heads, head_dim, dtype=torch.float8_e4m3fn):
        shape = (n_pages, n_layers, 2, n_kv_heads, page_size)
        self._over(torch.zeros(*shape, head_dim, dtype=torch.uint8, device="cuda").view(dtype), torch.zeros(shape, dtype=torch.uint8, device="cuda"))

    @classmethod
    def over(cls, codes, scale):
        """the same over a caller's arrays"""
        self = cls.__new__(cls)
        self._over(codes, scale)
        return self

    def _over(self, codes, scale):
        assert codes.dtype in KvPool8.CODES and codes.dim() == 6 and codes.shape[2] == 2, "codes [page][layer][k|v][kv_head][slot][head_dim] of float8_e4m3fn or int8 expected"
        assert scale.dtype is torch.uint8 and scale.shape == codes.shape[:5] and scale.get_device() == codes.get_device(), "a uint8 scale for each vector, beside them, expected"
        n_pages, n_layers, _, n_kv_heads, page_size, head_dim = codes.shape
        _here(codes)
        self.codes, self.scale, self.head_dim, self.kv_wide, self.device = codes, scale, head_dim, n_kv_heads * head_dim, codes.get_device()
        self.view = Kv8View(_p(codes), _p(scale), n_pages, page_size, n_layers, n_kv_heads, head_dim, KvPool8.CODES[codes.dtype])
        self.ref = C.byref(self.view)


def launch_rope_store8(q, k, v, q_out, pool, layer, pos, row, rope, n_q_heads):
    """q -> q_out, k and v -> codes and scales in the cache rows row[t] of the pool's layer.  rope None: k as it is; then q, q_out and pos are None and n_q_heads 0"""
    (n, kw), (nv, vw) = k.shape, v.shape
    (ks, k1), (vs, v1) = k.stride(), v.stride()
    assert k.dtype is v.dtype is torch.bfloat16 and n == nv and kw == vw == pool.kv_wide and k1 == v1 == 1, "bfloat16 rows of the heads of as many tokens expected"
    dev = pool.device
    assert k.get_device() == v.get_device() == row.get_device() == dev, "rows and pool on one device expected"
    _here(k)
    if n == 1:
        ks, vs = kw, kw
    if rope is None:
        assert q is None and q_out is None and pos is None and n_q_heads == 0, "queries and positions without a rotation"
        check(_lib.lib().qie_rope_store8(pool.ref, layer, None, 0, None, 0, k.data_ptr(), ks, v.data_ptr(), vs, None, None, _ints(row, n, "row"), n, 0, _st()))
        return
    (nq, wide), (no, ow) = q.shape, q_out.shape
    (qs, q1), (os, o1) = q.stride(), q_out.stride()
    assert q.dtype is q_out.dtype is torch.bfloat16 and nq == no == n and wide == ow == n_q_heads * pool.head_dim, "bfloat16 rows of the heads of as many tokens expected"
    assert q1 == o1 == 1 or wide <= 1, "rows of contiguous elements expected"
    assert q.get_device() == q_out.get_device() == pos.get_device() == rope.device == dev, "rows, positions and frequencies on one device expected"
    if n == 1:
        qs, os = wide, wide
    check(_lib.lib().qie_rope_store8(pool.ref, layer, q.data_ptr(), qs, q_out.data_ptr(), os, k.data_ptr(), ks, v.data_ptr(), vs, rope.ref, _ints(pos, n, "pos"),
                                     _ints(row, n, "row"), n, n_q_heads, _st()))


def launch_kv8_read(pool, layer, row, k, v):
    """cache rows row[i] of the pool's layer -> rows k[i], v[i] (either may be None) of the values that they stand for"""
    n, out = row.numel(), []
    for x in (k, v):
        if x is None:
            out += [None, 0]
            continue
        (m, wide), (stride, one) = x.shape, x.stride()
        assert x.dtype is torch.bfloat16 and m == n and wide == pool.kv_wide and one == 1 and x.get_device() == pool.device, \
            "bfloat16 rows of the pool's heads, one for each index, beside it expected"
        out += [x.data_ptr(), stride if n > 1 else wide]
    assert row.get_device() == pool.device, "rows and pool on one device expected"
    _here(row)
    check(_lib.lib().qie_kv8_read(pool.ref, layer, _ints(row, n, "row"), n, *out, _st()))


def launch_attn_batch8(Q, out, pool, layer, batch, n_q_heads, window=0, scale=0.0):
    """launch_attn_batch over a pool in 8 bits"""
    assert Q.dtype is out.dtype is torch.bfloat16 and Q.shape == out.shape == (batch.max_tokens, n_q_heads * pool.head_dim), "bfloat16 rows of the batch expected"
    if batch.heads8 < pool.head_dim:
        batch.reserve(pool, n_q_heads)
    assert Q.get_device() == out.get_device() == pool.device == batch.block_table.get_device(), "rows, pool and batch on one device expected"
    _here(Q)
    check(_lib.lib().qie_attention_batch8(pool.ref, layer, batch.ref, *_rows(Q), *_rows(out), n_q_heads, window, scale, _st()))


class LogitRules:
    """the lists and parameters of qie_logit_rules; None: no such rule"""

    def __init__(self, tok_start=None, tokens=None, *, gen_start=None, repetition=None, presence=None, frequency=None, bias_start=None, bias_ids=None, bias=None,
                 mask=None, mask_row=None):
        self.held = dict(tok_start=tok_start, tokens=tokens, gen_start=gen_start, repetition=repetition, presence=presence, frequency=frequency,
                         bias_start=bias_start, bias_ids=bias_ids, bias=bias, mask=mask, mask_row=mask_row)
        self.n_rows = self.device = None  # rows that every list has, and where they are
        for name, t in self.held.items():
            if t is None:
                continue
            assert t.dtype == (torch.float32 if name in ("repetition", "presence", "frequency", "bias") else torch.int32), f"{name}: {t.dtype}"
            _here(t)
            self.device = t.get_device()
            n = {"tokens": None, "bias_ids": None, "bias": None, "tok_start": t.numel() - 1, "bias_start": t.numel() - 1,
                 "mask": t.shape[0] if mask_row is None else None}.get(name, t.numel())
            if n is not None:
                self.n_rows = n if self.n_rows is None else min(self.n_rows, n)
        assert mask is None or mask.dim() == 2, "mask [masks][words]"
        assert bias is None or (bias_ids is not None and bias_ids.numel() == bias.numel()), "a bias for each id"
        r = self.view = LogitRulesView(**{name: _p(t) for name, t in self.held.items() if t is not None})
        r.n_tokens, r.n_bias = 0 if tokens is None else tokens.numel(), 0 if bias is None else bias.numel()
        r.n_masks, r.mask_words = (0, 0) if mask is None else mask.shape
        self.ref = C.byref(r)


def launch_logits(logits, out, rules):
    """the rules over rows [n_rows, vocab] of bfloat16 or float32 logits -> out (may be logits)"""
    (n, vocab), kind = logits.shape, logits.dtype
    assert kind is out.dtype and out.shape == logits.shape and (kind is torch.bfloat16 or kind is torch.float32), "bfloat16 or float32 logits, and out like them"
    assert rules.n_rows is None or rules.n_rows >= n, "rules for fewer rows"
    assert logits.get_device() == out.get_device() and (rules.device is None or rules.device == logits.get_device()), "logits and rules on one device expected"
    _here(logits)
    check(_lib.lib().qie_logits_process(*_rows(logits), *_rows(out), int(kind is torch.float32), n, vocab, rules.ref, _st()))
