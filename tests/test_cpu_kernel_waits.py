"""Kernels of attention over a cache in 8 bits start with a wait for the grids before them, whatever the call (csrc/launch.h): no load of theirs is in front of it.  Read off the source: no GPU."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qwen_inference_engine_b200", "csrc")


def kernels(name):
    src = re.sub(r" *//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    for m in re.finditer(r"__global__ [^;{]*?\b(\w+_kernel)\([^{]*\) \{\n(.*?)\n\}\n", src, flags=re.S):
        yield m.group(1), m.group(2)


@pytest.mark.parametrize("name,n", [("attn_batch8.cu", 3), ("attn_batch_split.cuh", 1), ("kv8_store.cu", 2)])
def test_waits_whatever_the_call(name, n):
    found = list(kernels(name))
    assert len(found) == n
    for kernel, body in found:
        lines = body.split("\n")
        assert lines.count("  pdl_wait();") == 1 and body.count("pdl_wait()") == 1, kernel  # one, under no condition
        at = lines.index("  pdl_wait();")
        assert lines.index("  pdl_trigger();") > at, kernel
        early = "\n".join(lines[:at])
        assert not re.search(r"\ba\.(q|out|work|status|q_start|kv_len|slots|block_table|pos|row|k|v|freq)\b|\bkv\.(codes|scale)\b|find_stretch|join_parts", early), kernel


def test_shared_arrays_have_the_alignment_of_their_accesses():
    """no __shared__ array of elements below 16 bytes, without an alignment of its own, that the file goes through 16 bytes at a time"""
    for name in ("attn_batch8.cu", "attn_batch_split.cuh", "kv8_store.cu"):
        src = re.sub(r" *//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        small = re.findall(r"__shared__ (?:bf16|float|int|uint8_t|uint32_t|long long|unsigned long long) (\w+)\[", src)
        for a in small:
            names = {a} | set(re.findall(r"\* *(\w+) = (?:reinterpret_cast<[^>]*>\()?%s\b" % a, src))
            for n in names:
                assert not re.search(r"reinterpret_cast<(?:const )?(?:uint4|float4|int4|uint2|float2)\*>\(&?%s\b" % n, src), (name, a)
