"""Layouts of accumulated weights, fp32 [sequences, KV heads, tokens]: rows that share memory are refused (workgroups add to them without
atomics), rows that are apart are taken in any order of sequences and heads (CPU)."""
import ctypes

import pytest
import torch

from alignedkv_amd import _lib
from alignedkv_amd.extension import serving_ops
from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
from tests.test_serving_overlaps import dry, halves  # noqa: F401
from tests.test_serving_refusals import Z, layer, lib, mem, prompt, says  # noqa: F401

POOL = 4096
APART = [((2, 3, 16), (48, 16, 1)), ((2, 3, 16), (16, 32, 1)), ((2, 3, 16), (100, 20, 1)), ((2, 3, 16), (17, 40, 1)), ((1, 3, 16), (0, 16, 1)), ((2, 1, 16), (16, 0, 1)),
         ((1, 1, 16), (0, 0, 1)), ((1, 1, 16), (5, 3, 1)), ((4, 2, 16), (16, 64, 1)), ((2, 2, 1), (2, 1, 7))]
SHARED = [((2, 2, 16), (16, 16, 1)), ((2, 3, 16), (32, 16, 1)), ((2, 3, 16), (16, 24, 1)), ((2, 3, 16), (0, 16, 1)), ((2, 3, 16), (48, 0, 1)), ((2, 1, 16), (8, 16, 1)),
          ((1, 2, 16), (48, 15, 1)), ((3, 2, 16), (16, 47, 1)), ((2, 3, 16), (48, 16, 2)), ((2, 2, 16), (33, 17, 0))]


@pytest.mark.parametrize("shape,stride", APART)
def test_rows_that_are_apart_are_taken(dry, shape, stride):  # noqa: F811
    B, H, n = shape
    w = torch.zeros(POOL).as_strided(shape, stride)
    assert len({w[b, h, t].data_ptr() for b in range(B) for h in range(H) for t in range(n)}) == B * H * n
    assert serving_ops._weights("weights", w, B, H, n, None) is w
    lens = torch.zeros(B, dtype=torch.int32)
    assert cuda_module.accumulate_weights(w, halves(B, 2 * H, 64), lens) is w
    assert cuda_module.attention_weights(halves(B, n, H, 64), halves(B, n, H, 64), torch.zeros(B, H, n), out=w) is w


@pytest.mark.parametrize("shape,stride", SHARED)
def test_rows_that_share_memory_are_refused(dry, shape, stride):  # noqa: F811
    B, H, n = shape
    w, lens = torch.zeros(POOL).as_strided(shape, stride), torch.zeros(B, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="weights: rows must be dense and must not overlap"):
        cuda_module.accumulate_weights(w, halves(B, 2 * H, 64), lens)
    with pytest.raises(RuntimeError, match="out: rows must be dense"):
        cuda_module.accumulate_weights(torch.zeros(shape), halves(B, 2 * H, 64), lens, out=w)
    with pytest.raises(RuntimeError, match="out: rows must be dense"):
        cuda_module.attention_weights(halves(B, n, H, 64), halves(B, n, H, 64), torch.zeros(B, H, n), out=w)
    assert not dry


def test_what_is_too_short(dry):  # noqa: F811
    with pytest.raises(RuntimeError, match="rows of 15 weights for 16 tokens"):
        serving_ops._weights("weights", torch.zeros(2, 2, 15), 2, 2, 16, None)


@pytest.mark.parametrize("shape,stride", [c for c in SHARED if c[1][2] == 1])
def test_the_c_entries_refuse_them(lib, mem, shape, stride):  # noqa: F811
    (B, H, n), (sb, sh, _) = shape, stride
    big = mem + 2048
    d = prompt(mem, bsz=B, seqlen=n, n_q_heads=H, n_kv_heads=H, **{x + "_stride": (0, 0, 0) for x in "qkv"})
    says(lib, lib.akv_attention_weights(ctypes.byref(d), mem + 512, 0, big, sb, sh, 0, Z), "attention_weights", "rows")
    says(lib, lib.akv_accumulate_weights(mem, n * H, n, mem, 64, mem, big, sb, sh, B, H, H, n, 1.0, Z), "accumulate_weights", "rows")
    a = layer(mem, bsz=B, n_kv_heads=H, max_seq_len=16)
    b = _lib.CacheLayer(*[mem + 1024 + 256 * i for i in range(11)], B, H, 3, 192, 64, 64)
    says(lib, lib.akv_evict(ctypes.byref(a), ctypes.byref(b), mem, n * H, n, big, sb, sh, 127, mem, 64, 0, 0, mem, 1 << 30, Z), "evict", "rows")          # (rows of 127 there)
    says(lib, lib.akv_evict(ctypes.byref(a), ctypes.byref(a), big, sb, sh, big, sb, sh, 16, mem, 64, 0, 0, mem, 1 << 30, Z), "evict", "rows")
