"""Outputs that share memory with an input, and weights whose rows share memory: refused before anything is launched (CPU).  Workgroups
write their rows while others still read theirs, and add to rows of their own only where the rows are apart."""
import ctypes

import pytest
import torch

from alignedkv_amd import _lib
from alignedkv_amd.extension import serving_ops
from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
from tests.test_serving_refusals import Z, layer, lib, mem, prompt, says  # noqa: F401


@pytest.fixture
def dry(monkeypatch):
    """The Python layer on host tensors: the checks of type, shape and device are left out, a call is noted instead of launched."""
    calls = []
    monkeypatch.setattr(serving_ops, "_tensor", lambda name, t, *a, **kw: t)
    monkeypatch.setattr(serving_ops, "_call", lambda fn, device, *args: calls.append(fn.__name__))
    return calls


def halves(*shape):
    return torch.zeros(shape, dtype=torch.half)


def floats_over(t, *shape):
    """fp32 memory that begins inside the storage of t."""
    return t.flatten().view(torch.float32)[8:8 + torch.Size(shape).numel()].view(shape)


def test_weights_of_a_prompt_that_overlap_what_is_read(dry):
    B, S, H, D = 2, 16, 4, 64
    q, k, lse = halves(B, S, H, D), halves(B, S, H, D), torch.zeros(B, H, S)
    for out in (lse, lse[:, :, :S], floats_over(q, B, H, S), floats_over(k, B, H, S)):
        with pytest.raises(RuntimeError, match="out: overlaps an input"):
            cuda_module.attention_weights(q, k, lse, out=out)
    slopes = torch.zeros(64)
    with pytest.raises(RuntimeError, match="out: overlaps an input"):
        cuda_module.attention_weights(q[:1, :1], k[:1, :1], lse[:1, :, :1], slopes=slopes[:H], out=slopes[2:2 + H].view(1, H, 1))
    assert not dry
    out = torch.zeros(B, H, S)
    assert cuda_module.attention_weights(q, k, lse, out=out) is out and dry == ["akv_attention_weights"]


def test_sums_that_overlap_the_probabilities(dry):
    probs, lens, weights = halves(2, 4, 64), torch.zeros(2, dtype=torch.int32), torch.zeros(2, 2, 32)
    with pytest.raises(RuntimeError, match="out: overlaps an input"):
        cuda_module.accumulate_weights(weights, probs, lens, out=floats_over(probs, 2, 2, 32))
    with pytest.raises(RuntimeError, match="out: overlaps an input"):
        cuda_module.accumulate_weights(floats_over(probs, 2, 2, 32), probs, lens)
    assert not dry
    cuda_module.accumulate_weights(weights, probs, lens)
    assert dry == ["akv_accumulate_weights"]


def test_attention_into_what_it_reads(dry):
    B, S, H, D = 1, 16, 2, 64
    q, k, v = halves(B, S, H, D), halves(B, S, H, D), halves(B, S, H, D)
    big = torch.zeros(B * S * H * D // 2 + 64, dtype=torch.int32)
    for kw in (dict(documents=big[:S].view(1, S)), dict(seq_lens=big[40:41]), dict(prefix_lens=big[-1:]), dict(slopes=big.view(torch.float32)[8:8 + H])):
        over = big.view(torch.half)[:q.numel()].view(q.shape) if "prefix_lens" not in kw else big.view(torch.half)[128:].view(q.shape)
        with pytest.raises(RuntimeError, match="out: overlaps an input"):
            cuda_module.prefill_attention(q, k, v, out=over, **kw)
    c = [torch.zeros(1, H, 1, D, 64, dtype=torch.uint8)] + [torch.zeros(1, H, 1, D, 32, dtype=torch.uint8) for _ in range(2)]
    w = [torch.zeros(1, H, 64, D, dtype=torch.uint8)] + [torch.zeros(1, H, 64, D // 2, dtype=torch.uint8) for _ in range(2)]
    rest = halves(1, 64, H, D), halves(1, 64, H, D)
    made = cuda_module.prepare_layer(c, w, torch.zeros(1, 1, H, D, dtype=torch.uint8), torch.zeros(1, 1, H, D, dtype=torch.uint8), *rest, torch.zeros(1, dtype=torch.int32))
    anc = torch.ones(S * H * D, dtype=torch.int64)
    d = [t[:, :4] for t in (q, k, v)]
    for out in (rest[0][:, :4], rest[1][:, 8:12], c[0].flatten().view(torch.half)[:4 * H * D].view(1, 4, H, D), w[1].flatten().view(torch.half)[-4 * H * D:].view(1, 4, H, D),
                anc.view(torch.half)[:4 * H * D].view(1, 4, H, D), q[:, 2:6]):
        with pytest.raises(RuntimeError, match="out: overlaps an input"):
            cuda_module.tree_attention(made, *d, anc[:4], out=out)
    assert not dry


def test_the_c_entries_refuse_them_too(lib, mem):  # noqa: F811
    d = prompt(mem, bsz=1, seqlen=2, q=mem, k=mem + 1024, v=mem + 2048, **{n + "_stride": (512, 256, 64) for n in "qkv"})       # 1 KB each
    free = mem + 3 * 1024
    for w in (free, free + 28, mem + 1020, mem + 2044):      # lse: 4 heads of 2 rows, 32 bytes
        says(lib, lib.akv_attention_weights(ctypes.byref(d), free, 0, w, 8, 2, 0, Z), "attention_weights", "overlap")
    for out in (mem, mem + 1008, mem + 2032, mem + 3056):
        says(lib, lib.akv_prefill_attention(ctypes.byref(d), out, None, 1, None, 0, Z), "prefill_attention", "overlap")
    says(lib, lib.akv_prefill_attention(ctypes.byref(prompt(mem, seqlen=1, bsz=1, v=mem + 1024)), mem + 2048, mem + 2048, 1, None, 0, Z), "overlap")    # out and lse
    acc = dict(weights=mem, probs=mem + 512, out=mem)        # 2 heads of 64 weights (512 bytes); 4 heads of 64 probabilities (512)
    for kw in (dict(out=mem + 4), dict(out=mem + 508), dict(out=mem + 1020), dict(weights=mem + 768, out=mem + 768), dict(weights=mem + 4, out=mem)):
        a = dict(acc, **kw)
        says(lib, lib.akv_accumulate_weights(a["weights"], 128, 64, a["probs"], 64, mem, a["out"], 128, 64, 1, 4, 2, 64, 1.0, Z), "accumulate_weights", "overlap")
    a, b = layer(mem, bsz=1, n_kv_heads=1), _lib.CacheLayer(*[mem + 1024 + 256 * i for i in range(11)], 1, 1, 3, 192, 64, 64)
    for to in (mem + 4, mem + 764):                          # weights: one row of 192
        says(lib, lib.akv_evict(ctypes.byref(a), ctypes.byref(b), mem, 192, 192, to, 192, 192, 192, mem + 2048, 64, 0, 0, mem, 1 << 30, Z), "evict", "overlap")
