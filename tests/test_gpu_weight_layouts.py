"""Accumulated weights that lie head by head, or apart with gaps: the same numbers as in a dense tensor, and nothing between the rows is touched."""
import pytest
import torch

from tests.test_gpu_tree import make_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("order", ["head by head", "gaps"])
def test_strided_weights(order):
    from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module as ops
    B, Hq, Hkv, D, S = 3, 8, 2, 64, 200
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    cache, _ = make_cache(B, Hq, Hkv, D, 64, [S, 130, 70], seed=1, track_weights=True)
    cap = cache.max_seq_len
    shape, stride = (B, Hkv, cap), (cap + 3, (cap + 3) * B, 1) if order == "head by head" else ((cap + 5) * Hkv + 2, cap + 5, 1)
    pool = torch.full((shape[0] * shape[1] * (cap + 5) + 64,), 7.0, device="cuda")
    view, dense = pool.as_strided(shape, stride, 9), torch.zeros(shape, device="cuda")
    view.zero_()
    q, k, lse = rn(B, S, Hq, D), rn(B, S, Hkv, D), torch.full((B, Hq, S), 3.0, device="cuda")
    probs = torch.rand(B, Hq, (cap + 7) // 8 * 8, generator=g, device="cuda").half()
    for w in (view, dense):
        assert ops.attention_weights(q, k, lse, seq_lens=cache.seq_lens[0], out=w) is w
        assert ops.accumulate_weights(w, probs, cache.seq_lens[0], decay=0.5) is w
    assert torch.equal(view, dense) and dense.abs().sum() > 0
    twin, _ = make_cache(B, Hq, Hkv, D, 64, [S, 130, 70], seed=1, track_weights=True)
    kept = [ops.evict(c.prepared(0), w, 64, sinks=2, recent=10) for c, w in ((cache, view), (twin, dense))]
    assert torch.equal(*kept) and torch.equal(view, dense) and torch.equal(cache.seq_lens[0], twin.seq_lens[0])
    hidden = torch.ones_like(pool, dtype=torch.bool)
    hidden.as_strided(shape, stride, 9).fill_(False)
    assert (pool[hidden] == 7.0).all()
