"""Ragged batches whose sequences get different numbers of splits, more sequences than a wave has lanes, and bounds of every kind."""
import math

import pytest
import torch

from tests.test_gpu_tree import check_tree, make_cache, randn, random_tree

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("lens,T,Hq,Hkv,D,kb", [
    ([5000, 70, 0, 1, 64, 2300], 3, 2, 1, 64, 64), ([63, 4100], 33, 4, 2, 128, 256), ([0, 0, 0], 2, 2, 2, 128, 64), ([9000], 40, 4, 1, 128, 256),
    ([1, 3000, 640], 64, 4, 1, 128, 64), ([700, 200, 200, 200, 200, 200, 200, 200, 1500], 9, 8, 8, 256, 64), ([64, 128, 192], 64, 6, 1, 128, 256)])
def test_ragged_batches(lens, T, Hq, Hkv, D, kb):
    B = len(lens)
    cache, g = make_cache(B, Hq, Hkv, D, kb, lens, seed=T)
    q, k, v = randn(g, B, T, Hq, D).half(), randn(g, B, T, Hkv, D).half(), randn(g, B, T, Hkv, D).half()
    anc = random_tree(T, T).cuda()
    for bound in (None, cache.max_seq_len, 0, min(100, cache.max_seq_len)):          # a bound that is too low costs time, not tokens
        check_tree(cache.verify(0, q, k, v, anc, bound=bound), cache, q, k, v, anc)


@pytest.mark.parametrize("B", [64, 65, 200, 300, 600])
def test_more_sequences_than_lanes(B):
    lens = [(37 * b) % 400 if b % 7 else 0 for b in range(B)]
    lens[-1] = 1300
    cache, g = make_cache(B, 2, 1, 64, 64, lens, seed=B)
    q, k, v = randn(g, B, 2, 2, 64).half(), randn(g, B, 2, 1, 64).half(), randn(g, B, 2, 1, 64).half()
    anc = torch.tensor([1, 3], device="cuda")
    check_tree(cache.verify(0, q, k, v, anc), cache, q, k, v, anc)


def test_lengths_that_change_between_replays_of_a_graph():
    lens = [130, 900, 1]
    cache, g = make_cache(3, 4, 2, 128, 64, lens, seed=9)
    q, k, v = randn(g, 3, 4, 4, 128).half(), randn(g, 3, 4, 2, 128).half(), randn(g, 3, 4, 2, 128).half()
    anc = torch.tensor([1, 3, 7, 15], device="cuda")
    run = lambda: cache.verify(0, q, k, v, anc, bound=cache.max_seq_len)      # noqa: E731
    run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for now in (lens, [64, 10, 0], [0, 0, 0], [130, 900, 1], [128, 320, 1]):
        cache.seq_lens[0].copy_(torch.tensor(now, dtype=torch.int32))         # (shorter than what is stored)
        for i, n in enumerate(now):
            cache.restk[0][i].fill_(0.25)
            cache.restv[0][i].fill_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, run())
        check_tree(out, cache, q, k, v, anc)
    assert math.isfinite(out.float().abs().max().item())
