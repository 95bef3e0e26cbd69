"""Masks of drafted trees with bits at and beyond the number of drafts: they name no draft, so neither what a row sees nor where it stands
changes with them (a draft stands at the length plus the number of other drafts it sees)."""
import pytest
import torch

from tests.test_gpu_tree import check_tree, make_cache, randn, random_tree

pytestmark = pytest.mark.gpu


def slopes_of(Hq):
    return torch.exp2(-4.0 * torch.arange(1, Hq + 1, device="cuda", dtype=torch.float32) / Hq)


@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,D,kb", [(1, 4, 4, 128, 64), (5, 8, 2, 128, 256), (16, 4, 1, 64, 64), (40, 4, 1, 128, 64), (63, 4, 2, 128, 256), (3, 2, 2, 256, 64)])
def test_bits_beyond_the_drafts_change_nothing(T, Hq, Hkv, D, kb, alibi):
    lens = [0, 70, 333]
    cache, g = make_cache(3, Hq, Hkv, D, kb, lens, seed=T)
    q, k, v = randn(g, 3, T, Hq, D).half(), randn(g, 3, T, Hkv, D).half(), randn(g, 3, T, Hkv, D).half()
    slopes = slopes_of(Hq) if alibi else None
    clean = torch.stack([random_tree(T, 7 * T + b) for b in range(3)]).cuda()
    low = (1 << T) - 1
    stray = clean.clone()
    stray[:, ::2] |= ~low                                 # every other draft, so that rows and tokens of both kinds meet
    stray[1] |= 1 << T if T < 63 else -1 << 63             # the first bit that names none, in a whole row
    want = cache.verify(0, q, k, v, clean, slopes=slopes)
    check_tree(want, cache, q, k, v, clean, slopes=slopes)
    assert torch.equal(cache.verify(0, q, k, v, stray, slopes=slopes), want)


@pytest.mark.parametrize("T", [2, 16, 64])
def test_every_draft_sees_every_draft(T):
    cache, g = make_cache(2, 4, 2, 128, 64, [130, 20], seed=T)
    q, k, v = randn(g, 2, T, 4, 128).half(), randn(g, 2, T, 2, 128).half(), randn(g, 2, T, 2, 128).half()
    slopes = slopes_of(4)
    named = torch.full((T,), (1 << T) - 1 if T < 64 else -1, dtype=torch.int64, device="cuda")
    out = cache.verify(0, q, k, v, torch.full((T,), -1, dtype=torch.int64, device="cuda"), slopes=slopes)
    check_tree(out, cache, q, k, v, named, slopes=slopes)
