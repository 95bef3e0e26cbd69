"""Eviction by accumulated attention weight: whole numbers and bytes, so everything is compared for equality."""
import math

import pytest
import torch

from tests.serving_forms import cached_tokens
from tests.test_gpu_tree import make_cache, randn

pytestmark = pytest.mark.gpu


def chosen(w, n, keep, sinks, recent):
    """The definition, one (sequence, head): w fp32 on the CPU."""
    flushed = n // 64 * 64
    if flushed <= keep:
        return list(range(flushed))
    must = [j for j in range(flushed) if j < sinks or j >= n - recent]
    rest = [j for j in range(flushed) if j not in set(must)]
    value = lambda j: -math.inf if math.isnan(w[j]) else w[j]  # noqa: E731
    rest.sort(key=lambda j: (math.isnan(w[j]), -value(j), j))
    return sorted(must + rest[:keep - len(must)])


def fill_weights(cache, g, kind):
    w = cache.weights[0]
    if kind == "spread":
        w.copy_(torch.rand(w.shape, generator=g, device="cuda") ** 6 * 100)
    elif kind == "ties":
        w.copy_((torch.rand(w.shape, generator=g, device="cuda") * 4).floor() * 0.25 - 0.25)     # -0.25, 0, 0.25, 0.5
        w[:, :, 3::7] *= -1.0                                                                     # both zeros, both signs
    elif kind == "equal":
        w.fill_(0.125)
    else:
        w.copy_(torch.randn(w.shape, generator=g, device="cuda") * 1e-3)
        w[:, :, 5::11] = math.nan
        w[:, :, 2::13] = math.inf
        w[:, :, 8::17] = -math.inf


@pytest.mark.parametrize("kind", ["spread", "ties", "equal", "odd"])
@pytest.mark.parametrize("kb,Hkv,D,keep,sinks,recent", [(64, 2, 64, 64, 0, 0), (256, 2, 128, 192, 4, 100), (64, 1, 256, 320, 0, 320), (256, 3, 64, 256, 256, 0),
                                                        (256, 1, 128, 1024, 7, 33)])
@pytest.mark.parametrize("in_place", [True, False])
def test_what_is_kept_and_where_it_goes(kind, kb, Hkv, D, keep, sinks, recent, in_place):
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    lens = [0, 1, 64, 200, 320, 389, 1500, 4200]
    cache, g = make_cache(len(lens), 2 * Hkv, Hkv, D, kb, lens, seed=keep, track_weights=True)
    fill_weights(cache, g, kind)
    w = cache.weights[0].clone()
    old = [[cached_tokens(cache, 0, b, h) for h in range(Hkv)] for b in range(len(lens))]
    colmax = cache.k_colmax[0].clone()
    before = [t.clone() for t in (*cache.k_planes[0], *cache.v_planes[0], cache.restk[0], cache.restv[0], cache.seq_lens[0], cache.weights[0])]
    to = None if in_place else RaggedGQACache(1, len(lens), keep + 64, 2 * Hkv, Hkv, D, k_block=kb, track_weights=True)
    if to is not None:
        to.weights[0].fill_(-1)
    kept = cache.evict(0, keep, sinks=sinks, recent=recent, into=to)
    new = cache if in_place else to
    if not in_place:
        for a, t in zip(before, (*cache.k_planes[0], *cache.v_planes[0], cache.restk[0], cache.restv[0], cache.seq_lens[0], cache.weights[0])):
            assert torch.equal(a.view(torch.uint8), t.view(torch.uint8)), "the source changed"
    assert torch.equal(new.k_colmax[0], colmax)
    for b, n in enumerate(lens):
        f = n // 64 * 64
        have = min(keep, f)
        assert int(new.seq_lens[0][b]) == have + n - f
        for h in range(Hkv):
            want = chosen(w[b, h].cpu().tolist(), n, keep, sinks, recent)
            assert kept[b, h].tolist() == want + [-1] * (keep - have), f"sequence {b} head {h}"
            at = torch.tensor(want + list(range(f, n)), device="cuda", dtype=torch.long)
            k, v = cached_tokens(new, 0, b, h)
            assert torch.equal(k, old[b][h][0][at]) and torch.equal(v, old[b][h][1][at]), f"sequence {b} head {h}"
            if not in_place or f > keep:
                left = len(at)
                assert torch.equal(new.weights[0][b, h, :left].view(torch.int32), w[b, h, at].view(torch.int32))
                assert (new.weights[0][b, h, left:] == 0).all()
            else:
                assert torch.equal(new.weights[0][b, h].view(torch.int32), w[b, h].view(torch.int32))


@pytest.mark.parametrize("kb", [64, 256])
def test_decoding_goes_on_as_on_a_cache_that_holds_the_kept_tokens(kb):
    """decode steps after an eviction in place, over planes whose unused places hold old tokens, against a fresh cache filled with
    the kept tokens: the same bits."""
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    lens, Hq, Hkv, D = [700, 450, 130], 8, 2, 128
    cache, g = make_cache(3, Hq, Hkv, D, kb, lens, room=120, seed=1, stale=False, track_weights=True)
    cache.weights[0].copy_(torch.rand(cache.weights[0].shape, generator=g, device="cuda"))
    cache.evict(0, 192, sinks=4, recent=40)
    fresh = RaggedGQACache(1, 3, cache.max_seq_len, Hq, Hkv, D, k_block=kb)
    for b in range(3):
        n = int(cache.seq_lens[0][b])
        kv = [cached_tokens(cache, 0, b, h) for h in range(Hkv)]
        fresh.prefill(0, b, torch.stack([t[0] for t in kv], 1)[None], torch.stack([t[1] for t in kv], 1)[None])
        assert n == min(192, lens[b] // 64 * 64) + lens[b] % 64
    fresh.k_colmax[0].copy_(cache.k_colmax[0])
    fresh.v_colmax[0].copy_(cache.v_colmax[0])
    for step in range(80):                       # crosses a flush
        q, k, v = randn(g, 3, 1, Hq, D).half(), randn(g, 3, 1, Hkv, D).half(), randn(g, 3, 1, Hkv, D).half()
        a, b = cache.decode(0, q, k, v, bound=300), fresh.decode(0, q, k, v, bound=300)
        assert torch.equal(a, b), f"step {step}"
    # the weights went on from what was kept (the third sequence kept everything: its row was not touched)
    n = cache.seq_lens[0].tolist()
    for b in range(2):
        assert (cache.weights[0][b, :, n[b] - 1] > 0).all() and (cache.weights[0][b, :, n[b]:] == 0).all()


def test_evict_captured_and_replayed():
    from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
    lens = [500, 333]
    cache, g = make_cache(2, 4, 2, 64, 64, lens, seed=6, track_weights=True)
    to, _ = make_cache(2, 4, 2, 64, 64, [1, 1], room=300, seed=7, track_weights=True)
    twin, _ = make_cache(2, 4, 2, 64, 64, [1, 1], room=300, seed=7, track_weights=True)
    layers = cache.prepared(0), to.prepared(0)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        kept = cuda_module.evict(layers[0], cache.weights[0], 128, recent=64, into=layers[1], into_weights=to.weights[0])
    for r in range(4):
        cache.weights[0].copy_(torch.rand(cache.weights[0].shape, generator=g, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        want = cuda_module.evict(layers[0], cache.weights[0], 128, recent=64, into=twin.prepared(0), into_weights=twin.weights[0])
        assert torch.equal(kept, want)
        for x, y in zip((*to.k_planes[0], *to.v_planes[0], to.seq_lens[0], to.weights[0]), (*twin.k_planes[0], *twin.v_planes[0], twin.seq_lens[0], twin.weights[0])):
            assert torch.equal(x, y), f"replay {r}"


def test_large_rows():
    """A row longer than one pass of a workgroup's threads many times over, weights that share their first digits."""
    from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
    cache, g = make_cache(1, 1, 1, 64, 256, [70001], seed=8, stale=False, track_weights=True)
    cache.weights[0].copy_(1.0 + torch.randint(0, 3000, cache.weights[0].shape, generator=g, device="cuda") * 2.0 ** -23)
    w = cache.weights[0][0, 0, :70001 // 64 * 64].clone()
    kept = cuda_module.evict(cache.prepared(0), cache.weights[0], 6400)[0, 0]
    order = w.sort(dim=0, descending=True, stable=True).indices[:6400].sort().values
    assert torch.equal(kept.long(), order)


def test_sums_into_rows_that_overlap_the_weights_are_refused():
    from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
    pool = torch.zeros(3, 2, 2, 64, device="cuda")
    probs, lens = torch.zeros(2, 4, 64, device="cuda", dtype=torch.half), torch.full((2,), 64, dtype=torch.int32, device="cuda")
    flat = pool.flatten()
    for out in (flat[64:64 + 256].view(2, 2, 64), flat[4:260].view(2, 2, 64), pool[:, 0].permute(1, 0, 2)[:, :2]):
        with pytest.raises(RuntimeError, match="out: "):
            cuda_module.accumulate_weights(pool[0], probs, lens, out=out)
    for out in (pool[0], pool[1], flat[256:512].view(2, 2, 64)):
        assert cuda_module.accumulate_weights(pool[0], probs, lens, out=out) is out
