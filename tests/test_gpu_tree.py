"""Attention of drafted tokens over the split-plane cache and the commit of accepted drafts (tests/serving_forms.py has the bounds)."""
import math
import random

import pytest
import torch

from tests.serving_forms import cached_tokens, check_rows, rows_form

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
    return cuda_module


def randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def make_cache(B, Hq, Hkv, D, kb, lens, room=80, seed=0, layers=1, stale=True, **kw):
    """A ragged cache holding lens[b] random tokens; what lies behind them is filled with bytes that read as not-a-number."""
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    g = torch.Generator(device="cuda").manual_seed(seed)
    c = RaggedGQACache(layers, B, max(lens) + room, Hq, Hkv, D, k_block=kb, **kw)
    for i in range(layers):
        if stale:
            for t in (*c.k_planes[i], *c.v_planes[i]):
                t.fill_(255)
            c.restk[i].fill_(math.nan)
            c.restv[i].fill_(math.inf)
        for b, n in enumerate(lens):
            if n == 0:
                continue
            k, v = randn(g, 1, n, Hkv, D), randn(g, 1, n, Hkv, D) * 0.5
            k[..., :4] *= 6.0
            c.prefill(i, b, k.half(), v.half())
    return c, g


def random_tree(T, seed):
    from alignedkv_amd.extension.serving_ops import tree_ancestors
    r = random.Random(seed)
    return tree_ancestors([r.randint(max(-1, t - 5), t - 1) for t in range(T)])


def check_tree(out, cache, q, k, v, anc, softcap=0.0, slopes=None, layer=0):
    B, T, Hq, D = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    for b in range(B):
        masks = [int(m) & ((1 << 64) - 1) for m in (anc[b] if anc.dim() == 2 else anc)]
        n = int(cache.seq_lens[layer][b])
        own = torch.tensor([[bool(m >> u & 1) for u in range(T)] for m in masks], device="cuda")
        pos = torch.tensor([n + bin(m & ~(1 << t)).count("1") for t, m in enumerate(masks)], device="cuda")
        see = torch.cat([torch.ones(T, n, dtype=torch.bool, device="cuda"), own], 1)
        gap = pos[:, None] - torch.cat([torch.arange(n, device="cuda"), pos])[None]
        for h in range(Hkv):
            ck, cv = cached_tokens(cache, layer, b, h)
            ck, cv = torch.cat([ck, k[b, :, h]]), torch.cat([cv, v[b, :, h]])
            for a in range(h * G, h * G + G):
                o, _, _, tol, _, _ = rows_form(q[b, :, a], ck, cv, see, D ** -0.5, softcap, None if slopes is None else slopes[a], gap)
                check_rows(out[b, :, a], o, tol, f"sequence {b} head {a}")


@pytest.mark.parametrize("kb", [64, 256])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("T,Hq,Hkv", [(1, 4, 4), (1, 12, 4), (3, 8, 1), (5, 4, 2), (17, 4, 4), (33, 6, 2), (64, 8, 2)])
def test_trees_over_ragged_caches(ops, kb, D, T, Hq, Hkv):
    lens = [0, 1, 63, 64, 65, 130, 320, 1025]
    cache, g = make_cache(len(lens), Hq, Hkv, D, kb, lens, seed=T)
    B = len(lens)
    q, k, v = (randn(g, B, T, Hq, D) * 1.5).half(), randn(g, B, T, Hkv, D).half(), (randn(g, B, T, Hkv, D) * 0.5).half()
    anc = torch.stack([random_tree(T, 10 * T + b) for b in range(B)]).cuda()
    before = [t.clone() for t in (*cache.k_planes[0], *cache.v_planes[0], cache.restk[0], cache.restv[0], cache.seq_lens[0])]
    out = cache.verify(0, q, k, v, anc)
    check_tree(out, cache, q, k, v, anc)
    for a, b in zip(before, (*cache.k_planes[0], *cache.v_planes[0], cache.restk[0], cache.restv[0], cache.seq_lens[0])):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), "the cache changed"
    assert torch.equal(out, cache.verify(0, q, k, v, anc)), "the same call twice differs"


@pytest.mark.parametrize("softcap,alibi", [(3.0, False), (0.0, True), (30.0, True)])
@pytest.mark.parametrize("T,Hq,Hkv,D,kb", [(1, 4, 4, 128, 64), (9, 4, 2, 64, 256), (40, 4, 1, 128, 256), (6, 2, 2, 256, 64)])
def test_capped_and_biased_scores(ops, softcap, alibi, T, Hq, Hkv, D, kb):
    lens = [700, 90, 5]
    cache, g = make_cache(3, Hq, Hkv, D, kb, lens, seed=T + D)
    q, k, v = (randn(g, 3, T, Hq, D) * 2).half(), randn(g, 3, T, Hkv, D).half(), randn(g, 3, T, Hkv, D).half()
    slopes = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device="cuda", dtype=torch.float32) / Hq) if alibi else None
    anc = random_tree(T, T).cuda()              # one tree for all sequences
    check_tree(cache.verify(0, q, k, v, anc, softcap=softcap, slopes=slopes), cache, q, k, v, anc, softcap, slopes)


def test_a_chain_is_the_default_and_a_bound_does_not_change_bits_beyond_its_cut(ops):
    cache, g = make_cache(2, 8, 2, 128, 256, [300, 515], seed=2)
    T = 6
    q, k, v = randn(g, 2, T, 8, 128).half(), randn(g, 2, T, 2, 128).half(), randn(g, 2, T, 2, 128).half()
    chain = torch.tensor([(1 << (t + 1)) - 1 for t in range(T)], device="cuda")
    out = cache.verify(0, q, k, v)
    assert torch.equal(out, cache.verify(0, q, k, v, chain))
    check_tree(out, cache, q, k, v, chain)
    for bound in (515, 576, cache.max_seq_len):
        check_tree(cache.verify(0, q, k, v, chain, bound=bound), cache, q, k, v, chain)
    given = torch.empty_like(q)
    assert ops.tree_attention(cache.prepared(0), q, k, v, chain, out=given) is given
    parts = (cache.k_planes[0], cache.v_planes[0], cache.k_colmax[0], cache.v_colmax[0], cache.restk[0], cache.restv[0], cache.seq_lens[0])
    assert torch.equal(given, ops.tree_attention(parts, q, k, v, chain))
    # views of a fused projection
    fused = torch.cat([q, k, v], 2)
    assert torch.equal(out, cache.verify(0, fused[:, :, :8], fused[:, :, 8:10], fused[:, :, 10:]))


def test_rows_that_see_nothing_and_values_that_are_not_numbers(ops):
    cache, g = make_cache(3, 4, 2, 128, 64, [0, 0, 70], seed=4)
    T = 5
    q, k, v = randn(g, 3, T, 4, 128).half(), randn(g, 3, T, 2, 128).half(), randn(g, 3, T, 2, 128).half()
    anc = torch.tensor([[0, 2, 0, 8, 24], [1, 3, 5, 9, 25], [1, 2, 4, 8, 16]], device="cuda")
    k[0, 0], v[0, 0] = math.nan, math.inf          # no row of sequence 0 sees draft 0
    v[2, 3, 1, 5] = math.inf                       # draft 3 of sequence 2: its own row, query heads 2 and 3, channel 5
    k[2, 4, 0] = math.nan                          # draft 4 of sequence 2: its own row, query heads 0 and 1
    q[1, 2, 0] = math.nan
    out = cache.verify(0, q, k, v, anc)
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[2, 3, 2:, 5] = True
    want[2, 4, :2] = True
    want[1, 2, 0] = True
    assert torch.equal(bad, want)
    assert (out[0, 0] == 0).all() and (out[0, 2] == 0).all()
    clean = [torch.where(torch.isfinite(t), t, torch.zeros_like(t)) for t in (q, k, v)]
    ref = cache.verify(0, *clean, anc)
    keep = ~want
    keep[2, 4, :2] = False
    keep[1, 2, 0] = False
    assert torch.equal(out[keep], ref[keep])


def test_offsets_beyond_32_bits(ops):
    """A cache whose planes pass 4 GiB: the last sequence's last head lies behind them."""
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    B, H, D, cap = 2, 4, 256, (1 << 22) // 2 + 64
    cache = RaggedGQACache(1, B, cap, H, H, D, k_block=256)
    assert cache.v_planes[0][0].numel() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(1)
    n = 200
    k, v = randn(g, 1, n, H, D).half(), (randn(g, 1, n, H, D) * 0.5).half()
    cache.prefill(0, 1, k, v)
    q, dk, dv = randn(g, B, 3, H, D).half(), randn(g, B, 3, H, D).half(), randn(g, B, 3, H, D).half()
    anc = torch.tensor([1, 3, 5], device="cuda")
    out = cache.verify(0, q, dk, dv, anc)
    small = RaggedGQACache(1, B, 300, H, H, D, k_block=256)
    small.prefill(0, 1, k, v)
    assert torch.equal(out, small.verify(0, q, dk, dv, anc))
    # a sequence that reaches beyond 4 GiB within one head would need 2^24 tokens; the far end of a head of 2^21 is read below
    cache.seq_lens[0][0] = cap // 64 * 64
    far = cache.verify(0, q, dk, dv, anc, bound=cap)
    assert torch.isfinite(far).all()            # zeros in the planes: 2^21 keys with score zero


@pytest.mark.parametrize("Hkv,D,T,kb", [(2, 128, 8, 64), (2, 128, 8, 256), (3, 64, 64, 64), (3, 64, 64, 256), (1, 256, 5, 64)])   # (the decode
def test_commit_equals_decode_steps(ops, Hkv, D, T, kb):               # step has no blocks of 256 tokens for head_dim 256)
    """After a commit the cache holds what as many decode steps leave: planes, column maxima, rest rows, lengths."""
    lens = [0, 1, 60, 63, 64, 100, 127, 250, 319]
    B = len(lens)
    kw = dict(room=70, layers=2, stale=False, seed=T)
    got, g = make_cache(B, Hkv, Hkv, D, kb, lens, **kw)
    want, _ = make_cache(B, Hkv, Hkv, D, kb, lens, **kw)
    k, v = randn(g, 2, B, T, Hkv, D).half(), randn(g, 2, B, T, Hkv, D).half()
    r = random.Random(T)
    paths = [sorted(r.sample(range(T), r.randint(0, T))) for _ in range(B)]
    paths[3] = list(range(T))
    paths[2] = [T - 1, 0, T - 1]                  # any order, a draft twice
    A = max(1, max(len(p) for p in paths))
    accepted = torch.tensor([p + [-1] * (A - len(p)) for p in paths], dtype=torch.int32, device="cuda")
    got.commit(k, v, accepted)
    for layer in range(2):
        one = torch.zeros(B, 1, Hkv, D, dtype=torch.half, device="cuda")
        for b in range(B):
            # one sequence at a time through the decode step, on a cache of its own
            from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
            solo = RaggedGQACache(1, 1, want.max_seq_len, Hkv, Hkv, D, k_block=kb)
            for a, t in zip((*solo.k_planes[0], *solo.v_planes[0], solo.k_colmax[0], solo.v_colmax[0], solo.restk[0], solo.restv[0], solo.seq_lens[0]),
                            (*want.k_planes[layer], *want.v_planes[layer], want.k_colmax[layer], want.v_colmax[layer], want.restk[layer], want.restv[layer], want.seq_lens[layer])):
                a.copy_(t[b:b + 1])
            solo.len_bound[0] = lens[b]
            for t in paths[b]:
                solo.decode(0, one[:1], k[layer, b:b + 1, t:t + 1], v[layer, b:b + 1, t:t + 1])
            n = int(solo.seq_lens[0])
            assert n == lens[b] + len(paths[b]) == int(got.seq_lens[layer][b])
            for a, t in zip((*solo.k_planes[0], *solo.v_planes[0], solo.k_colmax[0], solo.v_colmax[0]),
                            (*got.k_planes[layer], *got.v_planes[layer], got.k_colmax[layer], got.v_colmax[layer])):
                assert torch.equal(a, t[b:b + 1]), f"layer {layer} sequence {b}"
            assert torch.equal(solo.restk[0][:, :n % 64], got.restk[layer][b:b + 1, :n % 64])
            assert torch.equal(solo.restv[0][:, :n % 64], got.restv[layer][b:b + 1, :n % 64])


def test_commit_of_many_layers_capacity_and_rest_rows(ops):
    B, H, D, T, layers = 2, 2, 64, 4, 35          # more layers than one launch takes
    cache, g = make_cache(B, H, H, D, 64, [62, 10], room=4, layers=layers, seed=3)       # capacity 66
    k, v = randn(g, layers, B, T, H, D).half(), randn(g, layers, B, T, H, D).half()
    cache.seq_lens[7][1] = 65                     # one token below the capacity
    rest = [t.clone() for t in cache.restk]
    accepted = torch.tensor([[0, 1, 3, 4], [2, 3, -1, 1]], dtype=torch.int32, device="cuda")      # 4 and -1 end the paths
    cache.commit([t for t in k], [t for t in v], accepted)
    for i in range(layers):
        assert cache.seq_lens[i].tolist() == [65, 66 if i == 7 else 12]
        assert torch.equal(cache.restk[i][0, 0], k[i, 0, 3])                              # 62 + 3: the last one behind the flush
        assert torch.equal(cache.restk[i][0, 1:].view(torch.uint8), rest[i][0, 1:].view(torch.uint8))
        if i == 7:
            assert torch.equal(cache.restk[i][1, 1], k[i, 1, 2])
        else:
            assert torch.equal(cache.restk[i][1, 10:12], k[i, 1, 2:4])
            assert torch.equal(cache.restk[i][1, 12:].view(torch.uint8), rest[i][1, 12:].view(torch.uint8))
        kk, vv = cached_tokens(cache, i, 0, 1)
        assert torch.equal(kk[62:], k[i, 0][[0, 1, 3]][:, 1]) and torch.equal(vv[62:], v[i, 0][[0, 1, 3]][:, 1])


def test_verify_and_commit_in_graphs_on_two_streams(ops):
    """Two caches, a captured verify and commit each, replayed on two streams with eager work between; every replay against the
    eager calls on a twin."""
    T, B, Hq, Hkv, D = 4, 2, 8, 2, 128
    pairs = []
    for s in (1, 2):
        a, g = make_cache(B, Hq, Hkv, D, 256, [200, 310], seed=s, stale=False)
        b, _ = make_cache(B, Hq, Hkv, D, 256, [200, 310], seed=s, stale=False)
        q, k, v = randn(g, B, T, Hq, D).half(), randn(g, B, T, Hkv, D).half(), randn(g, B, T, Hkv, D).half()
        anc, acc = random_tree(T, s).cuda(), torch.tensor([[0, 1, -1], [2, -1, -1]], dtype=torch.int32, device="cuda")
        a.prepared(0)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = a.verify(0, q, k, v, anc, bound=a.max_seq_len)
            ops.tree_commit([a.prepared(0)], [k], [v], acc)
        pairs.append((a, b, q, k, v, anc, acc, graph, out, torch.cuda.Stream(), g))
    for r in range(16):
        for a, b, q, k, v, anc, acc, graph, out, st, g in pairs:
            for t in (q, k, v):
                t.copy_(randn(g, *t.shape).half())
            acc.copy_(torch.tensor([[r % 4, 1, -1], [2, 3, r % 3 - 1]], dtype=torch.int32))
        torch.cuda.synchronize()
        for p in pairs:
            with torch.cuda.stream(p[9]):
                p[7].replay()
        torch.cuda.synchronize()
        for a, b, q, k, v, anc, acc, graph, out, st, g in pairs:
            assert torch.equal(out, b.verify(0, q, k, v, anc, bound=b.max_seq_len)), f"replay {r}"
            b.commit([k], [v], acc)
            assert torch.equal(a.seq_lens[0], b.seq_lens[0])
            for x, y in zip((*a.k_planes[0], *a.v_planes[0], a.k_colmax[0], a.v_colmax[0]), (*b.k_planes[0], *b.v_planes[0], b.k_colmax[0], b.v_colmax[0])):
                assert torch.equal(x, y), f"replay {r}"
