"""Prompt attention and the weights tokens receive against the definitions in 64 bits (tests/serving_forms.py has the bounds)."""
import math

import pytest
import torch

from tests.serving_forms import U32, check_rows, prompt_see, rows_form

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
    return cuda_module


def inputs(B, S, Hq, Hkv, D, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    q, k, v = (torch.randn(B, S, H, D, generator=g, device="cuda") for H in (Hq, Hkv, Hkv))
    k[..., :4] *= 6.0
    return (q * spread).half(), k.half(), (v * 0.5).half()


def slopes_of(Hq):
    return torch.exp2(-8.0 * torch.arange(1, Hq + 1, device="cuda", dtype=torch.float32) / Hq)


def check_against_form(out, lse, q, k, v, softcap=0.0, slopes=None, lens=None, prefix=None, docs=None, scale=None, heads=None):
    B, S, Hq, D = q.shape
    G = Hq // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    at = torch.arange(S, device="cuda")
    gap = at[:, None] - at[None]
    for b in range(B):
        n = S if lens is None else max(0, min(S, int(lens[b])))
        see = prompt_see(n, S, "cuda", None if prefix is None else int(prefix[b]), None if docs is None else docs[b])
        for h in (range(Hq) if heads is None else heads):
            o, want_lse, _, tol, tol_lse, _ = rows_form(q[b, :, h], k[b, :, h // G], v[b, :, h // G], see, scale, softcap, None if slopes is None else slopes[h], gap)
            check_rows(out[b, :, h], o, tol, f"sequence {b} head {h}")
            got = lse[b, h].double()
            empty = torch.isinf(want_lse)
            assert torch.equal(torch.isinf(got), empty) and (got[empty] < 0).all()
            assert ((got - want_lse).abs()[~empty] <= tol_lse[~empty]).all(), f"lse of sequence {b} head {h}"


@pytest.mark.parametrize("S", [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 200, 257])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_causal_lengths(ops, S, D):
    q, k, v = inputs(2, S, 4, 2, D, seed=S)
    out, lse = ops.prefill_attention(q, k, v, return_lse=True)
    check_against_form(out, lse, q, k, v)
    assert torch.equal(out, ops.prefill_attention(q, k, v)), "the same call twice differs"


@pytest.mark.parametrize("softcap", [0.0, 2.0, 30.0])
@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("mask", ["causal", "lens", "prefix", "docs", "docs_prefix_lens"])
@pytest.mark.parametrize("B,S,Hq,Hkv,D", [(3, 150, 4, 4, 64), (2, 321, 6, 2, 128), (2, 130, 8, 1, 256)])
def test_score_forms_and_masks(ops, softcap, alibi, mask, B, S, Hq, Hkv, D):
    q, k, v = inputs(B, S, Hq, Hkv, D, seed=S + int(softcap), spread=2.0)
    i32 = dict(dtype=torch.int32, device="cuda")
    lens = prefix = docs = None
    if "lens" in mask:
        lens = torch.tensor([S, S // 2 + 3, 1][:B], **i32)
    if "prefix" in mask:
        prefix = torch.tensor([70, 0, S][:B], **i32)
    if "docs" in mask:
        g = torch.Generator().manual_seed(S)
        docs = torch.sort(torch.randint(0, 5, (B, S), generator=g), 1).values.to(torch.int32)
        docs[0] = torch.randint(0, 3, (S,), generator=g)            # not in runs
        docs[1, 20:90] = -1                                         # rows that see nothing
        docs = docs.cuda()
    slopes = slopes_of(Hq) if alibi else None
    kw = dict(softcap=softcap, slopes=slopes, seq_lens=lens, prefix_lens=prefix, documents=docs)
    out, lse = ops.prefill_attention(q, k, v, return_lse=True, **kw)
    check_against_form(out, lse, q, k, v, softcap, slopes, lens, prefix, docs)
    if docs is not None:
        assert (out[1, 20:90] == 0).all() and (lse[1, :, 20:90] == -math.inf).all()
    w = ops.attention_weights(q, k, lse, window=0, **kw)
    check_weights(w, q, k, lse, 0, softcap, slopes, lens, prefix, docs)


def check_weights(w, q, k, lse, window, softcap=0.0, slopes=None, lens=None, prefix=None, docs=None, start=None):
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]
    G = Hq // Hkv
    at = torch.arange(S, device="cuda")
    gap = at[:, None] - at[None]
    for b in range(B):
        n = S if lens is None else int(lens[b])
        see = prompt_see(n, S, "cuda", None if prefix is None else int(prefix[b]), None if docs is None else docs[b])
        if window:
            see = see & (at >= n - window)[:, None]
        for h in range(Hkv):
            want, rel, rows = torch.zeros(S, dtype=torch.float64, device="cuda"), 0.0, 0
            for a in range(h * G, h * G + G):
                _, own, p, _, _, r = rows_form(q[b, :, a], k[b, :, h], None, see, D ** -0.5, softcap, None if slopes is None else slopes[a], gap)
                ok = torch.isfinite(own)
                # exp(s - lse) with the lse that was handed in
                want += (p[ok] * torch.exp(own[ok] - lse[b, a, ok].double())[:, None]).sum(0)
                rel, rows = max(rel, r), rows + int(ok.sum())
            if start is not None:
                want = want + start[b, h].double()
            # every term within 2 rel (its score and the difference to lse), a sum of `rows` terms in 32 bits
            assert ((w[b, h].double() - want).abs() <= want * (2 * rel + rows * U32) + 1e-30).all(), f"weights of sequence {b} head {h}"


@pytest.mark.parametrize("B,S,Hq,Hkv,D,window", [(1, 1, 2, 1, 64, 0), (2, 33, 4, 4, 128, 5), (2, 300, 8, 2, 128, 64), (1, 190, 2, 2, 256, 500), (3, 97, 6, 2, 64, 1)])
def test_weights_of_a_window(ops, B, S, Hq, Hkv, D, window):
    q, k, v = inputs(B, S, Hq, Hkv, D, seed=window + S)
    lens = torch.tensor([S, max(1, S // 3), S - 1 if S > 1 else 1][:B], dtype=torch.int32, device="cuda")
    _, lse = ops.prefill_attention(q, k, v, seq_lens=lens, return_lse=True)
    w = ops.attention_weights(q, k, lse, seq_lens=lens, window=window)
    check_weights(w, q, k, lse, window, lens=lens)
    # added to a wider accumulator: entries beyond the length stay
    acc = torch.rand(B, Hkv, S + 9, device="cuda")
    before = acc.clone()
    assert ops.attention_weights(q, k, lse, seq_lens=lens, window=window, out=acc) is acc
    for b in range(B):
        n = int(lens[b])
        assert torch.equal(acc[b, :, n:], before[b, :, n:])
        # one more rounding of the sum
        assert ((acc[b, :, :n] - (before[b, :, :n] + w[b, :, :n])).abs() <= 2 * U32 * acc[b, :, :n]).all()


def test_values_that_are_not_numbers_reach_the_rows_that_see_them_and_no_others(ops):
    B, S, H, D = 2, 200, 2, 128
    q, k, v = inputs(B, S, H, H, D, seed=5)
    lens = torch.tensor([S, 77], dtype=torch.int32, device="cuda")
    docs = torch.zeros(B, S, dtype=torch.int32, device="cuda")
    docs[0, 100:] = 1
    docs[0, 50] = -1
    v[0, 50], k[0, 50] = math.inf, math.nan        # in no document
    v[0, 90, 1, 7] = math.inf                      # seen by rows 90 .. 99 of document 0, not by document 1
    v[0, 130, 0, 3] = math.nan                     # seen by rows 130 ..
    k[0, 180, 1] = math.nan                        # rows 180 .. of head 1 are undefined
    v[1, 77:], k[1, 77:], q[1, 77:] = math.nan, math.inf, math.nan     # padding
    out, lse = ops.prefill_attention(q, k, v, seq_lens=lens, documents=docs, return_lse=True)
    bad = ~torch.isfinite(out)
    want = torch.zeros_like(bad)
    want[0, 90:100, 1, 7] = True
    want[0, 130:, 0, 3] = True
    want[0, 180:, 1] = True
    assert torch.equal(bad, want)
    assert (out[1, 77:] == 0).all() and (lse[1, :, 77:] == -math.inf).all() and (out[0, 50] == 0).all()
    clean = v.clone()
    clean[~torch.isfinite(clean)] = 0
    kc = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
    ref = ops.prefill_attention(torch.where(torch.isfinite(q), q, torch.zeros_like(q)), kc, clean, seq_lens=lens, documents=docs)
    keep = ~want
    keep[0, 90:, 1] &= False        # (rows that saw the undefined key or value in some channel are compared below)
    assert torch.equal(out[keep], ref[keep])


def test_views_are_read_in_place_and_odd_ones_copied(ops):
    B, S, Hq, Hkv, D = 2, 140, 4, 2, 128
    g = torch.Generator(device="cuda").manual_seed(3)
    fused = torch.randn(B, S, (Hq + 2 * Hkv), D, generator=g, device="cuda").half()
    q, k, v = fused[:, :, :Hq], fused[:, :, Hq:Hq + Hkv], fused[:, :, Hq + Hkv:]
    want = ops.prefill_attention(q.contiguous(), k.contiguous(), v.contiguous())
    assert torch.equal(ops.prefill_attention(q, k, v), want)
    heads_first = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    assert torch.equal(ops.prefill_attention(*heads_first), want)
    odd = torch.empty(q.numel() + 1, dtype=torch.half, device="cuda")[1:].view(B, S, Hq, D)      # two bytes off a 16-byte boundary
    odd.copy_(q)
    last = torch.empty(B, S, Hkv, 2 * D, dtype=torch.half, device="cuda")[..., ::2]                # a strided last dimension
    last.copy_(k)
    assert torch.equal(ops.prefill_attention(odd, last, v.expand(B, S, Hkv, D)), want)
    one = k[:1].expand(B, S, Hkv, D)                                                                 # one prompt's keys for all: stride 0
    assert torch.equal(ops.prefill_attention(q, one, v), ops.prefill_attention(q, one.contiguous(), v))
    assert torch.equal(ops.attention_weights(q, k, torch.zeros(B, Hq, S, device="cuda")), ops.attention_weights(q.contiguous(), k.contiguous(), torch.zeros(B, Hq, S, device="cuda")))


def test_rows_behind_the_length_of_a_given_output_stay(ops):
    q, k, v = inputs(3, 100, 2, 2, 64, seed=1)
    lens = torch.tensor([100, 0, 37], dtype=torch.int32, device="cuda")
    out = torch.full((3, 100, 2, 64), 7.0, dtype=torch.half, device="cuda")
    got, lse = ops.prefill_attention(q, k, v, seq_lens=lens, out=out, return_lse=True)
    assert got is out and (out[1] == 7).all() and (out[2, 37:] == 7).all()
    full, full_lse = ops.prefill_attention(q, k, v, seq_lens=lens, return_lse=True)
    assert torch.equal(out[0], full[0]) and torch.equal(out[2, :37], full[2, :37]) and torch.equal(lse, full_lse)
    assert (full[1] == 0).all() and (full_lse[1] == -math.inf).all()


def test_offsets_beyond_32_bits(ops):
    S, D = 300, 128
    step = (1 << 24) - 8                        # the widest token stride: row 299 is 10 GB behind row 0
    big = torch.zeros(step * S, dtype=torch.half, device="cuda")
    view = big.view(1, S, 1, step)[..., :D]
    q, k, v = inputs(1, S, 1, 1, D, seed=9)
    want = ops.prefill_attention(q, k, v)
    view.copy_(k)
    assert torch.equal(ops.prefill_attention(q, view, v), want)
    view.copy_(v)
    assert torch.equal(ops.prefill_attention(q, k, view), want)
    view.copy_(q)
    assert torch.equal(ops.prefill_attention(view, k, v), want)


def test_another_stream_and_two_graphs_in_flight(ops):
    """Calls on two streams at once, and two captured graphs replayed on two streams between eager work: every replay against the
    eager result for the inputs it had."""
    B, S, Hq, Hkv, D = 2, 500, 8, 2, 128
    docs = torch.arange(S, device="cuda", dtype=torch.int32).div(130, rounding_mode="floor").to(torch.int32).expand(B, S).contiguous()
    sets = [inputs(B, S, Hq, Hkv, D, seed=s) for s in (1, 2)]
    call = lambda x: ops.prefill_attention(*x, documents=docs, softcap=20.0, return_lse=True)  # noqa: E731
    want = [call(x) for x in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for st, x in zip(streams, sets):
        with torch.cuda.stream(st):
            got.append(call(x))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert torch.equal(g[0], w[0]) and torch.equal(g[1], w[1])
    held, graphs, outs = [[t.clone() for t in x] for x in sets], [], []
    for x in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            o, lse = call(x)
            w = ops.attention_weights(x[0], x[1], lse, documents=docs, softcap=20.0, window=40)
        graphs.append(g)
        outs.append((o, lse, w))
    for r in range(4):
        fresh = [inputs(B, S, Hq, Hkv, D, seed=10 * r + s) for s in (1, 2)]
        for x, f in zip(held, fresh):
            for t, n in zip(x, f):
                t.copy_(n)
        torch.cuda.synchronize()
        for st, g in zip(streams, graphs):
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for f, o in zip(fresh, outs):
            eo, el = call(f)
            ew = ops.attention_weights(f[0], f[1], el, documents=docs, softcap=20.0, window=40)
            assert torch.equal(o[0], eo) and torch.equal(o[1], el) and torch.equal(o[2], ew), f"replay {r}"


@pytest.mark.parametrize("B,Hq,Hkv,cap,width", [(1, 1, 1, 1, 8), (3, 8, 2, 100, 128), (2, 6, 6, 2050, 2112), (2, 8, 1, 4097, 4160)])
@pytest.mark.parametrize("decay", [1.0, 0.5])
def test_accumulate_weights(ops, B, Hq, Hkv, cap, width, decay):
    g = torch.Generator(device="cuda").manual_seed(cap)
    probs = torch.rand(B, Hq, width, generator=g, device="cuda").half()
    store = torch.rand(B, Hkv, cap + 3, generator=g, device="cuda")
    w = store[:, :, 1:cap + 1]                  # rows apart, not 16-byte aligned
    lens = torch.tensor([cap, max(0, cap - 5), cap // 2][:B], dtype=torch.int32, device="cuda")
    before, around = w.clone(), store.clone()
    other = torch.full((B, Hkv, cap), 5.0, device="cuda")
    got = ops.accumulate_weights(w, probs, lens, decay=decay, out=other)
    assert got is other and torch.equal(w, before)
    assert ops.accumulate_weights(w, probs, lens, decay=decay) is w
    assert torch.equal(store[:, :, 0], around[:, :, 0]) and torch.equal(store[:, :, cap + 1:], around[:, :, cap + 1:])
    for b in range(B):
        n = int(lens[b])
        want = before[b, :, :n].double() * decay + probs[b, :, :n].double().view(Hkv, Hq // Hkv, n).sum(1)
        assert ((w[b, :, :n].double() - want).abs() <= (Hq // Hkv + 1) * U32 * want).all()
        assert torch.equal(other[b, :, :n], w[b, :, :n])
        assert torch.equal(w[b, :, n:], before[b, :, n:]) and (other[b, :, n:] == 5).all()


@pytest.mark.parametrize("parts", ["1", "2"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_whole_rows_and_rows_in_two_parts(ops, monkeypatch, parts, D):
    """Both forms of the kernel on the same calls: a workgroup's rows as one run over the tokens, or split over two halves of its waves."""
    from alignedkv_amd import load_library
    lib = load_library()
    monkeypatch.setenv("AKV_TUNE_PROMPT_PARTS", parts)
    lib.akv_reload_tuning()
    try:
        i32 = dict(dtype=torch.int32, device="cuda")
        for S in (1, 33, 64, 65, 130, 300, 389):
            q, k, v = inputs(2, S, 4, 2, D, seed=S)
            lens, prefix = torch.tensor([S, S // 2], **i32), torch.tensor([S // 3, 100], **i32)
            docs = torch.sort(torch.randint(-1, 4, (2, S)), 1).values.to(torch.int32).cuda()
            for kw in (dict(), dict(seq_lens=lens, prefix_lens=prefix, softcap=5.0), dict(documents=docs, seq_lens=lens, slopes=slopes_of(4))):
                out, lse = ops.prefill_attention(q, k, v, return_lse=True, **kw)
                check_against_form(out, lse, q, k, v, kw.get("softcap", 0.0), kw.get("slopes"), kw.get("seq_lens"), kw.get("prefix_lens"), kw.get("documents"))
        test_values_that_are_not_numbers_reach_the_rows_that_see_them_and_no_others(ops)
    finally:
        monkeypatch.delenv("AKV_TUNE_PROMPT_PARTS")
        lib.akv_reload_tuning()
