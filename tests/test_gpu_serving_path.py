"""The serving operators run together, as a server would: packed prompts, drafted and plain steps, commits, eviction; and the decoder's
paths that call them."""
import pytest
import torch

from tests.serving_forms import cached_tokens, check_rows, rows_form

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,D,kb", [(8, 2, 128, 256), (4, 4, 64, 64)])
def test_packed_prompts_drafts_commits_and_eviction(Hq, Hkv, D, kb):
    from alignedkv_amd.extension.serving_ops import tree_ancestors
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    g = torch.Generator(device="cuda").manual_seed(D)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").half()  # noqa: E731
    lens, B, layers, G = [150, 64, 301], 3, 2, Hq // Hkv
    cache = RaggedGQACache(layers, B, 600, Hq, Hkv, D, k_block=kb, track_weights=True)
    held = []                                                     # what every layer and sequence should hold
    for layer in range(layers):
        q, k, v = rn(1, sum(lens), Hq, D), rn(1, sum(lens), Hkv, D), rn(1, sum(lens), Hkv, D)
        out = cache.prefill_packed(layer, q, k, v, lens, window=48)
        start = 0
        mine = []
        for b, n in enumerate(lens):
            at = slice(start, start + n)
            see = torch.tril(torch.ones(n, n, dtype=torch.bool, device="cuda"))
            total = torch.zeros(Hkv, n, dtype=torch.float64, device="cuda")
            for h in range(Hq):
                o, _, p, tol, _, _ = rows_form(q[0, at, h], k[0, at, h // G], v[0, at, h // G], see, D ** -0.5)
                check_rows(out[0, at, h], o, tol, f"prompt {b} head {h}")
                total[h // G] += p[max(0, n - 48):].sum(0)
            assert (cache.weights[layer][b, :, :n].double() - total).abs().max() <= 1e-4 and (cache.weights[layer][b, :, n:] == 0).all()
            mine.append((k[0, at], v[0, at]))
            start += n
        held.append(mine)
    tree = torch.stack([tree_ancestors([-1, 0, 0, 1, -1]), tree_ancestors([-1, 0, 1, 2, 3]), tree_ancestors([-1, -1, 1, 1, 0])]).cuda()
    paths = [[0, 1, 3], [0, 1, 2, 3, 4], [1]]
    accepted = torch.tensor([p + [-1] * (5 - len(p)) for p in paths], dtype=torch.int32, device="cuda")
    for _ in range(3):
        drafts = []
        for layer in range(layers):
            q, k, v = rn(B, 5, Hq, D), rn(B, 5, Hkv, D), rn(B, 5, Hkv, D)
            out = cache.verify(layer, q, k, v, tree)
            drafts.append((k, v))
            for b in range(B):
                own = torch.tensor([[bool(int(m) >> u & 1) for u in range(5)] for m in tree[b]], device="cuda")
                for h in range(Hq):
                    ck, cv = (torch.cat([held[layer][b][s][:, h // G], (k, v)[s][b, :, h // G]]) for s in (0, 1))
                    see = torch.cat([torch.ones(5, ck.shape[0] - 5, dtype=torch.bool, device="cuda"), own], 1)
                    o, _, _, tol, _, _ = rows_form(q[b, :, h], ck, cv, see, D ** -0.5)
                    check_rows(out[b, :, h], o, tol, f"drafts of sequence {b} head {h}")
        cache.commit([d[0] for d in drafts], [d[1] for d in drafts], accepted, most=5)
        for layer in range(layers):
            for b in range(B):
                held[layer][b] = tuple(torch.cat([held[layer][b][s], drafts[layer][s][b][paths[b]]]) for s in (0, 1))
        # and a plain step of every sequence
        for layer in range(layers):
            q, k, v = rn(B, 1, Hq, D), rn(B, 1, Hkv, D), rn(B, 1, Hkv, D)
            cache.decode(layer, q, k, v)
            held[layer] = [tuple(torch.cat([held[layer][b][s], (k, v)[s][b]]) for s in (0, 1)) for b in range(B)]
    for layer in range(layers):
        assert cache.seq_lens[layer].tolist() == [held[layer][b][0].shape[0] for b in range(B)]
        for b in range(B):
            for h in range(Hkv):
                ck, cv = cached_tokens(cache, layer, b, h)
                assert torch.equal(ck, held[layer][b][0][:, h]) and torch.equal(cv, held[layer][b][1][:, h])
    cache.refresh_bounds()
    assert cache.len_bound[0] == max(cache.seq_lens[0].tolist())
    kept = cache.evict(0, 128, sinks=4, recent=40)
    for b in range(B):
        n = held[0][b][0].shape[0]
        f = n // 64 * 64
        for h in range(Hkv):
            at = torch.cat([kept[b, h][kept[b, h] >= 0].long(), torch.arange(f, n, device="cuda")])
            ck, cv = cached_tokens(cache, 0, b, h)
            assert torch.equal(ck, held[0][b][0][at, h]) and torch.equal(cv, held[0][b][1][at, h])
    q, k, v = rn(B, 2, Hq, D), rn(B, 2, Hkv, D), rn(B, 2, Hkv, D)
    assert torch.isfinite(cache.verify(0, q, k, v)).all()
    with pytest.raises(RuntimeError, match="positions"):
        cache.verify(0, q, k, v, slopes=torch.ones(Hq, device="cuda"))
    cache.prefill(0, 1, rn(1, 70, Hkv, D), rn(1, 70, Hkv, D))              # a sequence starts anew: its weights too
    assert int(cache.seq_lens[0][1]) == 70 and (cache.weights[0][1] == 0).all()


def small(**kw):
    from alignedkv_amd.model.decoder_harness import DecoderConfig
    return DecoderConfig(num_hidden_layers=2, hidden_size=512, num_attention_heads=4, num_key_value_heads=2, intermediate_size=512, vocab_size=500,
                         max_position_embeddings=512, **kw)


@pytest.mark.parametrize("kw", [dict(attn_softcap=5.0), dict(alibi=True), dict(attn_softcap=20.0, alibi=True)])
def test_decoder_with_capped_and_biased_scores_tracks_dense_torch(kw):
    from alignedkv_amd.model.decoder_harness import RandomLlamaDecoder, make_cache
    cfg = small(**kw)
    model = RandomLlamaDecoder(cfg, seed=1)
    prompt = torch.randint(0, cfg.vocab_size, (2, 90), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
    ref_tokens, ref_logits = model.generate(prompt, 50, make_cache("dense_torch", cfg, 2, 256))
    cache = make_cache("alignedkv_device_lengths", cfg, 2, 256)
    _, logits = model.generate(prompt, 50, cache, forced_tokens=ref_tokens)
    assert cache.inner.seq_lens[0].tolist() == [139, 139]
    # two layers of fp16 activations: the bound of the other decoder tests with every plane read
    assert (logits - ref_logits).abs().max().item() <= 2e-2 * max(1.0, ref_logits.abs().max().item())
    graphed = make_cache("alignedkv_graph", cfg, 2, 256)
    _, again = model.generate_graphed(prompt, 50, graphed, forced_tokens=ref_tokens)
    assert torch.equal(again, logits)


@pytest.mark.parametrize("kw", [dict(), dict(attn_softcap=10.0), dict(alibi=True)])
def test_drafted_decoding_accepts_only_what_the_model_chooses(kw):
    """Drafts that are right, wrong and branching: every token that comes out is the arg-max of logits that dense attention over the same
    tokens confirms."""
    from alignedkv_amd.model.decoder_harness import RandomLlamaDecoder, make_cache
    cfg = small(**kw)
    model = RandomLlamaDecoder(cfg, seed=3)
    B, n, steps = 3, 61, 40
    prompt = torch.randint(0, cfg.vocab_size, (B, n), device="cuda", generator=torch.Generator(device="cuda").manual_seed(4))
    truth, _ = model.generate(prompt, steps + 10, make_cache("dense_torch", cfg, B, 256))

    def propose(history, draft_len):
        drafts, parents = [], []
        for b, h in enumerate(history):
            done = len(h) - n
            right = truth[b, done:done + 3].tolist()
            # a branch that goes wrong beside the one that (mostly) is right
            drafts.append([(right[0] + 1) % cfg.vocab_size] + right + [7])
            parents.append([-1, -1, 1, 2, 0])
        return drafts, parents

    stats = {}
    cache = make_cache("alignedkv_drafted", cfg, B, 256)
    out = model.generate_drafted(prompt, steps, cache, propose=propose, stats=stats)
    assert out.shape == (B, steps) and stats["accepted"] > 0 and stats["passes"] < steps
    _, logits = model.generate(prompt, steps, make_cache("dense_torch", cfg, B, 256), forced_tokens=out)
    best = logits.max(-1).values.T                                        # [B, steps]
    chosen = torch.gather(logits.permute(1, 0, 2), 2, out[:, :, None])[..., 0]
    scale = max(1.0, logits.abs().max().item())
    assert (best - chosen).max().item() <= 4e-2 * scale, "a token was accepted that dense attention would not have chosen"
    n_tok = cache.inner.seq_lens[0].clone()
    assert int(n_tok.min()) >= n + steps - 1 and int(n_tok.max()) <= n + steps + 4
    with pytest.raises(RuntimeError, match="device_positions"):
        cache.get_seq_length()
    step = model.forward(out[:, -1:], cache, positions=cache.device_positions())    # plain steps go on from lengths that differ
    assert torch.isfinite(step).all() and (cache.inner.seq_lens[0] == n_tok + 1).all()
    chain = model.generate_drafted(prompt, 12, make_cache("alignedkv_drafted", cfg, B, 256), draft_len=3)
    assert chain.shape == (B, 12)


def test_decoder_goes_on_under_eviction():
    from alignedkv_amd.model.decoder_harness import RandomLlamaDecoder, make_cache
    cfg = small()
    model = RandomLlamaDecoder(cfg, seed=5)
    prompt = torch.randint(0, cfg.vocab_size, (2, 200), device="cuda", generator=torch.Generator(device="cuda").manual_seed(6))
    cache = make_cache("alignedkv_evict", cfg, 2, 320)
    tokens, logits = model.generate(prompt, 100, cache, keep=128)
    assert cache.get_seq_length() == 299 and cache._dropped > 0
    assert cache.inner.seq_lens[0].tolist() == [299 - cache._dropped] * 2 and 299 - cache._dropped < 128 + 64
    assert torch.isfinite(logits).all() and tokens.shape == (2, 100)
    assert cache.device_positions().tolist() == [299]
