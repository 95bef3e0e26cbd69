"""The weights that RaggedGQACache.decode accumulates, against the probabilities of each step in 64 bits, and reads at the far end of a long
head.

Bounds of a probability that the step records (u = fp16's half step 2^-11): a score of the planes is fp16(acc * fp16(1 / sqrt(D))) and one
of the rest buffer fp16(fp16(acc) / sqrt(D)), at most three roundings of its size, so |ds| <= d = 3 u max|s| + (D + 8) 2^-24 max sum |q k| scale
+ 2^-24 (below fp16's normal range); a probability then within 2 d + 2^-20 relative (expm1 of it: d is not tiny), rounded to fp16 (u, or 2^-25).
The sum over the heads of a group and the running sum are in 32 bits."""
import math

import pytest
import torch

from tests.serving_forms import U16, U32, cached_tokens, check_rows, rows_form
from tests.test_gpu_tree import make_cache, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("Hq,Hkv,D,kb,lens", [(8, 2, 128, 256, [61, 200, 0, 130]), (4, 4, 64, 64, [126, 5]), (12, 4, 128, 64, [63, 64, 700]), (4, 1, 256, 64, [190, 33]),
                                              (16, 1, 128, 256, [300, 510]), (2, 2, 128, 64, [1100])])
def test_steps_add_their_probabilities(Hq, Hkv, D, kb, lens):
    B, G, steps = len(lens), Hq // Hkv, 6                # (61 + 6, 126 + 6, 63 + 6, 190 + 6 and 510 + 6 cross a flush)
    cache, g = make_cache(B, Hq, Hkv, D, kb, lens, seed=Hq + D, stale=False, track_weights=True)
    cache.reference = True
    cache.weights[0].copy_(torch.rand(cache.weights[0].shape, generator=g, device="cuda"))
    cache.probs.fill_(0.5)                               # a record that a step leaves out would show
    for step in range(steps):
        q, k, v = randn(g, B, 1, Hq, D).half(), randn(g, B, 1, Hkv, D).half(), randn(g, B, 1, Hkv, D).half()
        before = cache.weights[0].clone()
        cache.decode(0, q, k, v)
        for b in range(B):
            n = int(cache.seq_lens[0][b])
            assert n == lens[b] + step + 1
            assert torch.equal(cache.weights[0][b, :, n:], before[b, :, n:])
            for h in range(Hkv):
                ck = cached_tokens(cache, 0, b, h)[0].double()
                want, slack = torch.zeros(n, dtype=torch.float64, device="cuda"), torch.zeros(n, dtype=torch.float64, device="cuda")
                for a in range(h * G, h * G + G):
                    x = q[b, 0, a].double()
                    s = ck @ x * D ** -0.5
                    d = 3 * U16 * s.abs().max().item() + (D + 8) * U32 * (ck.abs() @ x.abs()).max().item() * D ** -0.5 + 2.0 ** -24
                    p = torch.softmax(s, 0)
                    want += p
                    slack += p * (math.expm1(2 * d + 2.0 ** -20) * (1 + U16) + U16) + 2.0 ** -25
                got = cache.weights[0][b, h, :n].double() - before[b, h, :n].double()
                total = before[b, h, :n].double() + want + slack
                assert ((got - want).abs() <= slack + (G + 1) * U32 * total).all(), f"step {step} sequence {b} head {h}: {((got - want).abs() - slack).max().item():.2e} over"


@pytest.mark.parametrize("Hq,Hkv,D,kb", [(8, 2, 128, 256), (4, 4, 128, 64)])
def test_steps_with_fetch_decisions_add_what_they_recorded(Hq, Hkv, D, kb):
    lens, G = [150, 64, 319], Hq // Hkv
    cache, g = make_cache(3, Hq, Hkv, D, kb, lens, seed=2, stale=False, track_weights=True)
    for step in range(4):
        before = cache.weights[0].clone()
        cache.probs.fill_(0.5)
        cache.decode(0, randn(g, 3, 1, Hq, D).half(), randn(g, 3, 1, Hkv, D).half(), randn(g, 3, 1, Hkv, D).half())
        for b in range(3):
            n = lens[b] + step + 1
            got = cache.probs[b, :, :n].double().view(Hkv, G, n).sum(1)
            grown = cache.weights[0][b, :, :n].double() - before[b, :, :n].double()
            assert ((grown - got).abs() <= (G + 1) * U32 * (cache.weights[0][b, :, :n].double() + got)).all()
            # a head's probabilities sum to 1, each within 2^-11 of itself or 2^-25
            assert ((grown.sum(1) - G).abs() <= G * (U16 + 2.0 ** -18 + n * 2.0 ** -25)).all()


def test_the_far_end_of_a_long_head_is_read():
    """A head of 2^21 tokens: only the last 64 in the planes and the rest buffer differ from zero, and carry keys that take the weight."""
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    B, H, D, cap = 2, 4, 256, (1 << 21) + 64
    cache = RaggedGQACache(1, B, cap, H, H, D, k_block=256)
    assert cache.v_planes[0][0].numel() > 1 << 32
    g = torch.Generator(device="cuda").manual_seed(3)
    n, T = (1 << 21) + 5, 3
    q, dk, dv = randn(g, B, T, H, D).half(), randn(g, B, T, H, D).half(), randn(g, B, T, H, D).half()
    far = n // 64 * 64 - 64
    for b in range(B):
        cache.seq_lens[0][b] = n
        k, v = randn(g, 64, H, D) * 0.25, randn(g, 64, H, D)
        k += 4.0 * q[b, :1].float()                     # scores of about 4 sqrt(D) for the first draft
        k, v = k.half(), v.half()
        for h in range(H):
            for planes, x, k_side in ((cache.k_planes[0], k[:, h], True), (cache.v_planes[0], v[:, h], False)):
                w = x.view(torch.int16).to(torch.int32)
                parts = [(w >> 8) & 255, (w >> 4) & 15, w & 15]
                for i, (p, part) in enumerate(zip(planes, parts)):
                    part = (part.T if k_side else part).contiguous()
                    if i:
                        part = part[:, 0::2] << 4 | part[:, 1::2]
                    part = part.to(torch.uint8)
                    if k_side:
                        at = far % 256 // (2 if i else 1)
                        p[b, h, far // 256, :, at:at + part.shape[1]] = part
                    else:
                        p[b, h, far:far + 64] = part
        cache.restk[0][b, :5], cache.restv[0][b, :5] = randn(g, 5, H, D).half(), randn(g, 5, H, D).half()
    anc = torch.tensor([1, 2, 4], device="cuda")
    out = cache.verify(0, q, dk, dv, anc, bound=cap)
    # every token in front has the score 0 and the value 0: as one token of a weight of `far`
    for b in range(B):
        for h in range(H):
            ck, cv = (torch.cat([t[far:], new]) for t, new in zip(cached_tokens(cache, 0, b, h), (dk[b, :, h], dv[b, :, h])))
            assert ck.shape[0] == 64 + 5 + T
            s = q[b, :, h].double() @ ck.double().T * D ** -0.5
            hidden = torch.cat([torch.zeros(T, 69, dtype=torch.bool, device="cuda"), ~torch.eye(T, dtype=torch.bool, device="cuda")], 1)
            s[hidden] = -math.inf
            top = s.max(1, keepdim=True).values.clamp(min=0)
            e = torch.exp(s - top)
            z = e.sum(1, keepdim=True) + far * torch.exp(-top)
            o = e @ cv.double() / z
            _, _, _, tol, _, rel = rows_form(q[b, :, h], ck, cv, ~hidden, D ** -0.5)
            # beside the bounds of the tokens that are told apart: a sum of `far` equal terms in 32 bits, in at most 2^14 rounds
            check_rows(out[b, :, h], o, tol + (2 * rel + 2.0 ** -10) * (e @ cv.double().abs() / z), f"sequence {b} head {h}")
            assert (o[0].abs() > 0.1).any()
