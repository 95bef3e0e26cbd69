"""The serving operators over the split-plane cache: prompt attention with capped, biased and masked scores, the attention weight
each cached token has received, attention of a tree of drafted tokens over the cache, the commit of accepted drafts, and
eviction by accumulated weight.  `own` False: each operator in elementary torch operations; True: the framework's calls."""
import math
import random

import torch

own = False

BLOCK = 64        # tokens of the rest buffer, the unit in which tokens enter the planes


def listed():
    return [
        # one short prompt of a multi-head model whose scores are capped: what the first token waits for (latency)
        dict(name="prefill_short", op="prefill", B=1, S=128, Hq=32, Hkv=32, D=128, softcap=30.0, alibi=False, prefix=0.0, docs=0, ragged=0.0),
        # a padded batch with a bidirectional prefix and a distance bias, odd length
        dict(name="prefill_padded", op="prefill", B=6, S=2021, Hq=16, Hkv=16, D=64, softcap=0.0, alibi=True, prefix=0.25, docs=0, ragged=0.7),
        # several prompts packed into one row, grouped-query heads, capped scores: the largest prompt call
        dict(name="prefill_packed", op="prefill", B=1, S=8192, Hq=32, Hkv=8, D=128, softcap=50.0, alibi=False, prefix=0.0, docs=3, ragged=0.0),
        # which prompt tokens the last rows of a long prompt look at, before an eviction
        dict(name="weights_prompt", op="observe", B=2, S=8000, Hq=32, Hkv=8, D=128, softcap=0.0, alibi=False, window=64, ragged=0.3),
        # the same bookkeeping after one decode step
        dict(name="weights_decode", op="accumulate", B=8, L=8100, Hq=32, Hkv=8, ragged=0.5, decay=1.0),
        # a single drafted token (the plain step of a model with capped scores) at batch 1
        dict(name="tree_single", op="tree", B=1, T=1, L=1024, Hq=32, Hkv=32, D=128, k_block=64, softcap=30.0, alibi=False, ragged=0.0),
        # sixteen drafts over a ragged batch with grouped-query heads
        dict(name="tree_ragged", op="tree", B=8, T=16, L=8150, Hq=32, Hkv=8, D=128, k_block=256, softcap=0.0, alibi=False, ragged=0.5),
        # the widest tree over a long cache
        dict(name="tree_wide", op="tree", B=4, T=64, L=32768, Hq=32, Hkv=8, D=128, k_block=256, softcap=0.0, alibi=True, ragged=0.0),
        # accepted drafts of one layer and one sequence, and of many layers of a ragged batch
        dict(name="commit_one", op="commit", layers=1, B=1, T=5, L=1000, H=32, D=128, k_block=64, ragged=0.0),
        dict(name="commit_layers", op="commit", layers=24, B=8, T=16, L=700, H=8, D=128, k_block=256, ragged=0.6),
        # a prompt squeezed into a small serving cache, and a long ragged batch cut to an eighth
        dict(name="evict_short", op="evict", B=1, L=1024, H=32, D=128, k_block=64, keep=256, sinks=4, recent=64, ragged=0.0),
        dict(name="evict_long", op="evict", B=8, L=32000, H=8, D=128, k_block=256, keep=4096, sinks=4, recent=512, ragged=0.4),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["prefill", "prefill", "observe", "accumulate", "tree", "tree", "commit", "evict"])
    D = rng.choice([64, 128, 128, 128, 256])
    Hq, Hkv = rng.choice([(32, 32), (32, 8), (32, 8), (16, 16), (16, 2), (12, 4), (8, 1), (40, 8)])
    B = _log(rng, 1, 8)
    ragged = rng.choice([0.0, round(rng.uniform(0.1, 0.95), 3)])
    cap, alibi = rng.choice([0.0, 30.0, 50.0]), rng.random() < 0.3
    if op == "prefill":
        S = _log(rng, 16, 8192)
        if S * S * Hq * D > 8192 * 8192 * 16 * 64:
            D = 64
            Hq, Hkv = rng.choice([(16, 16), (12, 4), (16, 2)])
        B = max(1, min(B, 8192 * 8192 * 16 * 64 // (S * S * Hq * D)))
        kind = rng.choice(["plain", "prefix", "docs", "docs"])
        return dict(op=op, B=B, S=S, Hq=Hq, Hkv=Hkv, D=D, softcap=cap, alibi=alibi, prefix=round(rng.uniform(0.05, 0.6), 3) if kind == "prefix" else 0.0,
                    docs=rng.randint(2, 12) if kind == "docs" else 0, ragged=ragged)
    if op == "observe":
        return dict(op=op, B=max(1, B // 2), S=_log(rng, 64, 8192), Hq=Hq, Hkv=Hkv, D=D, softcap=cap, alibi=alibi, window=rng.randint(8, 128), ragged=ragged)
    if op == "accumulate":
        return dict(op=op, B=B, L=_log(rng, 100, 32768), Hq=Hq, Hkv=Hkv, ragged=ragged, decay=rng.choice([1.0, 0.875]))
    kb = rng.choice([64, 256])
    if op == "tree":
        L, T = min(_log(rng, 32, 32768), 4 * 32768 * 8 * 128 // (Hkv * D)), _log(rng, 1, 64)
        B = max(1, min(B, 4 * 32768 * 8 * 128 // (L * Hkv * D), 4 * 32768 * 64 * 32 * 128 // (L * T * Hq * D)))
        return dict(op=op, B=B, T=T, L=L, Hq=Hq, Hkv=Hkv, D=D, k_block=kb, softcap=cap, alibi=alibi, ragged=ragged)
    if op == "commit":
        return dict(op=op, layers=rng.randint(1, 24), B=B, T=_log(rng, 1, 64), L=_log(rng, 40, 700), H=min(Hkv, 8), D=D, k_block=kb, ragged=ragged)
    L = _log(rng, 300, 32000)
    B = max(1, min(B, 8 * 32000 * 8 * 128 // (L * Hkv * D)))
    keep = BLOCK * rng.randint(1, max(1, L // 128))
    return dict(op=op, B=B, L=L, H=Hkv, D=D, k_block=kb, keep=keep, sinks=rng.choice([0, 4]), recent=min(keep - 4, rng.choice([0, 64, 200])), ragged=ragged)


# ---- sizes that a case stands for ---------------------------------------------------------------------------------------------

def _lens(case, full):
    """Lengths of the sequences, the longest `full`, spread down to (1 - ragged) of it."""
    B, r = case["B"], case["ragged"]
    return [max(1, int(full * (1 - r * b / max(1, B - 1)))) for b in range(B)]


def _doc_sizes(case):
    """Sizes of the packed documents: in the proportions 1 : 2 : 3 ..."""
    n, S = min(case["docs"], case["S"]), case["S"]
    cuts = [S * k * (k + 1) // (n * (n + 1)) for k in range(n + 1)]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _pairs(case):
    """Visible (row, token) pairs of a prompt batch."""
    if case.get("docs"):
        return case["B"] * sum(n * (n + 1) // 2 for n in _doc_sizes(case))
    total = 0
    for n in _lens(case, case["S"]):
        p = int(case.get("prefix", 0.0) * n)
        total += n * (n + 1) // 2 + p * (p - 1) // 2
    return total


def work(case):
    op, D = case["op"], case.get("D", 0)
    if op == "prefill":
        rows = case["B"] * case["S"] if case["docs"] else sum(_lens(case, case["S"]))
        return dict(bytes=rows * (2 * case["Hq"] + 2 * case["Hkv"]) * D * 2 + rows * case["Hq"] * 4, flops=4 * D * case["Hq"] * _pairs(case))
    if op == "observe":
        rows = sum(_lens(case, case["S"]))
        w = [(n, min(n, case["window"])) for n in _lens(case, case["S"])]
        seen = sum(k * n - k * (k - 1) // 2 for n, k in w)
        return dict(bytes=rows * case["Hkv"] * (D * 2 + 4) + sum(k for _, k in w) * case["Hq"] * (D * 2 + 4), flops=2 * D * case["Hq"] * seen)
    if op == "accumulate":
        n = sum(_lens(case, case["L"]))
        return dict(bytes=n * (case["Hq"] * 2 + case["Hkv"] * 8), flops=n * case["Hq"])
    if op == "tree":
        n, T = sum(_lens(case, case["L"])), case["T"]
        drafts = case["B"] * T * D * 2
        return dict(bytes=n * case["Hkv"] * D * 4 + drafts * (2 * case["Hkv"] + 2 * case["Hq"]), flops=4 * D * case["Hq"] * T * n)
    if op == "commit":
        rows = case["layers"] * case["B"] * case["H"] * D * 4
        return dict(bytes=rows * (case["T"] // 2 + 1) * 2, flops=rows)
    n = _lens(case, case["L"])
    kept = sum(min(case["keep"], m // BLOCK * BLOCK) + m % BLOCK for m in n)
    return dict(bytes=case["H"] * (sum(n) * 4 + kept * (D * 4 * 2 + 4)), flops=case["H"] * sum(n))


# ---- inputs ------------------------------------------------------------------------------------------------------------------------

def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)


def _keys(g, *shape):
    """Keys [..., heads, D] with four channels of each head ten times as large, as trained models have them."""
    k = _normal(g, *shape)
    ch = torch.rand(shape[-2:], generator=g, device="cuda").argsort(-1)[:, :4]
    return k * torch.ones(shape[-2:], device="cuda", dtype=torch.float16).scatter_(1, ch, 10.0)


def _slopes(case):
    h = torch.arange(1, case["Hq"] + 1, device="cuda", dtype=torch.float32)
    return torch.exp2(-8.0 * h / case["Hq"]) if case.get("alibi") else None


def _len_tensor(case, full, seed):
    n = _lens(case, full)
    random.Random(seed).shuffle(n)
    return torch.tensor(n, dtype=torch.int32, device="cuda")


def _split(x):
    """fp16 values as (high byte, bits 7:4, bits 3:0)."""
    b = x.view(torch.int16).to(torch.int32)
    return ((b >> 8) & 255).to(torch.uint8), ((b >> 4) & 15).to(torch.uint8), (b & 15).to(torch.uint8)


def _pair(n):
    """Nibbles two a byte, the even one in the high half."""
    return (n[..., 0::2] << 4) | n[..., 1::2]


def _planes(x, k_block=None):
    """Planes of fp16 [B, H, L, D]: token-major, or channel-major in blocks of k_block tokens."""
    if k_block is not None:
        B, H, L, D = x.shape
        x = x.view(B, H, L // k_block, k_block, D).transpose(3, 4).contiguous()
    hi, mid, last = _split(x)
    return [hi, _pair(mid), _pair(last)]


def _cache(case, g, H, cap, layers=None):
    """The planes, column maxima and rest buffers of one layer (or `layers` of them, stacked) with room for cap tokens."""
    lead, B, D, kb = [] if layers is None else [layers], case["B"], case["D"], case["k_block"]
    cap = -(-cap // kb) * kb
    n = layers or 1
    k, v = _keys(g, n * B, cap, H, D), _normal(g, n * B, cap, H, D) * 0.5
    kp, vp = _planes(k.transpose(1, 2).contiguous(), kb), _planes(v.transpose(1, 2).contiguous())
    rk, rv = _keys(g, n * B, BLOCK, H, D), _normal(g, n * B, BLOCK, H, D) * 0.5
    expo = lambda x: ((x.view(torch.int16) >> 10) & 31).amax(1, keepdim=True).to(torch.uint8)  # noqa: E731
    shaped = lambda t: t.view(*lead, B, *t.shape[1:])  # noqa: E731
    return dict(k_planes=[shaped(t) for t in kp], v_planes=[shaped(t) for t in vp], k_colmax=shaped(expo(k)), v_colmax=shaped(expo(v)),
                restk=shaped(rk), restv=shaped(rv))


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    op, B = case["op"], case["B"]
    s = dict(case=case)
    if op in ("prefill", "observe"):
        S, Hq, Hkv, D = case["S"], case["Hq"], case["Hkv"], case["D"]
        s.update(q=_normal(g, B, S, Hq, D), k=_keys(g, B, S, Hkv, D), v=_normal(g, B, S, Hkv, D) * 0.5, slopes=_slopes(case), lens=None, prefix=None, docs=None)
        if case.get("docs"):
            n = _doc_sizes(case)
            random.Random(seed).shuffle(n)
            s["docs"] = torch.repeat_interleave(torch.arange(len(n), dtype=torch.int32), torch.tensor(n)).expand(B, S).contiguous().cuda()
        elif case["ragged"]:
            s["lens"] = _len_tensor(case, S, seed)
        if case.get("prefix"):
            n = s["lens"] if s["lens"] is not None else torch.full((B,), S, device="cuda")
            s["prefix"] = (n.double() * case["prefix"]).to(torch.int32)
        if op == "observe":
            n = s["lens"].long() if s["lens"] is not None else torch.full((B,), S, device="cuda")
            rows = (n[:, None] - case["window"] + torch.arange(case["window"], device="cuda")).clamp(min=0)      # [B, window]
            sc = _scores_of_rows(s, rows, torch.float32)
            s["lse"] = torch.zeros(B, Hq, S, device="cuda").scatter_(2, rows[:, None].expand(B, Hq, -1), torch.logsumexp(sc, -1))
    elif op == "accumulate":
        L, Hq = case["L"], case["Hq"]
        width = -(-(L + 1) // BLOCK) * BLOCK
        s["lens"] = _len_tensor(case, L, seed)
        sc = torch.randn(B, Hq, width, generator=g, device="cuda") * 2
        sc = sc.masked_fill(torch.arange(width, device="cuda") >= s["lens"].view(B, 1, 1), -math.inf)
        s["probs"] = torch.softmax(sc, -1).half()
        s["weights"] = torch.rand(B, case["Hkv"], L, generator=g, device="cuda")
        s["out"] = torch.zeros_like(s["weights"])
    elif op == "tree":
        T, Hq, Hkv, D = case["T"], case["Hq"], case["Hkv"], case["D"]
        s.update(_cache(case, g, Hkv, case["L"]), lens=_len_tensor(case, case["L"], seed), q=_normal(g, B, T, Hq, D), k=_keys(g, B, T, Hkv, D),
                 v=_normal(g, B, T, Hkv, D) * 0.5, slopes=_slopes(case))
        r, masks = random.Random(seed), []
        for _ in range(B):          # each draft hangs on an earlier one or on the cache
            row = []
            for t in range(T):
                parent = r.randint(max(-1, t - 4), t - 1)
                row.append((1 << t) | (row[parent] if parent >= 0 else 0))
            masks.append([m - (1 << 64) if m >> 63 else m for m in row])
        s["ancestors"] = torch.tensor(masks, dtype=torch.int64, device="cuda")
    elif op == "commit":
        N, T, H, D = case["layers"], case["T"], case["H"], case["D"]
        s.update(_cache(case, g, H, case["L"] + T + BLOCK, N))
        n = _len_tensor(case, case["L"], seed)
        s["start"] = n.expand(N, B).contiguous()
        s["lens"] = s["start"].clone()
        s["restk0"], s["restv0"] = s["restk"].clone(), s["restv"].clone()
        s["k"], s["v"] = _keys(g, N * B, T, H, D).view(N, B, T, H, D), (_normal(g, N * B, T, H, D) * 0.5).view(N, B, T, H, D)
        count = torch.randint(1, T + 1, (B, 1), generator=g, device="cuda")
        at = torch.arange(T, device="cuda")
        path = torch.rand(B, T, generator=g, device="cuda").masked_fill(at >= count, 2.0).argsort(-1)       # `count` drafts of each sequence ...
        path = path.masked_fill(at >= count, T).sort(-1).values                                             # ... in order
        s["accepted"] = path.masked_fill(path >= T, -1).to(torch.int32)
    else:
        H, L = case["H"], case["L"]
        s.update(_cache(case, g, H, L), lens=_len_tensor(case, L, seed))
        cap = s["v_planes"][0].shape[2]
        s["weights"] = torch.rand(B, H, cap, generator=g, device="cuda") ** 4
        room = dict(case, L=case["keep"] + BLOCK)
        s["to"] = {n: [torch.zeros_like(t) for t in v] if isinstance(v, list) else torch.zeros_like(v)
                   for n, v in _cache(room, torch.Generator(device="cuda").manual_seed(0), H, case["keep"] + BLOCK).items()}
        s["to"]["lens"] = torch.zeros_like(s["lens"])
        s["to"]["weights"] = torch.zeros(B, H, s["to"]["v_planes"][0].shape[2], device="cuda")
    return s


# ---- the plain forms ---------------------------------------------------------------------------------------------------------------

def _scores_of_rows(s, rows, dtype):
    """Scores [B, Hq, R, S] of the query rows [B, R] of a prompt, -inf where a row does not see a token."""
    q, k, c = s["q"], s["k"], s["case"]
    B, S, Hq, D = q.shape
    Hkv, R = k.shape[2], rows.shape[1]
    qr = torch.gather(q, 1, rows[:, :, None, None].expand(B, R, Hq, D)).to(dtype)
    qr = qr.view(B, R, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    x = (qr @ k.to(dtype).permute(0, 2, 3, 1).contiguous()).view(B, Hq, R, S) * D ** -0.5
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    i, j = rows[:, :, None], torch.arange(S, device=q.device)
    if s["slopes"] is not None:
        x = x - s["slopes"].to(dtype).view(1, Hq, 1, 1) * (i - j).abs()[:, None]
    see = j <= i
    if s["prefix"] is not None:
        see = see | (j < s["prefix"].view(B, 1, 1))
    if s["lens"] is not None:
        see = see & (j < s["lens"].view(B, 1, 1)) & (i < s["lens"].view(B, 1, 1))
    if s["docs"] is not None:
        see = see & (torch.gather(s["docs"], 1, rows)[:, :, None] == s["docs"][:, None])
    return x.masked_fill_(~see[:, None], -math.inf)


def _softmax(x):
    """exp(x - max) and its sum; a row of -inf gives zeros and a sum of zero."""
    m = x.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, torch.zeros_like(m), m)
    e = torch.exp(x - m)
    return e, e.sum(-1, keepdim=True), m


def _prefill(s):
    q, v = s["q"], s["v"]
    B, S, Hq, D = q.shape
    Hkv = v.shape[2]
    x = _scores_of_rows(s, torch.arange(S, device=q.device).expand(B, S), torch.float32)
    e, l, m = _softmax(x)
    o = (e.view(B, Hkv, -1, S) @ v.float().transpose(1, 2).contiguous()).view(B, Hq, S, D) / l.clamp(min=1e-30)
    return o.transpose(1, 2).half(), (torch.log(l) + m).squeeze(-1)


def _observe(s):
    c, q = s["case"], s["q"]
    B, S, Hq, _ = q.shape
    n = s["lens"].long() if s["lens"] is not None else torch.full((B,), S, device=q.device)
    at = n[:, None] - c["window"] + torch.arange(c["window"], device=q.device)
    rows = at.clamp(min=0)
    x = _scores_of_rows(s, rows, torch.float32)
    p = torch.exp(x - torch.gather(s["lse"], 2, rows[:, None].expand(B, Hq, -1))[..., None])
    p = p.masked_fill((at < 0).view(B, 1, -1, 1), 0.0)
    return p.sum(2).view(B, c["Hkv"], -1, S).sum(2)


def _accumulate(s):
    c = s["case"]
    w, L = s["weights"], s["weights"].shape[-1]
    got = s["probs"][:, :, :L].float().view(c["B"], c["Hkv"], -1, L).sum(2)
    return torch.where(torch.arange(L, device=w.device) < s["lens"].view(-1, 1, 1), w * c["decay"] + got, s["out"])


def _nibbles(p):
    return torch.stack([p >> 4, p & 15], -1).flatten(-2)


def _joined(planes):
    hi, mid, last = planes
    b = (hi.to(torch.int32) << 8) | (_nibbles(mid).to(torch.int32) << 4) | _nibbles(last)
    return b.to(torch.int16).view(torch.float16)


def _cached(s):
    """Keys and values [B, H, cap + 64, D] in 32 bits: the planes, then the rest buffer, and the position of each (its token's, or none)."""
    k = _joined(s["k_planes"]).transpose(3, 4).flatten(2, 3)
    v = _joined(s["v_planes"])
    cap = v.shape[2]
    at = torch.arange(cap, device=v.device).expand(v.shape[0], cap)
    n = s["lens"].long()[:, None]
    flushed = n // BLOCK * BLOCK
    rest = flushed + torch.arange(BLOCK, device=v.device)
    pos = torch.cat([at.masked_fill(at >= flushed, -1), rest.masked_fill(rest >= n, -1)], 1)
    join = lambda a, r: torch.cat([a, r.transpose(1, 2)], 2).float()  # noqa: E731
    return join(k, s["restk"]), join(v, s["restv"]), pos


def _tree(s):
    c, q = s["case"], s["q"]
    B, T, Hq, D = q.shape
    Hkv = c["Hkv"]
    k, v, pos = _cached(s)
    k, v = torch.cat([k, s["k"].transpose(1, 2).float()], 2), torch.cat([v, s["v"].transpose(1, 2).float()], 2)
    bits = (s["ancestors"][:, :, None] >> torch.arange(T, device=q.device)) & 1                  # [B, T, T]
    depth = s["lens"].long()[:, None] + bits.sum(-1) - torch.diagonal(bits, dim1=1, dim2=2)      # [B, T]
    see = torch.cat([(pos >= 0)[:, None].expand(-1, T, -1), bits.bool()], 2)
    gap = (depth[:, :, None] - torch.cat([pos, depth], 1)[:, None]).abs()
    qg = q.float().view(B, T, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    x = (qg @ k.transpose(2, 3).contiguous()).view(B, Hq, T, -1) * D ** -0.5
    if c["softcap"]:
        x = torch.tanh(x / c["softcap"]) * c["softcap"]
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, Hq, 1, 1) * gap[:, None]
    e, l, _ = _softmax(x.masked_fill(~see[:, None], -math.inf))
    v = v.masked_fill(~see.any(1)[:, None, :, None], 0.0)
    o = (e.view(B, Hkv, -1, e.shape[-1]) @ v).view(B, Hq, T, D) / l.clamp(min=1e-30)
    return o.transpose(1, 2).half()


def _expo(x):
    return ((x.view(torch.int16) >> 10) & 31).to(torch.uint8)


def _commit(s):
    c, dev = s["case"], s["k"].device
    N, B, T, H, D = s["k"].shape
    kb = c["k_block"]
    n = s["lens"][0].long()
    r, bi = n % BLOCK, torch.arange(B, device=dev)
    ok = (s["accepted"] >= 0).long().cumprod(1).bool()                                           # [B, A]
    count = ok.sum(1)
    pick = s["accepted"].long().clamp(min=0)
    row = torch.where(ok, r[:, None] + torch.arange(T, device=dev), 2 * BLOCK)                   # beyond the last row: dropped
    flush, left = r + count >= BLOCK, (r + count - BLOCK).clamp(min=0)
    blk, sub = (n - r) // kb, (n - r) % kb // BLOCK
    for x, planes, rest, colmax, k_side in ((s["k"], s["k_planes"], s["restk"], s["k_colmax"], True), (s["v"], s["v_planes"], s["restv"], s["v_colmax"], False)):
        got = x[:, bi[:, None], pick]                                                            # [N, B, A, H, D]
        grown = torch.cat([rest, torch.zeros(N, B, BLOCK + 1, H, D, dtype=x.dtype, device=dev)], 2)
        grown[:, bi[:, None], row] = got
        tile = grown[:, :, :BLOCK].transpose(2, 3)                                               # [N, B, H, 64, D]
        parts = _split(tile.transpose(3, 4).contiguous() if k_side else tile.contiguous())
        for p, part in zip(planes, (parts[0], _pair(parts[1]), _pair(parts[2]))):
            if k_side:
                at = p.view(*p.shape[:-1], kb // BLOCK, -1)
                old = at[:, bi, :, blk, :, sub]                                                  # [B, N, H, D, 64]
                at[:, bi, :, blk, :, sub] = torch.where(flush.view(B, 1, 1, 1, 1), part.transpose(0, 1), old)
            else:
                at = p.view(N, B, H, -1, BLOCK, p.shape[-1])
                old = at[:, bi, :, (n - r) // BLOCK]                                             # [B, N, H, 64, D]
                at[:, bi, :, (n - r) // BLOCK] = torch.where(flush.view(B, 1, 1, 1, 1), part.transpose(0, 1), old)
        j = torch.arange(BLOCK, device=dev)
        appended = (j >= r[:, None]) & (j < (r + count)[:, None]) & ~flush[:, None]
        moved = flush[:, None] & (j < left[:, None])
        rest.copy_(torch.where(moved.view(1, B, BLOCK, 1, 1), grown[:, :, BLOCK:2 * BLOCK], torch.where(appended.view(1, B, BLOCK, 1, 1), grown[:, :, :BLOCK], rest)))
        colmax.copy_(torch.maximum(colmax, _expo(got).masked_fill(~ok.view(1, B, T, 1, 1), 0).amax(2, keepdim=True)))
    s["lens"].add_(count.to(torch.int32))


def _select(w, lens, c):
    """The kept tokens of each (sequence, head), ascending, -1 behind the last."""
    B, H, cap = w.shape
    j, flushed = torch.arange(cap, device=w.device), (lens.long() // BLOCK * BLOCK).view(B, 1, 1)
    must = (j < c["sinks"]) | (j >= lens.long().view(B, 1, 1) - c["recent"])
    key = torch.where(must.expand(B, H, cap), math.inf, w).masked_fill((j >= flushed).expand(B, H, cap), -math.inf)
    best = key.sort(dim=-1, descending=True, stable=True).indices[..., :c["keep"]]
    best = torch.where(torch.arange(best.shape[-1], device=w.device) < flushed, best, cap).sort(-1).values
    best = torch.nn.functional.pad(best, (0, c["keep"] - best.shape[-1]), value=cap)
    return torch.where(best == cap, -1, best)


def _evict(s):
    c, to, w = s["case"], s["to"], s["weights"]
    B, H, cap = w.shape
    kept = _select(w, s["lens"], c)                                                              # [B, H, keep]
    room = to["v_planes"][0].shape[2]
    n = s["lens"].long()
    flushed = n // BLOCK * BLOCK
    have = flushed.clamp(max=c["keep"])
    src = torch.nn.functional.pad(kept, (0, room - c["keep"]), value=-1)
    fill = src >= 0
    at = src.clamp(min=0)
    for p, t, per in zip(s["v_planes"], to["v_planes"], (1, 2, 2)):
        t.copy_(torch.where(fill[..., None], torch.gather(p, 2, at[..., None].expand(*at.shape, p.shape[-1])), t))
    flat = lambda p: p.transpose(3, 4).flatten(2, 3)  # noqa: E731
    kb, D = c["k_block"], c["D"]
    hi, mid, last = s["k_planes"]
    for i, p in enumerate((hi, _nibbles(mid), _nibbles(last))):
        got = torch.gather(flat(p), 2, at[..., None].expand(*at.shape, D))                       # [B, H, room, D]
        t = to["k_planes"][i]
        old = flat(t if i == 0 else _nibbles(t))
        new = torch.where(fill[..., None], got, old).view(B, H, -1, kb, D).transpose(3, 4).contiguous()
        t.copy_(new if i == 0 else _pair(new))
    j = torch.arange(room, device=w.device)
    rest_at = (flushed - have).view(B, 1, 1) + j                                                 # where a rest token's weight comes from
    rest_in = (j >= have.view(B, 1, 1)) & (j < (n - flushed + have).view(B, 1, 1))
    moved = torch.gather(w, 2, rest_at.clamp(max=cap - 1).expand(B, H, room))
    to["weights"].copy_(torch.where(fill, torch.gather(w, 2, at), torch.where(rest_in, moved, 0.0)))
    to["restk"].copy_(s["restk"])
    to["restv"].copy_(s["restv"])
    to["k_colmax"].copy_(s["k_colmax"])
    to["v_colmax"].copy_(s["v_colmax"])
    to["lens"].copy_(n - flushed + have)
    return kept.to(torch.int32)


def _handles(s):
    """The framework's descriptors of a cache's layers, which a program makes once, when it makes the cache."""
    if "handles" not in s:
        from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
        parts = (*s["k_planes"], *s["v_planes"], s["k_colmax"], s["v_colmax"], s["restk"], s["restv"], s["lens"])
        rows = zip(*parts) if s["lens"].dim() == 2 else [parts]
        s["handles"] = [cuda_module.prepare_layer(r[0:3], r[3:6], *r[6:]) for r in rows]
    return s["handles"]


def run(state):
    s = state
    c = s["case"]
    op = c["op"]
    if own:
        from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
    if op == "prefill":
        if own:
            return cuda_module.prefill_attention(s["q"], s["k"], s["v"], softcap=c["softcap"], slopes=s["slopes"], seq_lens=s["lens"], prefix_lens=s["prefix"],
                                                 documents=s["docs"], return_lse=True)
        return _prefill(s)
    if op == "observe":
        if own:
            return cuda_module.attention_weights(s["q"], s["k"], s["lse"], softcap=c["softcap"], slopes=s["slopes"], seq_lens=s["lens"], window=c["window"])
        return _observe(s)
    if op == "accumulate":
        if own:
            return cuda_module.accumulate_weights(s["weights"], s["probs"], s["lens"], decay=c["decay"], out=s["out"])
        return _accumulate(s)
    if op == "tree":
        if own:
            return cuda_module.tree_attention(_handles(s)[0], s["q"], s["k"], s["v"], s["ancestors"], softcap=c["softcap"], slopes=s["slopes"], bound=c["L"])
        return _tree(s)
    if op == "commit":
        # every pass starts from the same cache: the rest buffers and the lengths are taken back first
        torch._foreach_copy_([s["restk"], s["restv"], s["lens"]], [s["restk0"], s["restv0"], s["start"]])
        if own:
            cuda_module.tree_commit(_handles(s), s["k"], s["v"], s["accepted"])
        else:
            _commit(s)
        return {n: s[n] for n in ("k_planes", "v_planes", "k_colmax", "v_colmax", "restk", "restv", "lens")}
    if own:
        kept = cuda_module.evict(_handles(s)[0], s["weights"], c["keep"], sinks=c["sinks"], recent=c["recent"], into=_handles(s["to"])[0],
                                 into_weights=s["to"]["weights"])
    else:
        kept = _evict(s)
    return dict({n: s["to"][n] for n in ("k_planes", "v_planes", "k_colmax", "v_colmax", "restk", "restv", "lens", "weights")}, kept=kept)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------------

def _attend(x, v):
    """Weights and outputs of one head from its scores [R, N] (-inf: not seen) and values [N, D]."""
    top = x.max(1, keepdim=True).values.nan_to_num(neginf=0.0)
    e = (x - top).exp()
    z = e.sum(1, keepdim=True)
    o = e @ v / torch.where(z > 0, z, torch.ones_like(z))
    return o, (z.log() + top)[:, 0]


def _modified(x, case, slope, gap):
    if case["softcap"]:
        x = case["softcap"] * (x / case["softcap"]).tanh()
    return x if slope is None else x - slope.double() * gap


def exact(case, seed):
    s = prepare(case, seed)
    op, B = case["op"], case["B"]
    if op in ("prefill", "observe"):
        q, k, v = s["q"], s["k"].double(), s["v"].double()
        S, Hq, D, G = case["S"], case["Hq"], case["D"], case["Hq"] // case["Hkv"]
        o, lse = torch.zeros(B, S, Hq, D, dtype=torch.float64, device="cuda"), torch.full((B, Hq, S), -math.inf, dtype=torch.float64, device="cuda")
        seen = torch.zeros(B, case["Hkv"], S, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = int(s["lens"][b]) if s["lens"] is not None else S
            first = max(0, n - case["window"]) if op == "observe" else 0
            i, j = torch.arange(first, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            hidden = j > i
            if s["prefix"] is not None:
                hidden &= j >= int(s["prefix"][b])
            if s["docs"] is not None:
                hidden |= s["docs"][b][i] != s["docs"][b][j]
            for h in range(Hq):
                x = _modified(q[b, first:n, h].double() @ k[b, :n, h // G].T.contiguous() / math.sqrt(D), case, None if s["slopes"] is None else s["slopes"][h], (i - j).abs())
                x[hidden] = -math.inf
                if op == "observe":
                    seen[b, h // G, :n] += (x - s["lse"][b, h, first:n].double()[:, None]).exp().sum(0)
                else:
                    o[b, :n, h], lse[b, h, :n] = _attend(x, v[b, :n, h // G])
        return seen if op == "observe" else (o, lse)
    if op == "accumulate":
        w = s["out"].double()
        for b in range(B):
            n, G = int(s["lens"][b]), case["Hq"] // case["Hkv"]
            w[b, :, :n] = s["weights"][b, :, :n].double() * case["decay"]
            for h in range(case["Hq"]):
                w[b, h // G, :n] += s["probs"][b, h, :n].double()
        return w
    if op == "tree":
        T, Hq, D, G = case["T"], case["Hq"], case["D"], case["Hq"] // case["Hkv"]
        o = torch.zeros(B, T, Hq, D, dtype=torch.float64, device="cuda")
        for b in range(B):
            n = int(s["lens"][b])
            whole = n - n % BLOCK
            masks = [int(m) & ((1 << 64) - 1) for m in s["ancestors"][b]]
            place = torch.tensor([n + bin(m).count("1") - 1 for m in masks], device="cuda")
            hidden = torch.tensor([[not (m >> u) & 1 for u in range(T)] for m in masks], device="cuda")
            gap = (place[:, None] - torch.cat([torch.arange(n, device="cuda"), place])[None]).abs()
            for h in range(case["Hkv"]):
                sides = []
                for planes, rest, new in ((s["k_planes"], s["restk"], s["k"]), (s["v_planes"], s["restv"], s["v"])):
                    if planes is s["k_planes"]:
                        rows = [p[b, h].permute(0, 2, 1).reshape(-1, D) for p in (planes[0], _nibbles(planes[1]), _nibbles(planes[2]))]
                    else:
                        rows = [planes[0][b, h], _nibbles(planes[1][b, h]), _nibbles(planes[2][b, h])]
                    word = rows[0][:whole].int() * 256 + rows[1][:whole].int() * 16 + rows[2][:whole].int()
                    sides.append(torch.cat([word.to(torch.int16).view(torch.float16), rest[b, :n - whole, h], new[b, :, h]]).double())
                for a in range(h * G, h * G + G):
                    x = _modified(s["q"][b, :, a].double() @ sides[0].T.contiguous() / math.sqrt(D), case, None if s["slopes"] is None else s["slopes"][a], gap)
                    x[:, n:][hidden] = -math.inf
                    o[b, :, a] = _attend(x, sides[1])[0]
        return o
    return None
