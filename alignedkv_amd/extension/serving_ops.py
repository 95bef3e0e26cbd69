"""Serving operators over the split-plane cache as methods of `cuda_module`: prompt attention (capped, biased and masked scores),
the attention weight tokens received, attention of a tree of drafted tokens, the commit of accepted drafts, and eviction by
accumulated weight.  No counterpart in the reference.  Marshalling over the C ABI (include/alignedkv.h): shapes and strides
come from the tensors, which are fp16 / fp32 / int32 here rather than uint8 views; every launch goes to the current stream of the
tensors' device; workspaces come from torch's allocator per call (inside a graph capture: from the graph's own pool)."""
from __future__ import annotations

import ctypes
import math

import torch

from .._lib import CacheLayer, PromptDesc, check, load_library
from .KV_cache_cpp_extention import _AlignedKVModule, _ptr, _require, _stream_ptr

rest_tokens = 64


def _tensor(name, t, dtype, shape, device=None, contiguous=True):
    """Checks one argument; shape entries of None are free.  (A call is a few microseconds of host time altogether: the common case is
    told in one expression, what is wrong with an argument is worked out only where something is.)"""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.is_cuda and t.shape == shape and (device is None or t.device == device) \
            and (not contiguous or t.is_contiguous()):
        return t
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if t.dtype != dtype:
        raise RuntimeError(f"{name}: expected dtype {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"{name}: expected a tensor on the GPU, got device {t.device}")
    if device is not None and t.device != device:
        raise RuntimeError(f"{name}: on {t.device}, other arguments on {device}")
    if t.dim() != len(shape) or any(w is not None and s != w for s, w in zip(t.shape, shape)):
        want = "[" + ", ".join("*" if w is None else str(w) for w in shape) + "]"
        raise RuntimeError(f"{name}: expected shape {want}, got {list(t.shape)}")
    if contiguous and not t.is_contiguous():
        raise RuntimeError(f"{name}: must be contiguous")
    return t


def _dims(name, t, n):
    """The shape of an argument of n dimensions."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    s = t.shape
    if len(s) != n:
        raise RuntimeError(f"{name}: expected {n} dimensions, got shape {list(s)}")
    return s


def _call(fn, device, *args):
    """One library call on `device`, its current stream last; raises what the library reports."""
    if device.index == torch.cuda.current_device():
        rc = fn(*args, _stream_ptr(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, _stream_ptr(device))
    if rc != 0:
        check(rc)


def _number(name, x, low, strict):
    x = float(x)
    if not math.isfinite(x) or x < low or (strict and x == low) or x >= 1e30:
        raise RuntimeError(f"{name}: {x} must be finite and {'above' if strict else 'at least'} {low}")
    return x


def _apart(name, out, *inputs):
    """Refuses an `out` that shares memory with an input: workgroups write theirs while others still read."""
    def span(t):
        return t.data_ptr(), t.data_ptr() + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()
    lo, hi = span(out)
    for t in inputs:
        if t is not None and t.numel():
            a, b = span(t)
            if a < hi and lo < b:
                raise RuntimeError(f"{name}: overlaps an input")


def _strided(name, t):
    """(pointer, strides) of a [batch, tokens, heads, head_dim] fp16 view, or of a contiguous copy where the kernels cannot read the view."""
    a, b, c, d = s = t.stride()
    if d != 1 or (a | b | c) & 7 or b >= 1 << 24 or t.data_ptr() & 15:
        a, b, c = s = _used_strides(t)      # (torch calls a tensor contiguous whatever the strides of its dimensions of one entry)
        if d != 1 or (a | b | c) & 7 or b >= 1 << 24 or t.data_ptr() & 15:
            t = t.contiguous()
            if t.data_ptr() % 16:
                t = t.clone()
            s = _used_strides(t)
    return t, s


def _used_strides(t):
    """The strides but the last, 0 where a dimension has one entry."""
    return tuple(0 if n == 1 else x for n, x in zip(t.shape[:3], t.stride()))


def _prompt(q, k, v, scale, softcap, slopes, seq_lens, prefix_lens, documents):
    """An akv_prompt_desc, what it describes (B, S, Hq, Hkv, D), the device, and the tensors behind it."""
    B, S, Hq, D = shape = _dims("q", q, 4)
    dev = q.device
    _tensor("q", q, torch.half, shape, contiguous=False)
    Hkv = _dims("k", k, 4)[2]
    _tensor("k", k, torch.half, (B, S, Hkv, D), dev, contiguous=False)
    if v is not None:
        _tensor("v", v, torch.half, (B, S, Hkv, D), dev, contiguous=False)
    if D not in (64, 128, 256):
        raise RuntimeError(f"head_dim {D}: 64, 128 or 256")
    if B < 1 or S < 1 or Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise RuntimeError(f"q {list(q.shape)} and k {list(k.shape)}: at least one sequence and token, query heads a multiple of the KV heads")
    scale = D ** -0.5 if scale is None else _number("scale", scale, 0.0, True)
    softcap = _number("softcap", softcap, 0.0, False) if softcap else 0.0
    if slopes is not None:
        _tensor("slopes", slopes, torch.float32, (Hq,), dev)
    if seq_lens is not None:
        _tensor("seq_lens", seq_lens, torch.int32, (B,), dev)
    if prefix_lens is not None:
        _tensor("prefix_lens", prefix_lens, torch.int32, (B,), dev)
    if documents is not None:
        _tensor("documents", documents, torch.int32, (B, S), dev)
    q, qs = _strided("q", q)
    k, ks = _strided("k", k)
    vp, vs = None, ks
    if v is not None:
        v, vs = _strided("v", v)
        vp = v.data_ptr()
    desc = PromptDesc(q.data_ptr(), k.data_ptr(), vp, *qs[:3], *ks[:3], *vs[:3], _ptr(slopes), _ptr(seq_lens), _ptr(prefix_lens), _ptr(documents),
                      B, S, Hq, Hkv, D, scale, softcap)
    return desc, (B, S, Hq, Hkv, D), dev, (q, k, v)


def prefill_attention(self, q, k, v, *, scale=None, softcap=0.0, slopes=None, seq_lens=None, prefix_lens=None, documents=None, out=None,
                      return_lse=False):
    """Causal attention of a batch of prompts: q fp16 [B, S, Hq, D], k, v fp16 [B, S, Hkv, D] (views with a dense last dimension are read in
    place); returns fp16 [B, S, Hq, D], with return_lse also fp32 [B, Hq, S].
    score(i, j) = cap(scale q_i . k_j) - slopes[h] |i - j|, cap(x) = softcap tanh(x / softcap) (softcap 0: x); scale: 1 / sqrt(D).
    seq_lens int32 [B]: tokens at and beyond a length are padding (rows of zeros, lse -inf; with `out` given these rows are left as
    they were); prefix_lens int32 [B]: the first tokens are seen by every row; documents int32 [B, S]: rows see tokens of their own
    document only (several prompts packed in one row; a negative id sees nothing and is not seen).
    No gradient is recorded, as by every operator here."""
    lib = load_library()
    if v is None:
        raise TypeError("v: expected a torch.Tensor, got NoneType")
    desc, (B, S, Hq, _, D), dev, held = _prompt(q, k, v, scale, softcap, slopes, seq_lens, prefix_lens, documents)
    fill = out is None
    if fill:
        out = torch.empty((B, S, Hq, D), dtype=torch.half, device=dev)
    else:
        _tensor("out", out, torch.half, (B, S, Hq, D), dev)
        _apart("out", out, *held, slopes, seq_lens, prefix_lens, documents)
    lse = torch.empty((B, Hq, S), dtype=torch.float32, device=dev) if return_lse else None
    if lse is not None and not fill and seq_lens is not None:
        lse.fill_(-math.inf)
    ws, need = None, 0
    if documents is not None:
        need = lib.akv_prefill_attention_workspace_bytes(B, S)
        ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(lib.akv_prefill_attention, dev, ctypes.byref(desc), out.data_ptr(), _ptr(lse), 1 if fill else 0, _ptr(ws), need)
    return (out, lse) if return_lse else out


def attention_weights(self, q, k, lse, *, scale=None, softcap=0.0, slopes=None, seq_lens=None, prefix_lens=None, documents=None, window=0,
                      out=None):
    """The attention weight every prompt token received: fp32 [B, Hkv, S], summed over the query heads of each KV head and the last
    `window` rows of each sequence (0: all rows).  lse: what prefill_attention returned for the same q, k, masks and score form.
    out: fp32 [B, Hkv, >= S] (dense last dimension) to add the weights to instead; it is returned."""
    lib = load_library()
    desc, (B, S, Hq, Hkv, D), dev, (q, k, _) = _prompt(q, k, None, scale, softcap, slopes, seq_lens, prefix_lens, documents)
    _tensor("lse", lse, torch.float32, (B, Hq, S), dev)
    window = int(window)
    if window < 0:
        raise RuntimeError(f"window: {window} must be 0 (every row) or positive")
    add = out is not None
    if not add:
        out = torch.empty((B, Hkv, S), dtype=torch.float32, device=dev)
    else:
        _weights("out", out, B, Hkv, S, dev)
        _apart("out", out, q, k, lse, slopes, seq_lens, prefix_lens, documents)
    _call(lib.akv_attention_weights, dev, ctypes.byref(desc), lse.data_ptr(), min(window, 1 << 30), out.data_ptr(), out.stride(0), out.stride(1),
          1 if add else 0)
    return out


def _weights(name, t, B, H, n, device):
    """An accumulator: fp32 [B, H, >= n], rows dense and apart, sequence by sequence or head by head."""
    have = _dims(name, t, 3)[2]
    _tensor(name, t, torch.float32, (B, H, have), device, contiguous=False)
    if have >= n and t.is_contiguous():
        return t
    if have < n:
        raise RuntimeError(f"{name}: rows of {t.shape[2]} weights for {n} tokens")
    b, h, d = t.stride()
    by_sequence = (H == 1 or h >= have) and (B == 1 or b >= (H - 1) * h + have)
    by_head = (B == 1 or b >= have) and (H == 1 or h >= (B - 1) * b + have)
    if (d != 1 and have > 1) or not (by_sequence or by_head):
        raise RuntimeError(f"{name}: rows must be dense and must not overlap")
    return t


def accumulate_weights(self, weights, probs, seq_lens, *, decay=1.0, out=None):
    """Adds one decode step's probabilities to the accumulated weights: out[b, h, t] = decay * weights[b, h, t] + sum over the query heads
    of KV head h of probs[b, :, t] for t < seq_lens[b]; other entries are left as they were.  weights fp32 [B, Hkv, capacity]; probs
    fp16 [B, Hq, width], the record of the fused step (width a multiple of 8, at least the capacity); seq_lens int32 [B] after the step.
    out: where the sums go (default: weights itself); it is returned."""
    lib = load_library()
    B, Hq, width = shape = _dims("probs", probs, 3)
    dev = probs.device
    _tensor("probs", probs, torch.half, shape)
    _, Hkv, cap = _dims("weights", weights, 3)
    _weights("weights", weights, B, Hkv, cap, dev)
    if Hkv < 1 or Hq < 1 or Hq % Hkv:
        raise RuntimeError(f"probs {list(probs.shape)}, weights {list(weights.shape)}: query heads must be a multiple of the KV heads")
    if width % 8 or probs.data_ptr() % 16 or not 1 <= cap <= width:
        raise RuntimeError(f"probs: rows of {width} probabilities must be 16-byte aligned and cover the {cap} weights")
    _tensor("seq_lens", seq_lens, torch.int32, (B,), dev)
    decay = float(decay)
    if not math.isfinite(decay):
        raise RuntimeError("decay: must be finite")
    if out is None:
        out = weights
    else:
        _weights("out", out, B, Hkv, cap, dev)
    (wb, wh, _), (ob, oh, _), w, o, p, n = weights.stride(), out.stride(), weights.data_ptr(), out.data_ptr(), probs.data_ptr(), seq_lens.data_ptr()
    end = o + 4 * ((B - 1) * ob + (Hkv - 1) * oh + cap)
    if ((w != o or wb != ob or wh != oh) and w < end and o < w + 4 * ((B - 1) * wb + (Hkv - 1) * wh + cap)) or (p < end and o < p + 2 * B * Hq * width) \
            or (n < end and o < n + 4 * B):
        raise RuntimeError("out: overlaps an input")
    _call(lib.akv_accumulate_weights, dev, w, wb, wh, probs.data_ptr(), width, seq_lens.data_ptr(), o, ob, oh, B, Hq, Hkv, cap, decay)
    return out


class PreparedLayer:
    """One layer of a cache with a length per sequence, checked once: an akv_cache_layer and the tensors behind it.  Made by
    `cuda_module.prepare_layer`; the tensors must stay the ones it was made of."""

    def __init__(self, desc, device, keep):
        self.desc = desc
        self.device = device
        self.kind = (device, desc.bsz, desc.n_kv_heads, desc.head_dim)
        self.lens = desc.seq_lens
        self.pointers = tuple(t.data_ptr() for t in keep)
        self.places = frozenset(self.pointers)
        self._keep = keep

    def made_of(self, tensors) -> bool:
        """Whether these are the tensors it was made of."""
        return all(x is y for x, y in zip(self._keep, tensors))

    @property
    def seq_lens(self):
        return self._keep[-1]

    @property
    def tensors(self):
        return self._keep


def prepare_layer(self, k_planes, v_planes, k_exp_column_max, v_exp_column_max, restk, restv, seq_lens):
    """k_planes uint8 [B, H, blocks, D, k_block], [.., k_block / 2] twice; v_planes uint8 [B, H, capacity, D], [.., D / 2] twice; column maxima
    uint8 [B, 1, H, D]; restk, restv fp16 [B, 64, H, D]; seq_lens int32 [B].  Sequence b holds seq_lens[b] tokens, the whole 64s of them
    in the planes, the others in the rest buffers."""
    if len(k_planes) != 3 or len(v_planes) != 3:
        raise RuntimeError("k_planes and v_planes: three planes each (first_8, mid_4, last_4)")
    _tensor("k_first_8", k_planes[0], torch.uint8, (None,) * 5)
    B, H, blocks, D, kb = k_planes[0].shape
    dev = k_planes[0].device
    for name, t in (("k_mid_4", k_planes[1]), ("k_last_4", k_planes[2])):
        _tensor(name, t, torch.uint8, (B, H, blocks, D, kb // 2), dev)
    _tensor("v_first_8", v_planes[0], torch.uint8, (B, H, None, D), dev)
    cap = v_planes[0].shape[2]
    for name, t in (("v_mid_4", v_planes[1]), ("v_last_4", v_planes[2])):
        _tensor(name, t, torch.uint8, (B, H, cap, D // 2), dev)
    for name, t in (("k_exp_column_max", k_exp_column_max), ("v_exp_column_max", v_exp_column_max)):
        _tensor(name, t, torch.uint8, (B, 1, H, D), dev)
    for name, t in (("restk", restk), ("restv", restv)):
        _tensor(name, t, torch.half, (B, rest_tokens, H, D), dev)
    _tensor("seq_lens", seq_lens, torch.int32, (B,), dev)
    if D not in (64, 128, 256):
        raise RuntimeError(f"head_dim {D}: 64, 128 or 256")
    if kb not in (64, 256):
        raise RuntimeError(f"k_block {kb}: 64 or 256")
    if cap < 1 or blocks * kb < cap // rest_tokens * rest_tokens:
        raise RuntimeError(f"{blocks} K blocks of {kb} tokens for a capacity of {cap}")
    if not 1 <= B * H <= 65535:
        raise RuntimeError(f"{B} sequences x {H} KV heads: at least 1 and at most 65535 together")
    parts = (*k_planes, *v_planes, k_exp_column_max, v_exp_column_max, restk, restv, seq_lens)
    for t in (*k_planes, *v_planes, restk, restv):
        if t.data_ptr() % 16:
            raise RuntimeError("planes and rest buffers must be 16-byte aligned")
    return PreparedLayer(CacheLayer(*(t.data_ptr() for t in parts), B, H, blocks, cap, D, kb), dev, parts)


def _layer(self, layer):
    return layer if isinstance(layer, PreparedLayer) else self.prepare_layer(*layer)


def _aligned(t):
    if not t.is_contiguous():
        t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def tree_attention(self, layer, q, k, v, ancestors=None, *, scale=None, softcap=0.0, slopes=None, bound=None, out=None):
    """Attention of T drafted tokens per sequence (1 to 64) over the whole cache and over the drafts each of them sees: q fp16
    [B, T, Hq, D], k, v fp16 [B, T, Hkv, D]; returns fp16 [B, T, Hq, D].  Every plane is read (no fetch decisions); the cache is not
    changed.  layer: a PreparedLayer, or the seven arguments of prepare_layer.
    ancestors int64 [T] or [B, T]: bit u of entry t: draft t sees draft u (its own bit included); default: a chain, each draft sees
    itself and those before it.  Bits at and beyond T are not looked at.  Draft t stands at position length + (other drafts it sees), which
    is what `slopes` measures distances from.
    bound: upper bound of the lengths that sizes the launch (default: the capacity)."""
    lib = load_library()
    layer = _layer(self, layer)
    c, dev = layer.desc, layer.device
    B, H, D = c.bsz, c.n_kv_heads, c.head_dim
    _, T, Hq, _ = _dims("q", q, 4)
    _tensor("q", q, torch.half, (B, T, Hq, D), dev, contiguous=False)
    if not 1 <= T <= 64:
        raise RuntimeError(f"{T} drafted tokens: 1 to 64")
    if Hq < 1 or Hq % H:
        raise RuntimeError(f"{Hq} query heads: a multiple of the {H} KV heads")
    _tensor("k", k, torch.half, (B, T, H, D), dev, contiguous=False)
    _tensor("v", v, torch.half, (B, T, H, D), dev, contiguous=False)
    if ancestors is None:
        ancestors = chain_ancestors(T, dev)
    else:
        _tensor("ancestors", ancestors, torch.int64, (T,) if ancestors.dim() == 1 else (B, T), dev)
    scale = D ** -0.5 if scale is None else _number("scale", scale, 0.0, True)
    softcap = _number("softcap", softcap, 0.0, False) if softcap else 0.0
    if slopes is not None:
        _tensor("slopes", slopes, torch.float32, (Hq,), dev)
    bound = c.max_seq_len if bound is None else int(bound)
    if not 0 <= bound <= c.max_seq_len:
        raise RuntimeError(f"bound: {bound} outside [0, {c.max_seq_len}]")
    q, k, v = _aligned(q), _aligned(k), _aligned(v)
    if out is None:
        out = torch.empty((B, T, Hq, D), dtype=torch.half, device=dev)
    else:
        _tensor("out", out, torch.half, (B, T, Hq, D), dev)
        _apart("out", out, q, k, v, ancestors, slopes, *layer.tensors)
    need = lib.akv_tree_attention_workspace_bytes(B, Hq, H, D, T, bound)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    _call(lib.akv_tree_attention, dev, ctypes.byref(c), q.data_ptr(), k.data_ptr(), v.data_ptr(), ancestors.data_ptr(),
          1 if ancestors.dim() == 2 else 0, _ptr(slopes), scale, softcap, out.data_ptr(), T, Hq, bound, ws.data_ptr(), need)
    return out


def tree_commit(self, layers, k, v, accepted):
    """Appends accepted drafts to the cache of every layer, as that many decode steps would.  layers: a list of PreparedLayers (or of
    prepare_layer's arguments) of one shape; k, v: fp16 [layers, B, T, Hkv, D], or a list of [B, T, Hkv, D]; accepted int32 [B, A]
    (A at most 64): the accepted drafts of each sequence in order, ended by any entry outside [0, T), -1 say.  Tokens beyond the
    capacity are dropped."""
    lib = load_library()
    layers = [x if type(x) is PreparedLayer else self.prepare_layer(*x) for x in layers]
    if not layers:
        raise RuntimeError("layers: at least one")
    N, c, dev = len(layers), layers[0].desc, layers[0].device
    shape, kind = (c.bsz, None, c.n_kv_heads, c.head_dim), layers[0].kind
    for i, x in enumerate(layers):
        if x.kind != kind:
            raise RuntimeError(f"layers: layer {i} has another shape or device than layer 0")
    if len({x.lens for x in layers}) != N:
        raise RuntimeError("layers: the same layer (or the same lengths) twice")
    pointers, keep, T = [], [], None
    for name, t in (("k", k), ("v", v)):
        if isinstance(t, torch.Tensor):
            _tensor(name, t, torch.half, (N, c.bsz, _dims(name, t, 5)[2], c.n_kv_heads, c.head_dim), dev, contiguous=False)
            t = _aligned(t)
            keep.append(t)
            step = t.stride(0) * 2
            ps, here = [t.data_ptr() + i * step for i in range(N)], t.shape[2]
        else:
            if len(t) != N:
                raise RuntimeError(f"{name}: {len(t)} tensors for {N} layers")
            t = [_aligned(_tensor(name, x, torch.half, shape, dev, contiguous=False)) for x in t]
            keep.append(t)
            ps, here = [x.data_ptr() for x in t], t[0].shape[1]
            if any(x.shape[1] != here for x in t):
                raise RuntimeError(f"{name}: layers with different numbers of drafts")
        if T is not None and here != T:
            raise RuntimeError(f"v: {here} drafts, k holds {T}")
        T = here
        pointers.append((ctypes.c_void_p * N)(*ps))
    if not 1 <= T <= 64:
        raise RuntimeError(f"{T} drafted tokens: 1 to 64")
    _tensor("accepted", accepted, torch.int32, (c.bsz, _dims("accepted", accepted, 2)[1]), dev)
    if not 1 <= accepted.shape[1] <= 64:
        raise RuntimeError(f"accepted: {accepted.shape[1]} entries a sequence: 1 to 64")
    descs = (CacheLayer * N)(*(x.desc for x in layers))
    _call(lib.akv_tree_commit, dev, descs, N, pointers[0], pointers[1], accepted.data_ptr(), T, accepted.shape[1])


def evict(self, layer, weights, keep, *, sinks=0, recent=0, into=None, into_weights=None):
    """Keeps `keep` (a multiple of 64) of the tokens that each sequence and KV head has in the planes: the first `sinks`, those among
    the newest `recent` of the sequence, then the largest weights (ties: the lower index), in their order; the rest buffer follows and
    the lengths shrink to match.  Returns the kept tokens' old places, int32 [B, Hkv, keep] (-1 behind the last; all tokens where there
    are no more than `keep`).
    layer, into: PreparedLayers (or prepare_layer's arguments); into: another cache of the same batch, heads, head_dim and k_block that
    receives what is kept (default: the cache itself).  weights fp32 [B, Hkv, >= capacity]; they move along within themselves, or into
    into_weights where `into` is given (optional then)."""
    lib = load_library()
    src = _layer(self, layer)
    dst = src if into is None else _layer(self, into)
    c, d, dev = src.desc, dst.desc, src.device
    if src.kind != dst.kind or c.k_block != d.k_block:
        raise RuntimeError("into: must have the batch, heads, head_dim, k_block and device of the cache")
    in_place = src.pointers == dst.pointers
    if not in_place and not src.places.isdisjoint(dst.places):
        raise RuntimeError("into: shares some of its tensors with the cache")
    keep, sinks, recent = int(keep), int(sinks), int(recent)
    if keep < 64 or keep % 64:
        raise RuntimeError(f"keep: {keep} must be a positive multiple of 64")
    if sinks < 0 or recent < 0 or sinks + recent > keep:
        raise RuntimeError(f"sinks {sinks} and recent {recent} must fit into keep {keep}")
    if not in_place and d.max_seq_len < keep + rest_tokens - 1:
        raise RuntimeError(f"into: a capacity of {d.max_seq_len} cannot hold {keep} tokens and a rest buffer")
    B, H = c.bsz, c.n_kv_heads
    _weights("weights", weights, B, H, c.max_seq_len, dev)
    if in_place:
        if into_weights is not None and into_weights is not weights:
            raise RuntimeError("into_weights: in place the weights move within themselves")
        to = weights
    else:
        to = into_weights
        if to is not None:
            _weights("into_weights", to, B, H, keep + rest_tokens - 1, dev)
            if to.untyped_storage().data_ptr() == weights.untyped_storage().data_ptr():
                raise RuntimeError("into_weights: shares its storage with the weights")
    kept = torch.empty((B, H, keep), dtype=torch.int32, device=dev)
    need = lib.akv_evict_workspace_bytes(B, H, c.head_dim, c.k_block, keep, 1 if in_place else 0)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    ts = (to.data_ptr(), to.stride(0), to.stride(1), to.shape[2]) if to is not None else (None, 0, 0, 0)
    _call(lib.akv_evict, dev, ctypes.byref(c), ctypes.byref(d), weights.data_ptr(), weights.stride(0), weights.stride(1), *ts, kept.data_ptr(), keep, sinks,
          recent, ws.data_ptr(), need)
    return kept


def chain_ancestors(T: int, device) -> torch.Tensor:
    """The masks of T drafts in a row: draft t sees 0 .. t."""
    t = torch.arange(T, device=device, dtype=torch.int64)
    return -1 ^ (-2 << t)


def tree_ancestors(parents) -> torch.Tensor:
    """The masks of a tree of drafts from each draft's parent (-1: it follows the cache), a sequence of at most 64 integers in an order in
    which parents come first, or a list of those, one per sequence.  int64 [T] or [B, T] on the CPU."""
    if len(parents) and not isinstance(parents[0], int):
        return torch.stack([tree_ancestors(list(p)) for p in parents])
    masks = []
    if not 1 <= len(parents) <= 64:
        raise RuntimeError(f"{len(parents)} drafted tokens: 1 to 64")
    for t, p in enumerate(parents):
        if not -1 <= p < t:
            raise RuntimeError(f"parents: draft {t} follows draft {p}; parents come first")
        masks.append((1 << t) | (masks[p] if p >= 0 else 0))
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


for _f in (prefill_attention, attention_weights, accumulate_weights, prepare_layer, tree_attention, tree_commit, evict):
    setattr(_AlignedKVModule, _f.__name__, _f)
