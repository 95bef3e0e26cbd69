"""What the serving operators refuse, on the CPU: the C entry points before they touch the GPU, and the checks of the Python layer."""
import ctypes
import math

import pytest
import torch

import alignedkv_amd
from alignedkv_amd import _lib
from alignedkv_amd.extension import serving_ops
from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module

Z = ctypes.c_void_p(0)


@pytest.fixture(scope="module")
def lib():
    import os
    if not os.path.exists(_lib.LIB_PATH):
        alignedkv_amd.build()
    return alignedkv_amd.load_library()


@pytest.fixture(scope="module")
def mem():
    """16-byte aligned host memory standing in for device pointers: nothing is launched."""
    buf = ctypes.create_string_buffer(1 << 12)
    at = (ctypes.addressof(buf) + 255) // 256 * 256
    yield at
    del buf


def prompt(mem, **kw):
    d = _lib.PromptDesc()
    d.q = d.k = d.v = mem
    for n in "qkv":
        kw.setdefault(n + "_stride", (64 * 4 * 16, 64 * 4, 64))
    d.bsz, d.seqlen, d.n_q_heads, d.n_kv_heads, d.head_dim, d.scale, d.softcap = 1, 16, 4, 4, 64, 0.125, 0.0
    for n, x in kw.items():
        if n.endswith("_stride"):
            for i, s in zip("bsh", x):
                setattr(d, f"{n}_{i}", s)
        else:
            setattr(d, n, x)
    return d


def says(lib, rc, *words):
    assert rc == 1
    text = lib.akv_last_error().decode()
    for w in words:
        assert w in text, text


@pytest.mark.parametrize("kw,word", [
    (dict(q=None), "null pointer"), (dict(k=None), "null pointer"), (dict(v=None), "null pointer"), (dict(head_dim=96), "head_dim 96"),
    (dict(bsz=0), "bsz 0"), (dict(seqlen=0), "seqlen 0"), (dict(n_q_heads=6), "heads 6 / 4"), (dict(n_kv_heads=0), "heads"), (dict(n_q_heads=0), "heads"),
    (dict(scale=0.0), "scale"), (dict(scale=math.nan), "scale"), (dict(scale=math.inf), "scale"), (dict(softcap=-1.0), "softcap"), (dict(softcap=math.nan), "softcap"),
    (dict(k_stride=(0, 65, 64)), "multiples of 8"), (dict(v_stride=(0, -64, 64)), "not negative"), (dict(q_stride=(0, 1 << 24, 64)), "2^24"),
    (dict(bsz=70000), "65535"), (dict(seqlen=1 << 30, bsz=60000), "too many rows"), (dict(seqlen=(1 << 30) + 1), "seqlen")])
def test_prompt_descriptors(lib, mem, kw, word):
    says(lib, lib.akv_prefill_attention(ctypes.byref(prompt(mem, **kw)), mem, None, 1, None, 0, Z), word, "prefill_attention")


def test_prompt_calls(lib, mem):
    d = prompt(mem)
    says(lib, lib.akv_prefill_attention(None, mem, None, 1, None, 0, Z), "null descriptor")
    says(lib, lib.akv_prefill_attention(ctypes.byref(d), None, None, 1, None, 0, Z), "null pointer")
    says(lib, lib.akv_prefill_attention(ctypes.byref(d), mem + 2, None, 1, None, 0, Z), "aligned")
    says(lib, lib.akv_prefill_attention(ctypes.byref(prompt(mem, q=mem + 8)), mem, None, 1, None, 0, Z), "aligned")
    with_docs = prompt(mem, documents=mem)
    need = lib.akv_prefill_attention_workspace_bytes(1, 16)
    assert need >= 16 and lib.akv_prefill_attention_workspace_bytes(3, 65) >= 96
    assert lib.akv_prefill_attention_workspace_bytes(0, 16) == 0 and lib.akv_prefill_attention_workspace_bytes(1, -1) == 0
    says(lib, lib.akv_prefill_attention(ctypes.byref(with_docs), mem, None, 1, None, 0, Z), f"workspace of {need} bytes")
    says(lib, lib.akv_prefill_attention(ctypes.byref(with_docs), mem, None, 1, mem, need - 1, Z), "workspace")
    says(lib, lib.akv_attention_weights(ctypes.byref(d), None, 0, mem, 16, 16, 0, Z), "null pointer")
    says(lib, lib.akv_attention_weights(ctypes.byref(d), mem, -1, mem, 64, 16, 0, Z), "window -1")
    says(lib, lib.akv_attention_weights(ctypes.byref(d), mem, 0, mem, 64, 15, 0, Z), "rows of 15 weights")


def layer(mem, **kw):
    d = _lib.CacheLayer(*[mem + 256 * i for i in range(11)], 2, 2, 3, 192, 64, 64)
    for n, x in kw.items():
        setattr(d, n, x)
    return d


@pytest.mark.parametrize("kw,word", [(dict(k_mid_4=None), "null pointer"), (dict(seq_lens=None), "null pointer"), (dict(head_dim=32), "head_dim 32"), (dict(k_block=128), "k_block 128"),
                                     (dict(bsz=0), "bsz 0"), (dict(n_kv_heads=0), "0 KV heads"), (dict(bsz=40000), "65535"), (dict(n_max_blocks=2), "2 blocks of 64"),
                                     (dict(max_seq_len=0), "capacity of 0"), (dict(max_seq_len=(1 << 30) + 1, n_max_blocks=1 << 25), "capacity of")])
def test_cache_layers(lib, mem, kw, word):
    d = layer(mem, **kw)
    tree = (mem, mem, mem, mem, 0, None, 0.125, 0.0, mem, 4, 4, 100, mem, 1 << 30, Z)
    says(lib, lib.akv_tree_attention(ctypes.byref(d), *tree), word, "tree_attention")
    ptr = (ctypes.c_void_p * 1)(mem)
    says(lib, lib.akv_tree_commit(ctypes.byref(d), 1, ptr, ptr, mem, 4, 4, Z), word, "tree_commit")
    says(lib, lib.akv_evict(ctypes.byref(d), ctypes.byref(d), mem, 0, 0, None, 0, 0, 0, mem, 64, 0, 0, mem, 1 << 30, Z), word, "evict")
    odd = layer(mem, v_first_8=mem + 8)
    says(lib, lib.akv_tree_attention(ctypes.byref(odd), *tree), "aligned")


def test_tree_calls(lib, mem):
    d = layer(mem)

    def tree(q=mem, k=mem, v=mem, anc=mem, scale=0.125, cap=0.0, out=mem, T=4, Hq=4, bound=100, ws=mem, n=1 << 30):
        return lib.akv_tree_attention(ctypes.byref(d), q, k, v, anc, 0, None, scale, cap, out, T, Hq, bound, ws, n, Z)

    for name in ("q", "k", "v", "anc", "out"):
        says(lib, tree(**{name: None}), "null pointer")
    says(lib, tree(q=mem + 2), "aligned")
    for T in (0, 65, -3):
        says(lib, tree(T=T), f"{T} drafts")
    says(lib, tree(Hq=3), "heads 3 / 2")
    says(lib, tree(bound=193), "len_bound 193")
    says(lib, tree(bound=-1), "len_bound -1")
    says(lib, tree(scale=-1.0), "scale")
    says(lib, tree(cap=math.inf), "softcap")
    need = lib.akv_tree_attention_workspace_bytes(2, 4, 2, 64, 4, 100)
    assert need > 0 and lib.akv_tree_attention_workspace_bytes(2, 3, 2, 64, 4, 100) == 0 and lib.akv_tree_attention_workspace_bytes(2, 4, 2, 64, 65, 100) == 0
    says(lib, tree(n=need - 1), f"workspace of {need} bytes")
    says(lib, tree(ws=None), "workspace")
    ptr, two = (ctypes.c_void_p * 2)(mem, mem), (_lib.CacheLayer * 2)(layer(mem), layer(mem))
    says(lib, lib.akv_tree_commit(two, 2, ptr, ptr, mem, 4, 4, Z), "share their lengths")
    two[1] = layer(mem, head_dim=128)
    says(lib, lib.akv_tree_commit(two, 2, ptr, ptr, mem, 4, 4, Z), "another shape")
    for args, word in (((None, 1, ptr, ptr, mem, 4, 4), "null pointer"), ((two, 0, ptr, ptr, mem, 4, 4), "0 layers"), ((two, 1, ptr, ptr, None, 4, 4), "null pointer"),
                       ((two, 1, ptr, ptr, mem, 65, 4), "65 drafts"), ((two, 1, ptr, ptr, mem, 4, 0), "0 accepted"), ((two, 1, ptr, ptr, mem, 4, 65), "65 accepted"),
                       ((two, 1, (ctypes.c_void_p * 1)(None), ptr, mem, 4, 4), "null pointer")):
        says(lib, lib.akv_tree_commit(*args, Z), word)


def test_evict_calls(lib, mem):
    a, b = layer(mem), _lib.CacheLayer(*[mem + 1024 + 256 * i for i in range(11)], 2, 2, 3, 192, 64, 64)

    def evict(x=a, y=b, w=mem, wt=None, cap=0, kept=mem, keep=64, sinks=0, recent=0, ws=mem, n=1 << 30):
        return lib.akv_evict(ctypes.byref(x), ctypes.byref(y), w, 384, 192, wt, 384, 192, cap, kept, keep, sinks, recent, ws, n, Z)

    says(lib, evict(w=None), "null pointer")
    says(lib, evict(kept=None), "null pointer")
    for keep in (0, -64, 63, 100, (1 << 20) + 64):
        says(lib, evict(keep=keep), f"keep {keep}")
    says(lib, evict(sinks=-1), "sinks -1")
    says(lib, evict(recent=-1), "recent -1")
    says(lib, evict(sinks=40, recent=25), "must fit")
    says(lib, evict(sinks=2 ** 31 - 1, recent=2 ** 31 - 1), "must fit")
    mixed = _lib.CacheLayer.from_buffer_copy(b)
    mixed.k_first_8 = a.k_first_8
    says(lib, evict(y=mixed), "some of both")
    for f, x in (("bsz", 1), ("n_kv_heads", 1), ("head_dim", 128), ("k_block", 256)):
        other = _lib.CacheLayer.from_buffer_copy(b)
        setattr(other, f, x)
        says(lib, evict(y=other), "differ")
    says(lib, evict(keep=192), "cannot hold 192")
    says(lib, evict(wt=mem, cap=192), "weights move with the cache")
    says(lib, evict(wt=mem + 64, cap=100), "room for 100")
    says(lib, evict(y=a, wt=mem + 64, cap=192), "weights move with the cache")
    assert lib.akv_evict_workspace_bytes(2, 2, 64, 64, 64, 0) == 256 and lib.akv_evict_workspace_bytes(2, 2, 64, 64, 64, 1) == 256 + 2 * 2 * 64 * 64 * 2 * 2
    assert lib.akv_evict_workspace_bytes(2, 2, 64, 32, 64, 0) == 0 and lib.akv_evict_workspace_bytes(2, 2, 64, 64, 0, 0) == 0
    says(lib, evict(n=255), "workspace of 256 bytes")
    acc = (mem, 64, 64, mem, 64, mem, mem, 64, 64, 1, 4, 2, 64, 1.0)
    for i, x, word in ((0, None, "null"), (3, None, "null"), (5, None, "null"), (6, None, "null"), (9, 0, "bsz 0"), (10, 3, "heads 3 / 2"), (4, 60, "aligned rows"), (3, mem + 2, "aligned rows"),
                       (12, 65, "capacity 65"), (12, 0, "capacity 0"), (13, math.nan, "decay")):
        args = list(acc)
        args[i] = x
        says(lib, lib.akv_accumulate_weights(*args, Z), word)


def test_the_python_layer_names_what_is_wrong():
    half = torch.zeros(1, 4, 2, 64, dtype=torch.half)
    with pytest.raises(TypeError, match="q: expected a torch.Tensor"):
        cuda_module.prefill_attention(None, half, half)
    with pytest.raises(RuntimeError, match="q: expected dtype"):
        cuda_module.prefill_attention(half.float(), half, half)
    with pytest.raises(RuntimeError, match="q: expected a tensor on the GPU"):
        cuda_module.prefill_attention(half, half, half)
    with pytest.raises(RuntimeError, match="probs: expected dtype"):
        cuda_module.accumulate_weights(torch.zeros(1, 1, 8), torch.zeros(1, 1, 8), torch.zeros(1, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="three planes"):
        cuda_module.prepare_layer((half,), (half,), None, None, None, None, None)
    with pytest.raises(RuntimeError, match="at least one"):
        cuda_module.tree_commit([], half, half, None)
    for x in (-1.0, math.nan, math.inf):
        with pytest.raises(RuntimeError, match="softcap"):
            serving_ops._number("softcap", x, 0.0, False)
    with pytest.raises(RuntimeError, match="scale"):
        serving_ops._number("scale", 0.0, 0.0, True)


def test_masks_of_trees():
    f = serving_ops.tree_ancestors
    assert f([-1, 0, 0, 1, -1]).tolist() == [1, 3, 5, 11, 16]
    assert f([[-1, -1], [-1, 0]]).tolist() == [[1, 2], [1, 3]]
    chain = f(list(range(-1, 63)))
    assert chain.tolist() == serving_ops.chain_ancestors(64, "cpu").tolist() and chain[63].item() == -1
    assert serving_ops.chain_ancestors(1, "cpu").tolist() == [1]
    for bad in ([0], [-1, 1], [-2], []):
        with pytest.raises(RuntimeError):
            f(bad)
    with pytest.raises(RuntimeError, match="1 to 64"):
        f([-1] * 65)


def test_a_cache_without_weights_refuses_to_evict():
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    c = RaggedGQACache(1, 1, 100, 2, 1, 64, device="cpu")
    with pytest.raises(RuntimeError, match="track_weights"):
        c.evict(0, 64)
    c._evicted[0][0] = True
    with pytest.raises(RuntimeError, match="positions"):
        c.verify(0, None, None, None, slopes=torch.ones(2))


def test_an_output_that_overlaps_an_input_is_refused():
    pool = torch.zeros(4, 8, 16)
    serving_ops._apart("out", pool[0], pool[1], None, pool[2:])
    serving_ops._apart("out", pool[1], pool[:0])
    for out, other in ((pool[0], pool[0]), (pool[1], pool.flatten()[120:160]), (pool[:, 0], pool[2]), (pool[3], pool.expand(2, 4, 8, 16))):
        with pytest.raises(RuntimeError, match="out: overlaps an input"):
            serving_ops._apart("out", out, torch.zeros(3), other)


def test_a_prepared_layer_follows_the_tensors_of_its_cache():
    made = []
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    cache = RaggedGQACache(1, 2, 128, 2, 2, 64, device="cpu")
    class Module:                                            # noqa: E306
        @staticmethod
        def prepare_layer(*a):
            made.append(serving_ops.PreparedLayer(_lib.CacheLayer(), None, (*a[0], *a[1], *a[2:])))
            return made[-1]
    import alignedkv_amd.model.ragged_gqa_cache as module
    real, module.cuda_module = module.cuda_module, Module
    try:
        first = cache.prepared(0)
        assert cache.prepared(0) is first
        cache.seq_lens[0] = cache.seq_lens[0] + 1            # a caller's own tensor in the place of the cache's
        assert cache.prepared(0) is not first and cache.prepared(0).seq_lens is cache.seq_lens[0] and len(made) == 2
    finally:
        module.cuda_module = real


def test_a_step_that_is_taken_back_leaves_no_weights():
    from alignedkv_amd.model.decoder_harness import DecoderConfig, DeviceLengthCache
    cache = DeviceLengthCache(DecoderConfig(2, 128, 2, 2, 128, 50), 2, 128, device="cpu", track_weights=True)
    cache.inner.weights[1][0, 1, 3] = 2.0
    snap = cache.snapshot()
    cache.inner.weights[1].add_(1.0)
    cache.inner.seq_lens[0].add_(1)
    cache.restore(snap)
    assert cache.inner.weights[1].sum() == 2.0 and (cache.inner.seq_lens[0] == 0).all()
