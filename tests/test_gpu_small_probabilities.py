"""Rows in which one token takes nearly all the weight and its value is zero: the output is the sum of many small terms.

A probability is rounded to fp16 for the product with the values.  Relative to the row's largest it is then off by 2^-11 of itself, or, where fp16
is subnormal, by 2^-25 of fp16's scale.  The kernels scale a row so that its largest probability is at least 2^7 there, so that a term is off by
at most 2^-32 of the largest: the bounds of serving_forms.rows_form with N 2^-32 max|v| in the place of N 2^-25 max|v|."""
import pytest
import torch

from tests.serving_forms import cached_tokens, check_rows, rows_form

pytestmark = pytest.mark.gpu

NATS = [10.0, 15.0, 16.0, 17.0]


def tightened(tol, v):
    return tol - v.shape[0] * (2.0 ** -25 - 2.0 ** -32) * v.double().abs().max().item()


def sink_inputs(N, D, nats, g):
    """Keys and values [N, D], queries: token 0 scores about `nats` above the others, whose scores spread a little; its value is zero."""
    k = torch.randn(N, D, generator=g, device="cuda") * 0.125
    v = torch.rand(N, D, generator=g, device="cuda") * 0.5 + 0.75
    k[:, 0] = 0.0
    k[0] = 0.0
    k[0, 0], v[0] = nats * D ** 0.5 / 4.0, 0.0
    return k.half(), v.half()


def queries(R, H, D, g):
    q = torch.randn(R, H, D, generator=g, device="cuda")
    q[..., 0] = 4.0
    return q.half()


@pytest.mark.parametrize("bound", [None, 0])            # None: the sink and the others in splits of their own; 0: one split for all
@pytest.mark.parametrize("nats", NATS)
@pytest.mark.parametrize("T,Hq,D,kb", [(1, 1, 128, 64), (4, 4, 128, 256), (16, 4, 128, 64), (64, 4, 128, 256), (9, 2, 64, 64), (5, 1, 256, 64)])
def test_tree_over_a_cache_with_a_sink(T, Hq, D, kb, nats, bound):
    from alignedkv_amd.model.ragged_gqa_cache import RaggedGQACache
    N = 16384
    g = torch.Generator(device="cuda").manual_seed(int(nats))
    cache = RaggedGQACache(1, 1, N + 64, Hq, 1, D, k_block=kb)
    k, v = sink_inputs(N, D, nats, g)
    cache.prefill(0, 0, k[None, :, None], v[None, :, None])
    q = queries(T, Hq, D, g)
    dk, dv = torch.zeros(T, D, device="cuda").half(), torch.ones(T, D, device="cuda").half()
    anc = torch.ones(T, dtype=torch.int64, device="cuda") << torch.arange(T, device="cuda")
    out = cache.verify(0, q[None], dk[None, :, None], dv[None, :, None], anc, bound=bound)
    ck, cv = cached_tokens(cache, 0, 0, 0)
    ck, cv = torch.cat([ck, dk]), torch.cat([cv, dv])
    see = torch.cat([torch.ones(T, N, dtype=torch.bool, device="cuda"), torch.eye(T, dtype=torch.bool, device="cuda")], 1)
    for h in range(Hq):
        o, _, _, tol, _, _ = rows_form(q[:, h], ck, cv, see, D ** -0.5)
        check_rows(out[0, :, h], o, tightened(tol, cv), f"head {h}")


@pytest.mark.parametrize("nats", NATS)
@pytest.mark.parametrize("Hq,D", [(1, 64), (2, 128), (1, 256)])
def test_prompt_with_a_sink(Hq, D, nats):
    from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module
    S = 4000
    g = torch.Generator(device="cuda").manual_seed(int(nats) + D)
    k, v = sink_inputs(S, D, nats, g)
    q = queries(S, Hq, D, g)
    out, lse = cuda_module.prefill_attention(q[None], k[None, :, None], v[None, :, None], return_lse=True)
    rows = torch.cat([torch.arange(0, 200, 13), torch.arange(3500, S, 37)]).cuda()
    see = torch.arange(S, device="cuda")[None] <= rows[:, None]
    for h in range(Hq):
        o, want, _, tol, tol_lse, _ = rows_form(q[rows, h], k, v, see, D ** -0.5)
        check_rows(out[0, rows, h], o, tightened(tol, v), f"head {h}")
        assert ((lse[0, h, rows].double() - want).abs() <= tol_lse).all()


@pytest.mark.parametrize("parts", ["1", "2"])
def test_prompt_with_a_sink_in_both_forms(monkeypatch, parts):
    from alignedkv_amd import load_library
    lib = load_library()
    monkeypatch.setenv("AKV_TUNE_PROMPT_PARTS", parts)
    lib.akv_reload_tuning()
    try:
        test_prompt_with_a_sink(2, 128, 17.0)
    finally:
        monkeypatch.delenv("AKV_TUNE_PROMPT_PARTS")
        lib.akv_reload_tuning()
