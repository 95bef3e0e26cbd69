"""Views whose dimensions of one entry carry any stride (a slice of a padded buffer): torch counts them as contiguous, the kernels take them."""
import pytest
import torch

from alignedkv_amd.extension import serving_ops
from alignedkv_amd.extension.KV_cache_cpp_extention import cuda_module

VIEWS = [((1, 3, 4, 64), (3 * 256 + 4, 256, 64, 1)), ((1, 1, 4, 64), (3, 7, 64, 1)), ((1, 1, 1, 64), (1, 1, 1, 1)), ((2, 3, 1, 64), (200, 64, 4, 1)),
         ((2, 1, 2, 64), (128, 1 << 25, 64, 1)), ((2, 1, 2, 64), (136, 5, 72, 1))]


@pytest.mark.parametrize("shape,stride", VIEWS)
@pytest.mark.parametrize("start", [0, 1])
def test_strides_of_single_entries_do_not_matter(shape, stride, start):
    used = sum((n - 1) * s for n, s in zip(shape, stride)) + 64
    base = torch.arange(used + 1, dtype=torch.int16).view(torch.half)
    t = base.as_strided(shape, stride, start)
    got, s = serving_ops._strided("q", t)
    assert len(s) == 3 or len(s) == 4
    assert all(x >= 0 and x % 8 == 0 for x in s[:3]) and s[1] < 1 << 24 and got.data_ptr() % 16 == 0
    seen = torch.empty(0, dtype=torch.half).set_(got.untyped_storage(), got.storage_offset(), shape, (*s[:3], 1))
    assert torch.equal(seen.view(torch.int16), t.contiguous().view(torch.int16))
    if start == 0 and all(x % 8 == 0 for n, x in zip(shape, stride) if n > 1) and base.data_ptr() % 16 == 0:
        assert got.data_ptr() == t.data_ptr(), "read in place"


@pytest.mark.gpu
def test_a_slice_of_a_padded_buffer():
    g = torch.Generator(device="cuda").manual_seed(0)
    S, H, D = 70, 2, 64
    pads = [torch.randn(2 * (S * H * D + 4), generator=g, device="cuda").half().as_strided((2, S, H, D), (S * H * D + 4, H * D, D, 1))[:1] for _ in range(3)]
    dense = [p.clone(memory_format=torch.contiguous_format).reshape(-1).view(1, S, H, D) for p in pads]
    want, lse = cuda_module.prefill_attention(*dense, return_lse=True)
    assert torch.equal(cuda_module.prefill_attention(*pads), want)
    assert torch.equal(cuda_module.attention_weights(pads[0], pads[1], lse), cuda_module.attention_weights(dense[0], dense[1], lse))
