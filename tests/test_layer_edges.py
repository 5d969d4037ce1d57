"""Host checks of the operators around the attention, without a GPU: where padding and extreme arguments meet the contract."""
import pytest
import torch

import mlc_decode_amd as M


@pytest.mark.parametrize("k", [32, 96, 128, 160])
def test_largest_scales_are_of_the_weights_alone(k):
    """``top`` is each output's largest scale, not that of the inputs past the end."""
    g = torch.Generator().manual_seed(k)
    n = 37
    scale = torch.randint(1, 100, (n, k // 32), generator=g).to(torch.uint8)
    scale[3, 0], scale[5], scale[6] = 255, 255, 200
    p = M.pack_w_fp4(torch.zeros(n, k // 2, dtype=torch.uint8), scale)
    want = torch.where(scale == 255, 1, scale).amax(1)
    assert p.top.shape == (48,) and p.top.dtype == torch.uint8 and torch.equal(p.top[:n], want)
