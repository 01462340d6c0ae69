"""Bytes of a cache in 8 bits depend on their own row alone, the signs of its zeros among them."""
import pytest
import torch

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("head", [64, 20, 512])
def test_zeros_keep_their_sign(gpu, dtype, head):
    from matrix_b200 import lm

    k = torch.randn(8, 2, head, generator=torch.Generator().manual_seed(0)).to(dtype)
    k[:, :, 1], k[:, :, 2] = -0.0, 0.0
    k[:, :, 3], k[:, :, 4] = -2.0 ** -20, 2.0 ** -20  # below the type's smallest beside elements of 1
    slots = torch.arange(8).cuda()
    plain = lm.kv_cache(1, 8, 2, head, E4M3)
    lm.cache_write(plain, k.cuda(), k.cuda(), slots)
    k[3, 0, 5], k[6, 1, 7], k[6, 1, 8] = float("inf"), float("nan"), -float("inf")
    cache = lm.kv_cache(1, 8, 2, head, E4M3)
    lm.cache_write(cache, k.cuda(), k.cuda(), slots)
    for x, y in zip(cache[:2], plain[:2]):
        x, y = x.view(torch.uint8).cpu()[0], y.view(torch.uint8).cpu()[0]
        assert (x[:, :, (1, 3)] == 0x80).all() and (x[:, :, (2, 4)] == 0).all()
        assert (x[3, 0, 5] & 0x7F, x[6, 1, 7] & 0x7F, x[6, 1, 8] & 0x7F) == (0x7F, 0x7F, 0x7F)
        rows = torch.ones(8, 2, dtype=torch.bool)
        rows[3, 0] = rows[6, 1] = False
        assert torch.equal(x[rows], y[rows])
