"""GPU tests of page copies and forks at their edges (include/rdl_attention.h)."""
import pytest
import torch

import kv_q4_ref as q4
from rdlquant import attention as A
from test_gpu_kv_q4 import Pool, ints, stream

pytestmark = pytest.mark.gpu


WAYS = pytest.mark.parametrize("via", ["f16 page", "f32 page", "store", "store and norm"])


def small_rows(page, hd):
    least = 2.0 ** -24  # f16's
    x = torch.zeros(1, 1, page, hd)
    x[0, 0, 1] = -0.0
    x[0, 0, 2, ::3] = -0.0
    x[0, 0, 3], x[0, 0, 4] = least, -least
    x[0, 0, 5, 7], x[0, 0, 6, 7] = 4 * least, -4 * least   # 2^-22: the scale lies half way to f16's least number
    x[0, 0, 7, 40], x[0, 0, 8, 40] = 5 * least, -5 * least  # the least scale there is, beside a block of zeros
    x[0, 0, 9, 32:] = torch.randn(32, generator=torch.Generator().manual_seed(1)).half().float()
    x[0, 0, 10] = torch.arange(hd) * least
    return x


def put(via, x):
    """A 4-bit pool of one page whose K is x and whose V is -x."""
    page, hd = x.shape[2:]
    dst = Pool(1, page, 1, hd, "q4")
    if "page" in via:
        src = Pool(1, page, 1, hd, via[:3])
        src.k.copy_(x), src.v.copy_(-x)
        z = ints([0])
        A.copy_pages_dev([src.c], [dst.c], z.data_ptr(), z.data_ptr(), 1, stream())
    else:
        k, v, slots = x[0, 0].cuda(), -x[0, 0].cuda(), ints(list(range(page)))
        args = (dst.c, page, 0, 0, 0, 0, 0, k.data_ptr(), hd, v.data_ptr(), hd)
        if via == "store":
            A.store_dev(*args, 0, slots.data_ptr(), 0, 0, 0, stream())
        else:
            A.store_norm_dev(*args, 0, 0, 0.0, 0, slots.data_ptr(), 0, 0, 0, stream())
    return dst


@WAYS
def test_codes_of_blocks_whose_scale_is_zero(rq, gpu, via):
    """8 whichever way the values came: zeros of either sign, magnitudes up to 2^-22; and the blocks next above."""
    x = small_rows(16, 64)
    dst = put(via, x)
    for runs, y in ((dst.k, x), (dst.v, -x)):
        assert torch.equal(runs.codes.cpu(), q4.pack(q4.quantize(y)[1]))
        assert (q4.unpack(runs.codes.cpu())[0, 0, :7] == 8).all()
    assert (dst.both()[:, 0, 0, :7] == 0).all()


@WAYS
def test_scales_of_zeros(rq, gpu, via):
    """Zeros of either sign, in any order, are the same bytes: a zero counts as positive."""
    x = small_rows(16, 64)
    dst = put(via, x)
    for runs, y in ((dst.k, x), (dst.v, -x)):
        assert torch.equal(runs.scales.cpu().view(torch.int16), q4.quantize(y)[0].view(torch.int16))
        assert (runs.scales.cpu().view(torch.int16)[0, 0, :3] == -0x8000).all()
