"""4-bit attention of many sequences with few keys, each of which is one workgroup's."""
import random

import pytest
import torch

from rdlquant import attention as A
from test_gpu_kv_q4 import Pool, attend, check, ints, sequences, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,hd,heads,kvh,page,longest", [
    (64, 128, 32, 16, 64, 600), (64, 64, 16, 16, 16, 250), (48, 128, 32, 32, 32, 640), (64, 256, 16, 16, 16, 300), (40, 96, 40, 20, 64, 333)])
def test_a_step_is_as_its_halves(rq, gpu, n, hd, heads, kvh, page, longest):
    """More workgroups than run at once: the same bits as half as many sequences a call, whose lengths say that keys are few too."""
    torch.manual_seed(hd)
    r = random.Random(n)
    kv = [r.randint(1, longest) for _ in range(n)]
    kv[0], kv[1], kv[2] = longest, 1, 0
    pool = Pool(sum(-(-k // page) for k in kv) + 1, page, kvh, hd, "q4")
    tables = sequences(pool, kv, r)
    q, out = torch.randn(n, heads * hd, device="cuda"), torch.full((n, heads * hd), float("nan"), device="cuda")
    attend(pool, q, heads, [1] * n, kv, tables, hd ** -0.5, out, 1, longest)
    check(pool, q, heads, [1] * n, kv, tables, out, hd ** -0.5)
    halves = torch.full_like(out, float("nan"))
    for a, b in ((0, n // 2), (n // 2, n)):
        rs, kl = ints(list(range(b - a + 1))), ints(kv[a:b])
        A.attention_paged_dev(pool.c, q[a:b].data_ptr(), heads * hd, heads, b - a, rs.data_ptr(), kl.data_ptr(), b - a,
                              tables[a:b].data_ptr(), tables.shape[1], hd ** -0.5, halves[a:b].data_ptr(), heads * hd, 1, longest, stream())
    assert torch.equal(out, halves)
