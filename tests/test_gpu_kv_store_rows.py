"""Cache writes of many rows, some of which are left out, and page copies of heads and pages of all sizes."""
import pytest
import torch

from rdlquant import attention as A
from test_gpu_kv_q4 import Pool, ints, stream

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,hd", [(kv, hd) for hd in (8, 24, 32, 64, 96, 128, 136, 256) for kv in ("f16", "f32", "q4")
                                   if kv != "q4" or hd % 32 == 0])
@pytest.mark.parametrize("norms", ["qk", ""])
def test_rows_left_out_of_a_large_step(rq, gpu, kv, hd, norms):
    """515 rows, which workgroups take by two, against calls of fewer than 512, by one: the same bits, and nothing of
    the rows whose slot or position is outside, at even and odd places and at the end.  The tables stand between rows
    of NaN, which such a row would bring."""
    torch.manual_seed(hd)
    rows, heads, kvh, page, npos = 515, 3, 2, 64, 70
    width = (heads + 2 * kvh) * hd
    x = torch.randn(rows, width, device="cuda")
    pos = torch.randint(0, npos, (rows,), device="cuda").int()
    slots = torch.randperm(10 * page, device="cuda")[:rows].int()
    bad = {0: (-1, None), 1: (None, -1), 2: (None, npos), 7: (10 * page, None), 8: (None, npos + 3), 100: (None, -4), 101: (-5, None),
           256: (None, npos), 257: (None, npos), 512: (None, -1), 513: (None, npos), 514: (None, npos + 1)}
    for r, (s, p) in bad.items():
        if s is not None:
            slots[r] = s
        if p is not None:
            pos[r] = p
    tables = torch.full((2, npos + 16, hd // 2), float("nan"), device="cuda")
    ang = torch.rand(npos, hd // 2, device="cuda") * 6
    tables[0, 8:8 + npos], tables[1, 8:8 + npos] = ang.cos(), ang.sin()
    cos, sin = (t[8:].data_ptr() for t in tables)
    g = 1 + 0.3 * torch.randn(2, hd, device="cuda")
    got = []
    for cuts in ([0, rows], [0, 300, rows]):
        pool = Pool(10, page, kvh, hd, kv, fill=7.0)
        out = torch.full((rows, heads * hd), 5.0, device="cuda")
        for a, b in zip(cuts, cuts[1:]):
            at = [x[a:, i * hd:].data_ptr() for i in (0, heads, heads + kvh)]
            A.store_norm_dev(pool.c, b - a, at[0], width, out[a:].data_ptr(), heads * hd, heads, at[1], width, at[2], width,
                             g[0].data_ptr() if norms else 0, g[1].data_ptr() if norms else 0, 1e-6, pos[a:].data_ptr(),
                             slots[a:].data_ptr(), cos, sin, npos, stream())
        got.append([out, *pool.mem])
    assert all(torch.equal(a, b) for a, b in zip(*got))
    left = torch.zeros(rows, dtype=torch.bool, device="cuda")
    left[list(bad)] = True
    assert (got[0][0][left] == 5.0).all() and torch.isfinite(got[0][0]).all()
    if kv != "q4":  # as many positions are written as rows are in, none is NaN
        written = (got[0][1] != 7.0).any(-1).sum()
        assert written == (rows - len(bad)) * kvh and torch.isfinite(got[0][1]).all() and torch.isfinite(got[0][2]).all()


@pytest.mark.parametrize("a,b", [("f16", "f32"), ("f32", "f16"), ("f16", "f16"), ("f32", "f32")])
@pytest.mark.parametrize("hd,page,kvh", [(8, 16, 5), (24, 32, 3), (40, 16, 1), (80, 64, 2), (136, 16, 2), (256, 1024, 1)])
def test_copies_of_heads_and_pages_of_all_sizes(rq, gpu, a, b, hd, page, kvh):
    torch.manual_seed(hd)
    src, dst = Pool(4, page, kvh, hd, a, "padded"), Pool(3, page, kvh, hd, b, "positions")
    for t in (src.k, src.v):
        t.copy_(torch.randn(4, kvh, page, hd, device="cuda") * torch.logspace(-4, 4, page, device="cuda")[:, None])
    f, t = ints([3, 0]), ints([0, 2])
    A.copy_pages_dev([src.c], [dst.c], f.data_ptr(), t.data_ptr(), 2, stream())
    for x, y in ((src.k, dst.k), (src.v, dst.v)):
        assert torch.equal(y[0], x[3].to(y.dtype)) and torch.equal(y[2], x[0].to(y.dtype)) and y[1].isnan().all()
