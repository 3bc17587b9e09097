"""GPU tests of page copies and forks at their edges (include/rdl_attention.h)."""
import random

import pytest
import torch

import kv_q4_ref as q4
from rdlquant import attention as A
from test_gpu_kv_q4 import Pool, ints, plain_fork, run_fork, stream

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


# ---- forks ----------------------------------------------------------------------------------------------


def chained(n, page, seed):
    """n pairs of which every fourth child is the parent of later and of earlier pairs."""
    r = random.Random(seed)
    width, roots = 9, 1 + n // 5
    lens = [r.randrange(width * page + 1) for _ in range(roots + n)]
    tables = [[r.randrange(10000) for _ in range(width)] for _ in lens]
    children = list(range(roots, roots + n))
    r.shuffle(children)
    parents = [children[r.randrange(n)] if i % 4 == 3 else r.randrange(roots) for i in range(n)]
    parents = [p if p != c else 0 for p, c in zip(parents, children)]
    return tables, lens, page, parents, children, r.sample(range(20000, 60000), n + 7)


@pytest.mark.parametrize("n,page", [(4, 16), (63, 32), (64, 16), (65, 16), (150, 16), (700, 64), (2600, 32)])
def test_children_that_are_parents_spoil_their_own_copies_alone(rq, gpu, n, page):
    args = chained(n, page, n)
    parents, children = args[3:5]
    want, got = plain_fork(*args), run_fork(*args)
    assert got[3] == want[3] and got[4] == want[4]  # pages and summary
    own = {c for p, c in zip(parents, children) if p in set(children)}
    for s in range(len(args[1])):
        if s not in own:
            assert got[0][s] == want[0][s] and got[1][s] == want[1][s]
    assert all(g == w for g, w, c in zip(got[2], want[2], children) if c not in own)


def test_forks_on_streams_and_in_graphs(rq, gpu):
    r = random.Random(3)
    n, page, width = 60, 16, 7
    lens = [r.randrange(width * page + 1) for _ in range(20)] + [0] * n
    tables = [[r.randrange(10000) for _ in range(width)] for _ in lens]
    parents, children, free = [r.randrange(20) for _ in range(n)], list(range(20, 20 + n)), r.sample(range(20000, 60000), n)
    want = plain_fork(tables, lens, page, parents, children, free)
    f, c, fr = ints(parents), ints(children), ints(free)

    class Side:
        def __init__(self):
            self.stream = torch.cuda.Stream()
            self.t, self.k = ints(tables), ints(lens)
            self.out = [torch.zeros(s, dtype=torch.int32, device="cuda") for s in (n, n, 2)]

        def call(self):
            A.fork_dev(self.t.data_ptr(), width, self.k.data_ptr(), len(lens), page, f.data_ptr(), c.data_ptr(), n, fr.data_ptr(), n,
                       *(o.data_ptr() for o in self.out), self.stream.cuda_stream)

        def restore(self):
            self.t.copy_(ints(tables)), self.k.copy_(ints(lens))
            for o in self.out:
                o.fill_(-5)

        def check(self):
            assert (self.t.tolist(), self.k.tolist(), *(o.tolist() for o in self.out)) == want

    sides = [Side(), Side()]
    torch.cuda.synchronize()
    for _ in range(20):
        for s in sides:
            s.call()
    torch.cuda.synchronize()
    for s in sides:
        s.check()
    graphs = []
    for s in sides:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(s.stream), torch.cuda.graph(g, stream=s.stream):
            s.call()
        graphs.append(g)
    for _ in range(4):
        for s in sides:
            s.restore()
        torch.cuda.synchronize()
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for s in sides:
            s.check()


@pytest.mark.parametrize("n", [1, 3, 17, 40, 64, 65, 100])
@pytest.mark.parametrize("short", [0, 5])
def test_forks_of_long_rows(rq, gpu, n, short):
    """Rows of many pages, free lists that end within the pairs, parents and children that are none."""
    r = random.Random(n)
    width, page, roots = 1100, 16, 5
    lens = [width * page, width * page - 1, 64 * page + 3, 7, 20 * width * page] + [0] * n
    tables = [[r.randrange(10000) for _ in range(width)] for _ in lens]
    parents, children = [r.randrange(roots) for _ in range(n)], list(range(roots, roots + n))
    if n > 10:
        parents[4], children[7], parents[9] = -1, roots + n, children[9]
    want = sum(0 <= p < roots + n and 0 <= c < roots + n and p != c and min(lens[p], width * page) % page != 0
               for p, c in zip(parents, children))
    free = r.sample(range(20000, 60000), max(0, want - short))
    args = (tables, lens, page, parents, children, free)
    assert run_fork(*args) == plain_fork(*args)
