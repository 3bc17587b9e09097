"""GPU tests of the several-sequence operators (include/rdl_attention.h)
against plain 64-bit implementations (tests/attention_ref.py)."""
import math
import random
import threading

import pytest
import torch

import attention_ref as ref
from rdlquant import attention as A

pytestmark = pytest.mark.gpu
KV = {"f16": (torch.float16, A.DTYPE_F16), "f32": (torch.float32, A.DTYPE_F32)}


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


class Pool:
    """A pool in one of the orders, its memory filled with `fill`; k and v are [pages, kv heads, positions, hd] views."""

    def __init__(self, pages, page, kvh, hd, kv="f16", layout="heads", fill=float("nan")):
        dt, code = KV[kv]
        shape = {"heads": (pages, kvh, page, hd), "positions": (pages, page, kvh, hd),
                 "padded": (pages, kvh, page + 1, hd + 8)}[layout]
        self.mem = [torch.full(shape, fill, dtype=dt, device="cuda") for _ in range(2)]
        view = {"heads": lambda t: t, "positions": lambda t: t.transpose(1, 2), "padded": lambda t: t[:, :, :page, :hd]}
        self.k, self.v = (view[layout](t) for t in self.mem)
        s = self.k.stride()
        self.page, self.dtype = page, dt
        self.c = A.KvPool(self.k.data_ptr(), self.v.data_ptr(), code, pages, page, kvh, hd, s[0], s[1], s[2])

    def put(self, table, k, v):
        """Positions 0 .. len - 1 of a sequence."""
        n = k.shape[0]
        pos = torch.arange(n, device="cuda")
        ids = table[pos // self.page].long()
        self.k[ids, :, pos % self.page] = k.to(self.dtype)
        self.v[ids, :, pos % self.page] = v.to(self.dtype)


# ---- plan --------------------------------------------------------------------------------


def run_plan(cached, new, free, page, tables, m, extra=0):
    n = len(cached)
    t = ints(tables) if n else torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    out = [torch.full((k,), -77, dtype=torch.int32, device="cuda") for k in (n + 1 + 4, n + 4, m + 4, m + 4, m + 4, 8)]
    cd, nd, fr = ints(cached or [0]), ints(new or [0]), ints(free or [0])
    p = [o.data_ptr() for o in out]
    A.plan_dev(cd.data_ptr(), nd.data_ptr(), n, fr.data_ptr(), len(free), page, t.data_ptr(), t.shape[1], p[0], p[1], m,
               p[2], p[3], p[4], p[5], stream())
    got = [o.tolist() for o in out]
    for g, k in zip(got, (n + 1, n, m, m, m, 4)):  # nothing past the end of any output
        assert set(g[k:]) == {-77}
    return (t.tolist() if n else []), [g[:k] for g, k in zip(got, (n + 1, n, m, m, m, 4))]


def check_plan(cached, new, free, page, tables, m):
    want = ref.plan(cached, new, free, page, tables, m)
    table, got = run_plan(cached, new, free, page, tables, m)
    assert table == want[0]
    for g, w, name in zip(got, want[1:], ("row_start", "kv_len", "row_seq", "positions", "slots", "summary")):
        assert g == w, name


@pytest.mark.parametrize("n_seq,page,pad", [(1, 64, 0), (3, 16, 1), (17, 32, 0), (64, 128, 1000), (1024, 64, 7),
                                            (1025, 16, 0), (3000, 256, 5)])
def test_plan(rq, gpu, n_seq, page, pad):
    r = random.Random(n_seq)
    cached = [r.choice([0, 1, page - 1, page, page + 1, r.randrange(6 * page)]) for _ in range(n_seq)]
    new = [r.choice([0, 1, 1, 1, r.randrange(3 * page), page]) for _ in range(n_seq)]
    width = 9
    total = sum(-(-(c + n) // page) for c, n in zip(cached, new))
    pages = list(range(total + 3))
    r.shuffle(pages)
    tables = []
    for c in cached:
        had = -(-c // page)
        tables.append([pages.pop() for _ in range(had)] + [-5] * (width - had))
    check_plan(cached, new, pages, page, tables, sum(new) + pad)


def test_plan_no_sequences_and_no_rows(rq, gpu):
    check_plan([], [], [], 64, [], 5)
    check_plan([], [], [3], 64, [], 0)
    check_plan([64, 10], [0, 0], [7], 64, [[3, -1], [4, -1]], 0)
    check_plan([64, 10], [0, 0], [7], 64, [[3, -1], [4, -1]], 3)


@pytest.mark.parametrize("cached,new,free,width,m,flags", [
    ([10, 100], [70, 60], [9], 4, 130, 4),             # one free page for two
    ([10, 100], [200, 1], [9, 8, 7, 6], 3, 201, 2),    # the first sequence's table is too narrow
    ([10, 100], [7, 9], [9, 8], 4, 12, 8),             # rows past m are cut
    ([-3, 100], [7, -9], [9, 8], 4, 7, 1),             # negative lengths count as 0
    ([2**31 - 5, 3], [100, 2], [9, 8], 4, 20, 1 | 2),   # past 31 bits
    ([300, 3], [1, 1], [9], 4, 2, 2),                  # more cached than the table can name
])
def test_plan_flags(rq, gpu, cached, new, free, width, m, flags):
    tables = [[20 + i if i * 64 < c else -1 for i in range(width)] for c in cached]
    want = ref.plan(cached, new, free, 64, tables, m)
    assert want[-1][2] == flags
    check_plan(cached, new, free, 64, tables, m)


# ---- store -------------------------------------------------------------------------------


@pytest.mark.parametrize("hd", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("kv,layout", [("f16", "heads"), ("f32", "positions"), ("f16", "padded"), ("f32", "padded")])
@pytest.mark.parametrize("rope,in_place", [(True, False), (True, True), (False, False)])
def test_store(rq, gpu, hd, kv, layout, rope, in_place):
    torch.manual_seed(hd)
    rows, heads, kvh, page, npos = 37, 6, 2, 32, 90
    pool = Pool(5, page, kvh, hd, kv, layout)
    before = [t.clone() for t in pool.mem]
    qkv = torch.randn(rows, (heads + 2 * kvh) * hd + 4, device="cuda")  # strided rows
    q, k, v = (qkv[:, a * hd:b * hd] for a, b in ((0, heads), (heads, heads + kvh), (heads + kvh, heads + 2 * kvh)))
    q0 = q.clone()
    out = q if in_place else torch.full((rows, heads * hd), float("nan"), device="cuda")
    kept = out.clone()
    cap = 5 * page
    slots = torch.randperm(cap)[:rows].int()
    pos = torch.randint(0, npos, (rows,)).int()
    slots[3], slots[5], slots[7] = -1, cap, -(2**31)   # rows that are left out
    skipped = {3, 5, 7}
    if rope:
        pos[9], pos[11] = -1, npos
        skipped |= {9, 11}
    ang = torch.rand(npos, hd // 2, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    ps, sl = pos.cuda(), slots.cuda()
    A.store_dev(pool.c, rows, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), heads, k.data_ptr(),
                k.stride(0), v.data_ptr(), v.stride(0), ps.data_ptr(), sl.data_ptr(), cos.data_ptr() if rope else 0,
                sin.data_ptr() if rope else 0, npos if rope else 0, stream())
    live = [r for r in range(rows) if r not in skipped]
    at = pos[live].long().cuda()
    c, s = (cos[at], sin[at]) if rope else (torch.ones(len(live), hd // 2, device="cuda"),
                                            torch.zeros(len(live), hd // 2, device="cuda"))
    want, tol = ref.rope(q0[live].view(-1, heads, hd), c, s)
    assert ((out[live].view(-1, heads, hd).double() - want).abs() <= tol).all()
    for r in skipped:
        assert torch.equal(out[r].isnan(), kept[r].isnan()) and (in_place is False or torch.equal(out[r], kept[r]))
    wk, tk = ref.rope(k[live].reshape(-1, kvh, hd), c, s)
    wv = v[live].reshape(-1, kvh, hd).double()
    sel = slots[live].long().cuda()
    gk, gv = pool.k[sel // page, :, sel % page].double(), pool.v[sel // page, :, sel % page].double()
    half = 2.0**-11 if kv == "f16" else 0.0  # half a step of f16, and of its smallest numbers
    tiny = 2.0**-25 if kv == "f16" else 0.0
    assert ((gk - wk).abs() <= tk + (wk.abs() + tk) * half + tiny).all()
    assert torch.equal(gv, wv.to(pool.dtype).double())
    # every other element of the pool as it was
    mark = torch.zeros(5, kvh, page, hd, dtype=torch.bool, device="cuda")
    mark[sel // page, :, sel % page] = True
    fresh = Pool(5, page, kvh, hd, kv, layout)
    fresh.k.copy_(torch.where(mark, pool.k, fresh.k))
    fresh.v.copy_(torch.where(mark, pool.v, fresh.v))
    for got, was in zip(pool.mem, fresh.mem):
        assert torch.equal(got.isnan(), was.isnan())
    assert before[0].isnan().all()


def test_store_without_q_and_many_rows(rq, gpu):
    torch.manual_seed(3)
    rows, kvh, hd, page = 70000, 1, 8, 1024  # more rows than one grid axis holds
    pool = Pool(rows // page + 1, page, kvh, hd, "f16", fill=0.0)
    k, v = torch.randn(rows, hd, device="cuda"), torch.randn(rows, hd, device="cuda")
    sl = torch.randperm(pool.k.shape[0] * page, device="cuda")[:rows].int()
    A.store_dev(pool.c, rows, None, 0, None, 0, 0, k.data_ptr(), hd, v.data_ptr(), hd, None, sl.data_ptr(), 0, 0, 0,
                stream())
    at = sl.long()
    assert torch.equal(pool.k[at // page, 0, at % page], k.half())
    assert torch.equal(pool.v[at // page, 0, at % page], v.half())


# ---- attention over the cache ----------------------------------------------------------------


def close(got, want, bound):
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    err = (got - want)[fine].abs()
    assert (err <= bound[fine]).all(), float((err - bound[fine]).max())
    # f32-like as a whole: scores of up to about 2^4 carry 2^-24 2^4 a step, a dozen of which add up at random
    norm = want[fine].norm()
    if norm > 0:
        assert float(err.norm() / norm) <= 2.0**-18, float(err.norm() / norm)


class Batch:
    """Sequences of (cached, new) positions in a shuffled pool; unused places hold NaN."""

    def __init__(self, lens, heads, kvh, hd, kv="f16", page=64, layout="heads", seed=0, spread=1.0, pad=0, width=0):
        torch.manual_seed(seed)
        self.lens, self.heads, self.kvh, self.hd, self.page = lens, heads, kvh, hd, page
        need = [-(-(c + n) // page) for c, n in lens]
        self.width = max(max(need, default=1), 1) + width
        self.pool = Pool(sum(need) + 3, page, kvh, hd, kv, layout)
        order = torch.randperm(sum(need) + 3, device="cuda").int()
        self.table = torch.full((len(lens), self.width), -1, dtype=torch.int32, device="cuda")
        self.kv, at = [], 0
        for b, (c, n) in enumerate(lens):
            self.table[b, :need[b]] = order[at:at + need[b]]
            at += need[b]
            k, v = (torch.randn(c + n, kvh, hd, device="cuda").to(KV[kv][0]) for _ in range(2))
            self.pool.put(self.table[b], k, v)
            self.kv.append((k, v))
        starts = [0]
        for _, n in lens:
            starts.append(starts[-1] + n)
        self.rows, self.pad = starts[-1], pad
        self.row_start, self.kv_len = ints(starts), ints([c + n for c, n in lens])
        self.q = torch.randn(self.rows + pad, heads, hd, device="cuda") * spread
        self.scale = 1 / math.sqrt(hd)

    def run(self, max_rows=None, max_kv=None, q=None, out=None, s=None):
        q = self.q if q is None else q
        out = torch.full((self.rows + self.pad, self.heads, self.hd), -7.0, device="cuda") if out is None else out
        mr = max((n for _, n in self.lens), default=0) if max_rows is None else max_rows
        mk = max((c + n for c, n in self.lens), default=0) if max_kv is None else max_kv
        A.attention_paged_dev(self.pool.c, q.data_ptr(), q.stride(0), self.heads, self.rows + self.pad,
                              self.row_start.data_ptr(), self.kv_len.data_ptr(), len(self.lens),
                              self.table.data_ptr(), self.width, self.scale, out.data_ptr(), out.stride(0), mr, mk,
                              stream() if s is None else s)
        return out

    def want(self):
        outs = [ref.attention(self.q[int(a):int(a) + n], k, v, c, self.scale)
                for a, (c, n), (k, v) in zip(self.row_start.tolist(), self.lens, self.kv)]
        return torch.cat([o for o, _ in outs]), torch.cat([b for _, b in outs])

    def check(self, **kw):
        out = self.run(**kw)
        close(out[:self.rows], *self.want())
        assert (out[self.rows:] == -7.0).all()  # rows behind the last sequence


SHAPES = [(4, 1, 64), (8, 8, 128), (8, 2, 128), (3, 1, 80), (14, 2, 96), (6, 2, 256), (2, 2, 8), (40, 1, 40),
          (32, 8, 128), (20, 4, 200)]


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
def test_single_tokens(rq, gpu, heads, kvh, hd, kv):
    Batch([(0, 1), (1, 1), (62, 1), (63, 1), (64, 1), (127, 1), (700, 1), (31, 1)], heads, kvh, hd, kv, pad=2).check()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
def test_chunks(rq, gpu, heads, kvh, hd, kv):
    Batch([(0, 5), (0, 0), (130, 33), (1, 128), (511, 65), (64, 64), (300, 1), (3, 0), (0, 257)], heads, kvh, hd, kv,
          pad=3).check()


@pytest.mark.parametrize("page,layout,kv", [(16, "heads", "f16"), (32, "positions", "f16"), (128, "padded", "f16"),
                                            (1024, "heads", "f16"), (256, "positions", "f32"), (16, "padded", "f32")])
def test_pages_and_layouts(rq, gpu, page, layout, kv):
    Batch([(0, 17), (1500, 1), (2 * page - 1, 1), (2 * page, 3), (page - 1, 70)], 8, 2, 64, kv, page, layout).check()


@pytest.mark.parametrize("lens", [[(20000, 1)], [(5000, 1)] * 3, [(9000, 40)], [(3000, 300)], [(4100, 2), (17, 900)],
                                  [(12345, 8), (0, 1), (1, 1)]])
@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_long_caches(rq, gpu, lens, kv):
    Batch(lens, 8, 2, 128, kv).check()


@pytest.mark.parametrize("max_rows,max_kv", [(0, 0), (1, 1), (10000, 100000), (1, 100000), (100, 64)])
def test_hints_do_not_decide(rq, gpu, max_rows, max_kv):
    b = Batch([(900, 1), (20, 200), (2500, 7), (0, 1), (1999, 65)], 8, 2, 64, pad=1)
    b.check(max_rows=max_rows, max_kv=max_kv)


def test_large_and_small_scores(rq, gpu):
    # weights from about 1 to nothing; rows and keys of very different sizes
    for kv in ("f16", "f32"):
        b = Batch([(300, 40), (100, 1)], 4, 2, 64, kv, spread=6.0)
        b.q[::3] *= 1e-20
        b.q[1::7] *= 1e-3
        b.check()


def test_values_of_very_different_sizes(rq, gpu):
    # f32 keys and values from 1e-12 to 1e12 across positions: each row's own precision holds
    b = Batch([(500, 30), (40, 1)], 4, 2, 64, "f32")
    for (k, v), t in zip(b.kv, b.table):
        n = k.shape[0]
        v *= torch.logspace(-12, 12, n, device="cuda")[torch.randperm(n, device="cuda")][:, None, None]
        k *= torch.logspace(-12, 0, n, device="cuda")[torch.randperm(n, device="cuda")][:, None, None]
        b.pool.put(t, k, v)
    b.check()


def test_rows_that_see_nothing_are_zero(rq, gpu):
    b = Batch([(0, 6), (50, 2), (0, 70)], 4, 2, 64)
    b.kv_len = ints([2, 0, 66])  # fewer keys than rows: the first rows are before key 0
    out = b.run()
    assert (out[:4] == 0).all() and (out[6:8] == 0).all() and (out[8:12] == 0).all()
    k, v = b.kv[0]
    close(out[4:6], *ref.attention(b.q[4:6], k[:2], v[:2], 0, b.scale))
    k, v = b.kv[2]
    close(out[12:78], *ref.attention(b.q[12:78], k[:66], v[:66], 0, b.scale))
    b.kv_len = ints([-5, -(2**31), 0])
    assert (b.run() == 0).all()


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_masked_has_no_effect(rq, gpu, kv, bad):
    # keys and values behind a row's own place are NaN or infinite: rows before them stay exact
    b = Batch([(40, 30), (0, 90), (500, 1)], 4, 2, 64, kv)
    clean = b.want()
    hit = []
    for i, (a, (c, n), (k, v)) in enumerate(zip(b.row_start.tolist(), b.lens, b.kv)):
        if n < 2:
            continue
        j = c + n // 2
        k[j, :, 3] = bad
        v[j, :, 5] = bad
        v[j + 1] = bad
        b.pool.put(b.table[i], k, v)
        hit.append((a, a + n // 2, a + n))
    out = b.run()
    for lo, mid, hi in hit:
        close(out[lo:mid], clean[0][lo:mid], clean[1][lo:mid])
        if not math.isinf(bad):
            assert out[mid:hi].isnan().all()
    close(out[-1:], clean[0][-1:], clean[1][-1:])


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_values_that_are_not_finite_reach_the_rows_that_see_them(rq, gpu, kv):
    b = Batch([(70, 60), (300, 1), (0, 200)], 4, 2, 64, kv)
    for i, (k, v) in enumerate(b.kv):
        n = k.shape[0]
        v[n // 2, 0, 5] = float("inf")
        v[n - 1, 1, 7] = -float("inf")
        v[n - 1, 0, 9] = float("nan")
        b.pool.put(b.table[i], k, v)
    out = b.run()[:b.rows].double()
    want, bound = b.want()
    # where nothing infinite or NaN is summed the row is exact; where it is, the row is not finite
    fine = torch.isfinite(want)
    before = torch.zeros(b.rows, dtype=torch.bool, device="cuda")
    for a, (c, n), (k, _) in zip(b.row_start.tolist(), b.lens, b.kv):
        before[a:a + max(0, k.shape[0] // 2 - c)] = True  # rows that see none of them
    assert fine[before].all()
    close(out[before], want[before], bound[before])
    assert not torch.isfinite(out[~fine]).any()


def test_queries_that_are_not_finite_stay_in_their_rows(rq, gpu):
    b = Batch([(70, 60), (300, 1), (40, 1)], 4, 2, 64)
    want, bound = b.want()
    b.q[7, 1, 3] = float("nan")
    b.q[60, 2, 9] = float("inf")
    out = b.run()
    assert out[7, 1].isnan().all() and out[60, 2].isnan().all()
    keep = torch.ones(b.rows, 4, dtype=torch.bool, device="cuda")
    keep[7, 1] = keep[60, 2] = False
    close(out[keep], want[keep], bound[keep])


def test_pages_outside_the_pool_are_not_seen(rq, gpu):
    b = Batch([(300, 20), (100, 1)], 4, 2, 64)
    b.table[0, 1], b.table[0, 3], b.table[1, 0] = -1, b.pool.k.shape[0], 2**31 - 1
    out = b.run()
    gone = torch.zeros(320, dtype=torch.bool, device="cuda")
    gone[64:128] = gone[192:256] = True
    k, v = b.kv[0]
    for i in (0, 19):
        keep = ~gone & (torch.arange(320, device="cuda") <= 300 + i)
        close(out[i:i + 1], *ref.attention(b.q[i:i + 1], k[keep], v[keep], int(keep.sum()), b.scale))
    k, v = b.kv[1]
    close(out[20:21], *ref.attention(b.q[20:21], k[64:101], v[64:101], 37, b.scale))
    b.table.fill_(-3)
    assert (b.run() == 0).all()


def test_lengths_past_the_table_are_cut(rq, gpu):
    b = Batch([(100, 1), (60, 4)], 4, 2, 64)
    b.kv_len = ints([2**31 - 1, 2**31 - 1])  # the table names 128 positions, all on the pool's pages or none
    b.table[:, 1] = b.table[0, 1]
    b.pool.k.nan_to_num_(0.0)
    b.pool.v.nan_to_num_(0.0)
    out = b.run()
    for i, (r0, r1) in enumerate(((0, 1), (1, 5))):
        k, v = (ref.gather(p, b.table[i], 128, 64) for p in (b.pool.k, b.pool.v))
        close(out[r0:r1], *ref.attention(b.q[r0:r1], k, v, 1000, b.scale))


def test_more_rows_than_m_and_rows_before_zero(rq, gpu):
    b = Batch([(100, 3), (60, 9)], 4, 2, 64, pad=2)
    want, bound = b.want()
    b.row_start = ints([0, 3, 400])     # the second sequence claims 397 rows: its last is at kv_len - 1
    b.kv_len = ints([103, 461])         # so row 3 + i sees keys 0 .. 64 + i
    b.table = torch.cat([b.table, b.table[:, -1:].expand(2, 6)], 1).contiguous()
    b.width += 6
    b.table[1, 1:] = b.table[0, 0]
    b.pool.k.nan_to_num_(0.0)
    b.pool.v.nan_to_num_(0.0)
    out = b.run()
    close(out[:3], want[:3], bound[:3])
    k, v = (ref.gather(p, b.table[1], 461, 64) for p in (b.pool.k, b.pool.v))
    close(out[3:], *ref.attention(b.q[3:], k, v, 64, b.scale))
    b.row_start = ints([-4, 3, 12])     # rows before 0: that sequence is left out
    out = b.run()
    assert (out[:3] == -7.0).all()
    b.row_start = ints([5, 3, 12])      # a sequence that ends before it starts has no rows
    b.kv_len = ints([103, 69])
    assert (b.run()[:3] == -7.0).all()


def test_strided_rows(rq, gpu):
    b = Batch([(100, 40), (60, 1), (600, 1)], 8, 2, 64)
    wide = torch.full((b.rows, 3 * 8 * 64 + 12), 5.0, device="cuda")
    wide[:, :512] = b.q.view(b.rows, 512)
    out = wide[:, 516:516 + 512]  # q and out as parts of the same rows
    b.run(q=wide, out=out)
    close(out.reshape(b.rows, 8, 64), *b.want())
    assert (wide[:, 512:516] == 5.0).all() and (wide[:, 1028:] == 5.0).all()
    assert torch.equal(wide[:, :512], b.q.view(b.rows, 512))


def test_offsets_past_32_bits(rq, gpu):
    # a pool of more than 2^32 elements: the sequence's pages lie at both ends
    page, kvh, hd = 64, 8, 128
    pages = 2**32 // (page * kvh * hd) + 3
    k = torch.empty(pages, kvh, page, hd, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    c = A.KvPool(k.data_ptr(), v.data_ptr(), 1, pages, page, kvh, hd, *k.stride()[:3])
    ids = [pages - 1, 0, pages - 2, 1]
    torch.manual_seed(5)
    for p in ids:
        k[p], v[p] = torch.randn(2, kvh, page, hd, device="cuda").half()
    for rows in (1, 40):
        q = torch.randn(rows, 8, hd, device="cuda")
        out = torch.empty_like(q)
        table, rs, kl = ints([ids]), ints([0, rows]), ints([250])
        A.attention_paged_dev(c, q.data_ptr(), 8 * hd, 8, rows, rs.data_ptr(), kl.data_ptr(), 1, table.data_ptr(), 4,
                              0.1, out.data_ptr(), 8 * hd, rows, 250, stream())
        kk, vv = (ref.gather(p, table[0], 250, page) for p in (k, v))
        close(out, *ref.attention(q, kk, vv, 250 - rows, 0.1))
    # and the write there
    kr = torch.randn(1, kvh * hd, device="cuda")
    sl = ints([(pages - 1) * page + 5])
    A.store_dev(c, 1, None, 0, None, 0, 0, kr.data_ptr(), kvh * hd, kr.data_ptr(), kvh * hd, None, sl.data_ptr(), 0, 0,
                0, stream())
    assert torch.equal(k[pages - 1, :, 5], kr.view(kvh, hd).half())


def test_same_inputs_same_bits(rq, gpu):
    b = Batch([(3000, 1), (20, 200), (4000, 7)], 8, 2, 128)
    first = b.run()
    for _ in range(3):
        assert torch.equal(b.run(), first)


# ---- attention over packed prompts -----------------------------------------------------------


def run_packed(q, k, v, starts, scale, max_rows=0, m=None, out=None):
    kvh, hd = k.shape[1:]
    out = torch.full(q.shape, -7.0, device="cuda") if out is None else out
    A.attention_packed_dev(q.data_ptr(), q.stride(0), q.shape[1], k.data_ptr(), k.stride(0), v.data_ptr(),
                           v.stride(0), A.DTYPE_F16 if k.dtype == torch.float16 else A.DTYPE_F32, kvh, hd,
                           q.shape[0] if m is None else m, starts.data_ptr(), starts.numel() - 1, scale,
                           out.data_ptr(), out.stride(0), max_rows, stream())
    return out


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
@pytest.mark.parametrize("lens", [[1], [1, 2, 3, 0, 31, 32, 33], [64, 63, 65, 1], [300, 5, 129]])
def test_packed(rq, gpu, heads, kvh, hd, kv, lens):
    torch.manual_seed(hd + len(lens))
    rows = sum(lens) + 2
    qkv = torch.randn(rows, heads + 2 * kvh, hd, device="cuda")
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kvh].to(KV[kv][0]), qkv[:, heads + kvh:].to(KV[kv][0])
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    out = run_packed(q, k, v, ints(starts), 1 / math.sqrt(hd), max(lens))
    for a, z in zip(starts, starts[1:]):
        close(out[a:z], *ref.attention(q[a:z], k[a:z], v[a:z], 0, 1 / math.sqrt(hd)))
    assert (out[starts[-1]:] == -7.0).all()


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_packed_long(rq, gpu, kv):
    torch.manual_seed(1)
    lens = [2500, 1, 700, 64]
    rows = sum(lens)
    qkv = torch.randn(rows, 8, 128, device="cuda")
    q, k, v = qkv[:, :4], qkv[:, 4:6].to(KV[kv][0]), qkv[:, 6:].to(KV[kv][0])
    starts = [0, 2500, 2501, 3201, 3265]
    for hint in (0, 2500, 3):
        out = run_packed(q, k, v, ints(starts), 0.09, hint)
        for a, z in zip(starts, starts[1:]):
            close(out[a:z], *ref.attention(q[a:z], k[a:z], v[a:z], 0, 0.09))


@pytest.mark.parametrize("heads,kvh,hd", SHAPES)
def test_packed_prompts_split_beforehand(rq, gpu, heads, kvh, hd):
    # f32 prompts long enough that their keys are made f16 parts once a call; sizes around its tiles
    torch.manual_seed(hd)
    lens = [700, 1, 64, 65, 129, 900]
    rows = sum(lens) + 3
    qkv = torch.randn(rows, heads + 2 * kvh, hd, device="cuda")
    q, k, v = qkv[:, :heads], qkv[:, heads:heads + kvh], qkv[:, heads + kvh:]
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    out = run_packed(q, k, v, ints(starts), 1 / math.sqrt(hd), max(lens))
    for a, z in zip(starts, starts[1:]):
        close(out[a:z], *ref.attention(q[a:z], k[a:z], v[a:z], 0, 1 / math.sqrt(hd)))
    assert (out[starts[-1]:] == -7.0).all()
    first = out.clone()
    assert torch.equal(run_packed(q, k, v, ints(starts), 1 / math.sqrt(hd), max(lens)), first)


def test_packed_split_beforehand_wide_and_not_finite(rq, gpu):
    torch.manual_seed(4)
    n, hd = 1500, 64
    q, k, v = torch.randn(3, n, 4, hd, device="cuda")
    # values of very different sizes from tile to tile, tiles of zeros among them
    size = torch.logspace(-12, 12, n, device="cuda")[torch.randperm(n, device="cuda")][:, None, None]
    v = v * size
    k = k * torch.logspace(-8, 0, n, device="cuda")[torch.randperm(n, device="cuda")][:, None, None]
    k[64:192], v[128:256] = 0.0, 0.0
    close(run_packed(q, k, v, ints([0, n]), 0.1), *ref.attention(q, k, v, 0, 0.1))
    # values that are not finite reach the rows that see them and no others
    want, bound = ref.attention(q, k, v, 0, 0.1)
    k[1000, 1], v[1100, 2, 7], v[1200, :, 3] = float("nan"), float("inf"), float("nan")
    out = run_packed(q, k, v, ints([0, n]), 0.1)
    close(out[:1000], want[:1000], bound[:1000])
    close(out[1000:1100, 0], want[1000:1100, 0], bound[1000:1100, 0])
    assert out[1000:, 1].isnan().all()
    assert (out[1100:, 2, 7] == float("inf")).all()
    assert out[1200:, :, 3].isnan().all()
    close(out[1100:, 0, 8:], want[1100:, 0, 8:], bound[1100:, 0, 8:])


@pytest.mark.parametrize("n", [3, 40, 1500])
@pytest.mark.parametrize("power", [-118, -60, 60, 110])
def test_f32_values_of_extreme_size(rq, gpu, n, power):
    """Values by a power of two: the outputs by the same one, but for f32's last step near zero."""
    torch.manual_seed(n)
    q, k, v = torch.randn(3, n, 4, 64, device="cuda")
    v = v.sign() * v.abs().clamp(0.01, 4.0)
    a = run_packed(q, k, v, ints([0, n]), 0.1)
    b = run_packed(q, k, v * 2.0**power, ints([0, n]), 0.1)
    want, bound = ref.attention(q, k, v, 0, 0.1)
    close(a, want, bound)
    close(b.double() * 2.0**-power, want, bound + 2.0 ** (-149 - power))


def test_packed_split_beforehand_captured(rq, gpu):
    torch.manual_seed(6)
    q, k, v = torch.randn(3, 1200, 4, 64, device="cuda")
    starts = ints([0, 1200])
    out = torch.zeros_like(q)
    run_packed(q, k, v, starts, 0.1, out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        run_packed(q, k, v, starts, 0.1, out=out)
    for lens in ([0, 1200], [0, 500], [3, 1100]):
        for t in (q, k, v):
            t.normal_()
        starts.copy_(ints(lens))
        out.fill_(-7.0)
        g.replay()
        a, z = lens
        got = out.clone()
        torch.randn(1000, device="cuda").sum().item()
        assert torch.equal(run_packed(q, k, v, starts, 0.1), got)
        close(got[a:z], *ref.attention(q[a:z], k[a:z], v[a:z], 0, 0.1))


@pytest.mark.parametrize("n_seq", [65, 200, 4097])
def test_many_sequences(rq, gpu, n_seq):
    # more than one step of the search for a tile's sequence; sequences without rows among them
    r = random.Random(n_seq)
    lens = [r.choice([0, 1, 1, 2, 5, 70]) if n_seq < 1000 or i % 97 == 0 else r.choice([0, 1, 6]) for i in range(n_seq)]
    torch.manual_seed(n_seq)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    q, k, v = torch.randn(3, starts[-1] + 1, 2, 64, device="cuda")
    out = run_packed(q, k.half(), v.half(), ints(starts), 0.1, max(lens))
    seq = torch.repeat_interleave(torch.arange(n_seq), torch.tensor(lens)).cuda()
    i = torch.arange(starts[-1], device="cuda")
    for h in range(2):
        kk, vv = k[:-1, h].half().double(), v[:-1, h].half().double()
        s = (q[:-1, h].double() @ kk.T.contiguous()) * 0.1
        s = s.masked_fill((seq[:, None] != seq) | (i > i[:, None]), -math.inf)
        want = torch.softmax(s, -1) @ vv
        # |scores| below 8: weights off by 2^-17 at most (ref.attention), sums of at most 70 values below 6
        assert (out[:-1, h].double() - want).abs().max() <= 2.0**-17 * 6 * 4
    assert (out[-1] == -7.0).all()
    # the same as a step over a cache: every row its own sequence's tail
    b = Batch([(r.choice([0, 3, 64]), n) for n in lens[:200]], 4, 2, 64, page=16)
    b.check()


def test_packed_rows_before_the_first_and_bad_starts(rq, gpu):
    q, k, v = torch.randn(3, 20, 2, 64, device="cuda")
    out = run_packed(q, k, v, ints([4, 10]), 0.1)  # rows 0 .. 3 belong to nobody
    close(out[4:10], *ref.attention(q[4:10], k[4:10], v[4:10], 0, 0.1))
    assert (out[:4] == -7.0).all() and (out[10:] == -7.0).all()
    out = run_packed(q, k, v, ints([-6, 8, 500]), 0.1)  # before row 0: left out; past m: cut
    assert (out[:8] == -7.0).all()
    close(out[8:], *ref.attention(q[8:], k[8:], v[8:], 0, 0.1))
    out = run_packed(q, k, v, ints([12, 3, 2**31 - 1]), 0.1)
    close(out[3:], *ref.attention(q[3:], k[3:], v[3:], 0, 0.1))


def chunks_and_tokens(n_seq):
    """Chunks of 2 to 140 rows and single tokens behind caches of very different lengths."""
    r = random.Random(n_seq)
    return [(r.choice([0, 3, 700, 1900]) + r.randrange(60), r.choice([1, 1, 2, 20, 33, 140])) for _ in range(n_seq)]


@pytest.mark.parametrize("n_seq,heads,kvh,hd", [(2, 32, 8, 128), (5, 8, 1, 64), (16, 14, 2, 96), (3, 4, 2, 256),
                                                (64, 2, 1, 64), (70, 2, 1, 64)])
@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_chunks_whose_keys_are_split(rq, gpu, n_seq, heads, kvh, hd, kv):
    """Up to 64 sequences share the splits out on the device; more take the launch's own span."""
    b = Batch(chunks_and_tokens(n_seq), heads, kvh, hd, kv=kv, pad=3)
    b.check()
    for hints in ((0, 0), (2, 300), (100000, 1 << 20)):
        out = b.run(*hints)
        close(out[:b.rows], *b.want())


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_split_chunks_captured(rq, gpu, kv):
    b = Batch([(2500, 90), (30, 1), (900, 200), (1400, 1)], 8, 2, 64, kv=kv)
    out = torch.full((b.rows, 8, 64), -7.0, device="cuda")
    b.run(out=out)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        b.run(out=out)
    starts, lens = b.row_start.clone(), b.kv_len.clone()
    for drop in (0, 500, 0, 1300):  # fewer keys of each cache, other splits
        b.kv_len.copy_((lens - drop).clamp(min=0))
        b.q.normal_()
        out.fill_(-7.0)
        g.replay()
        got = out.clone()
        torch.randn(1000, device="cuda").sum().item()
        assert torch.equal(b.run(), got)
        if drop == 0:
            close(got, *b.want())
    assert torch.equal(b.row_start, starts)


@pytest.mark.parametrize("kv", ["f16", "f32"])
def test_sequences_that_share_rows_leave_later_calls_alone(rq, gpu, kv):
    """Split key ranges are joined by counters that the launches of a stream share."""
    b = Batch([(2990, 20), (2990, 0), (2990, 20), (1500, 0)], 4, 2, 64, kv=kv)
    want = b.run(max_rows=0, max_kv=0)
    proper = b.row_start, b.kv_len
    for _ in range(3):
        b.row_start, b.kv_len = ints([0, 20, 0, 20, 40]), ints([3010, 2990, 1400, 1500])
        b.run(max_rows=0, max_kv=0)
        b.row_start, b.kv_len = proper
        assert torch.equal(b.run(max_rows=0, max_kv=0), want)
    close(want, *b.want())


def test_packed_nan_behind_a_row(rq, gpu):
    torch.manual_seed(2)
    for dt in (torch.float16, torch.float32):
        q, k, v = torch.randn(3, 100, 2, 64, device="cuda")
        k, v = k.to(dt), v.to(dt)
        want, bound = ref.attention(q, k, v, 0, 0.1)
        k[50], v[60], v[70] = float("nan"), float("inf"), float("nan")
        out = run_packed(q, k, v, ints([0, 100]), 0.1)
        close(out[:50], want[:50], bound[:50])
        assert out[50:].isnan().all()


# ---- the operators together --------------------------------------------------------------------


class Server:
    """Plan, store and attention of consecutive steps, as a serving loop runs them, beside a per-sequence reference."""

    def __init__(self, n_seq, heads, kvh, hd, kv, page, rows, pages, width, seed=0):
        torch.manual_seed(seed)
        self.n, self.heads, self.kvh, self.hd, self.page, self.m = n_seq, heads, kvh, hd, page, rows
        self.pool = Pool(pages, page, kvh, hd, kv)
        self.free = torch.randperm(pages).tolist()
        self.table = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda")
        self.cached, self.new = ints([0] * n_seq), ints([0] * n_seq)
        self.free_dev = ints(self.free)
        z = lambda k: torch.zeros(k, dtype=torch.int32, device="cuda")  # noqa: E731
        self.row_start, self.kv_len, self.summary = z(n_seq + 1), z(n_seq), z(4)
        self.row_seq, self.positions, self.slots = z(rows), z(rows), z(rows)
        ang = torch.arange(width * page)[:, None] * 100.0 ** (-torch.arange(hd // 2) / (hd // 2))
        self.cos, self.sin = ang.cos().cuda(), ang.sin().cuda()
        self.qkv = torch.zeros(rows, (heads + 2 * kvh) * hd, device="cuda")
        self.out = torch.zeros(rows, heads * hd, device="cuda")
        self.held = [[torch.zeros(0, kvh, hd, device="cuda", dtype=self.pool.dtype)] * 2 for _ in range(n_seq)]

    def launch(self):
        s, hd = stream(), self.hd
        p = self.qkv.data_ptr()
        w = self.qkv.stride(0)
        A.plan_dev(self.cached.data_ptr(), self.new.data_ptr(), self.n, self.free_dev.data_ptr(),
                   self.free_dev.numel(), self.page, self.table.data_ptr(), self.table.shape[1],
                   self.row_start.data_ptr(), self.kv_len.data_ptr(), self.m, self.row_seq.data_ptr(),
                   self.positions.data_ptr(), self.slots.data_ptr(), self.summary.data_ptr(), s)
        A.store_dev(self.pool.c, self.m, p, w, p, w, self.heads, p + 4 * self.heads * hd, w,
                    p + 4 * (self.heads + self.kvh) * hd, w, self.positions.data_ptr(), self.slots.data_ptr(),
                    self.cos.data_ptr(), self.sin.data_ptr(), self.cos.shape[0], s)
        A.attention_paged_dev(self.pool.c, p, w, self.heads, self.m, self.row_start.data_ptr(), self.kv_len.data_ptr(),
                              self.n, self.table.data_ptr(), self.table.shape[1], 0.11, self.out.data_ptr(),
                              self.heads * hd, 0, 0, s)

    def step(self, new, go=None):
        """One step; the inputs change in place, as a captured graph needs."""
        hd, kvh = self.hd, self.kvh
        lens = [h[0].shape[0] for h in self.held]
        self.cached.copy_(ints(lens))
        self.new.copy_(ints(new))
        fresh = torch.randn_like(self.qkv)
        self.qkv.copy_(fresh)
        self.out.fill_(-7.0)
        (go or self.launch)()
        torch.cuda.synchronize()
        rows, taken, flags, longest = self.summary.tolist()
        assert (rows, flags, longest) == (sum(new), 0, max(a + b for a, b in zip(lens, new)))
        r = 0
        for b, n in enumerate(new):
            x = fresh[r:r + n].view(n, self.heads + 2 * kvh, hd)
            c, s = (t[lens[b]:lens[b] + n] for t in (self.cos, self.sin))
            q = ref.rope(x[:, :self.heads], c, s)[0].float()  # rounded as the rows in place are, to a step
            k = ref.rope(x[:, self.heads:self.heads + kvh], c, s)[0].float()
            got = ref.gather(self.pool.k, self.table[b], lens[b] + n, self.page)[lens[b]:]
            off = (got.double() - k.double()).abs()
            assert (off <= k.double().abs() * 2.0**-10 + 1e-6).all()
            # the cache's own values from here on: roundings of k to f16 may differ by one step
            v = x[:, self.heads + kvh:].to(self.pool.dtype)
            self.held[b] = [torch.cat([h, f]) for h, f in zip(self.held[b], (got, v))]
            rotated = self.qkv[r:r + n, :self.heads * hd].view(n, self.heads, hd)
            assert ((rotated - q).abs() <= q.abs() * 2.0**-21 + 1e-6).all()
            close(self.out[r:r + n].view(n, self.heads, hd),
                  *ref.attention(rotated, *self.held[b], lens[b], torch.tensor(0.11, dtype=torch.float32).item()))
            r += n
        assert (self.out[r:] == -7.0).all()
        del self.free[:taken]
        self.free_dev.copy_(ints((self.free + [0] * 10000)[:self.free_dev.numel()]))


@pytest.mark.parametrize("kv,page", [("f16", 64), ("f32", 16)])
def test_serving_steps(rq, gpu, kv, page):
    sv = Server(5, 8, 2, 64, kv, page, 96, 200, 400 // page)
    r = random.Random(2)
    sv.step([7, 0, 40, 1, 3])
    sv.step([1, 1, 1, 1, 1])
    for _ in range(4):
        sv.step([r.choice([0, 1, 1, 9, 18]) for _ in range(5)])
    sv.step([0, 0, 0, 0, 0])
    sv.step([1, 90, 1, 1, 1])


def test_captured_steps_follow_their_inputs(rq, gpu):
    """One captured graph, replayed over steps of different lengths, with eager work of the same operators between;
    a second graph on the same stream has its own work memory."""
    sv, other = (Server(6, 8, 2, 128, "f16", 64, 64, 400, 60, seed=i) for i in (1, 2))
    sv.step([5, 1, 0, 20, 1, 1])  # eager first
    graphs = []
    for x in (sv, other):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x.launch()
        graphs.append(g)
    for new in ([1, 1, 1, 1, 1, 1], [0, 50, 1, 1, 1, 1], [1, 1, 1, 1, 1, 1], [10, 10, 10, 10, 10, 10]):
        sv.step(new, graphs[0].replay)
        other.step(new[::-1], graphs[1].replay)
        torch.randn(1000, device="cuda").sum().item()
    sv.step([2, 1, 1, 3, 1, 1])
    # replays of both back to back
    sv.step([1, 1, 1, 1, 1, 0], lambda: (graphs[0].replay(), graphs[1].replay()))


def test_two_streams_at_once(rq, gpu):
    a, b = Batch([(4000, 1)] * 3, 8, 2, 128, seed=1), Batch([(2000, 30), (6000, 1)], 8, 2, 128, seed=2)
    wa, wb = a.run(), b.run()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]

    def go(i, x):
        for _ in range(10):
            with torch.cuda.stream(streams[i]):
                o = torch.zeros_like(wa if i == 0 else wb)
                x.run(out=o, s=streams[i].cuda_stream)
                outs[i].append(o)

    threads = [threading.Thread(target=go, args=(i, x)) for i, x in enumerate((a, b))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for i, w in enumerate((wa, wb)):
        assert all(torch.equal(o, w) for o in outs[i])
    for s in streams:
        rq.release_stream_work(s.cuda_stream)


# ---- sizes at the ends of f32 --------------------------------------------------------------------


@pytest.mark.parametrize("power", [-118, -112, -60, 60, 112, 118])
def test_f32_queries_and_keys_of_opposite_extremes(rq, gpu, power):
    """Queries by 2^-power and keys by 2^power: ordinary scores, in every kernel that takes f32 keys."""
    def sized(x):  # every element keeps its 24 bits at 2^-118
        return x.sign() * x.abs().clamp(0.01, 4.0)

    for lens in ([(300, 1), (40, 1), (0, 1), (2500, 1)], [(130, 90), (0, 40), (1500, 33)]):
        b = Batch(lens, 4, 2, 64, "f32")
        b.q = sized(b.q) * 2.0**-power
        b.kv = [(sized(k) * 2.0**power, v) for k, v in b.kv]
        for t, (k, v) in zip(b.table, b.kv):
            b.pool.put(t, k, v)
        b.check()
    for n in (3, 40, 1500):
        torch.manual_seed(n)
        q, k, v = torch.randn(3, n, 4, 64, device="cuda")
        q, k = sized(q) * 2.0**-power, sized(k) * 2.0**power
        close(run_packed(q, k, v, ints([0, n]), 0.125), *ref.attention(q, k, v, 0, 0.125))


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("n", [1, 3, 40, 1500])
def test_large_queries_and_keys_without_a_product(rq, gpu, kv, n):
    """Queries and keys that share no dimension: scores of 0 whatever their sizes, the average of the values seen."""
    torch.manual_seed(n)
    q, k, v = torch.randn(3, n, 4, 64, device="cuda")
    q[..., 32:], k[..., :32] = 0.0, 0.0
    q, scale = q * 2.0**100, 2.0**60
    k = k.half() if kv == "f16" else k * 2.0**110
    v = v.to(k.dtype)
    want = v.double().cumsum(0) / torch.arange(1, n + 1, device="cuda")[:, None, None]
    # the weights are equal and exact; values of 22 bits, n f32 sums, a division, a product
    bound = (v.double().abs().cumsum(0) / torch.arange(1, n + 1, device="cuda")[:, None, None]) * (n + 16) * 2.0**-23
    out = run_packed(q, k, v, ints([0, n]), scale)
    assert ((out.double() - want).abs() <= bound).all()
    b = Batch([(n - 1, 1), (5, 0), (0, n)], 4, 4, 64, kv)  # the same over pages
    for i in (0, 2):
        b.pool.put(b.table[i], k, v)
    b.q, b.scale = torch.cat([q[-1:], q]), scale
    out = b.run().double()
    assert ((out[0] - want[-1]).abs() <= bound[-1]).all() and ((out[1:] - want).abs() <= bound).all()


@pytest.mark.parametrize("n", [3, 40, 1500])
def test_scores_near_the_end_of_f32(rq, gpu, n):
    """Scores about 2^119 beside parts whose product would pass f32: the keys of the largest score share the weight."""
    torch.manual_seed(n)
    q, k = torch.zeros(2, n, 2, 64, device="cuda")
    v = torch.randn(n, 2, 64, device="cuda")
    q[..., 0], k[..., 2] = 2.0**100, 2.0**80
    q[..., 1] = 2.0**70
    size = torch.tensor([1.0, 2.0, 4.0], device="cuda")[torch.randint(0, 3, (n,), device="cuda")]
    k[..., 1] = 2.0**50 * size[:, None]
    out = run_packed(q, k, v, ints([0, n]), 0.125).double()
    b = Batch([(0, n), (n - 1, 1)], 2, 2, 64, "f32")
    for t in b.table:
        b.pool.put(t, k, v)
    b.q = torch.cat([q, q[-1:]])
    b.scale = 0.125
    paged = b.run().double()
    top = size[None] == size.cummax(0).values[:, None]
    w = torch.where(torch.ones(n, n, device="cuda").tril() > 0, top, False).double()
    w /= w.sum(1, keepdim=True)
    want = (w @ v.double().view(n, 128)).view(n, 2, 64)
    bound = (w @ v.double().abs().view(n, 128)).view(n, 2, 64) * (n + 16) * 2.0**-23
    assert ((out - want).abs() <= bound).all()
    assert ((paged[:n] - want).abs() <= bound).all() and ((paged[n] - want[-1]).abs() <= bound[-1]).all()


@pytest.mark.parametrize("power", [4, 11, 21, 26])
@pytest.mark.parametrize("n", [40, 700, 1500])
def test_equal_large_scores_weigh_alike(rq, gpu, n, power):
    """Equal scores of about 2^power beside f32 values whose sizes fall from key to key: equal weights."""
    torch.manual_seed(n)
    q = torch.zeros(n, 2, 64, device="cuda")
    k = torch.zeros(n, 2, 64, device="cuda")
    q[..., 0] = 2.0 ** (power // 2)
    k[..., 0] = 2.0 ** (power - power // 2) * 1.375
    # a first key whose score lies below the others': the running maximum moves, and the outputs' unit with it
    k[0, :, 0] -= (6 if power < 26 else 32) / 2.0 ** (power // 2)
    v = torch.randn(n, 2, 64, device="cuda")
    v = v.sign() * v.abs().clamp(0.5, 2.0)
    v *= 2.0 ** -(torch.arange(n, device="cuda") * (24 / n)).floor()[:, None, None]
    want, _ = ref.attention(q, k, v, 0, 1.0)
    mean, _ = ref.attention(q, k, v.abs(), 0, 1.0)
    # keys and scores are exact in 22 and in 24 bits and the largest is exact, so the weights are off by a rounding of
    # the first key's exponent and of its exponential; values of 22 bits, n f32 sums, a division, a product
    bound = mean * (n + 32) * 2.0**-23
    out = run_packed(q, k, v, ints([0, n]), 1.0).double()
    assert ((out - want).abs() <= bound).all(), float(((out - want).abs() / bound).max())
    b = Batch([(0, n), (n - 1, 1)], 2, 2, 64, "f32")
    for t in b.table:
        b.pool.put(t, k, v)
    b.q, b.scale = torch.cat([q, q[-1:]]), 1.0
    out = b.run().double()
    assert ((out[:n] - want).abs() <= bound).all() and ((out[n] - want[-1]).abs() <= bound[-1]).all()


@pytest.mark.parametrize("n", [3, 40, 1500])
def test_f32_parts_round_to_nearest(rq, gpu, n):
    """A row that sees one key returns that key's values to 23 bits, and its errors have both signs."""
    torch.manual_seed(n)
    v = torch.randn(n, 4, 64, device="cuda")
    v = v.sign() * v.abs().clamp(0.01, 4.0)  # nothing far below a row's largest
    q, k = torch.zeros_like(v), torch.zeros_like(v)
    i = torch.arange(n, device="cuda")[:, None] * 128.0
    q[..., 0], q[..., 1], k[..., 0], k[..., 1] = 1.0, -i, i, 1.0  # a score of 0 for the row's own key, -128 and less before
    outs = [run_packed(q, k, v, ints([0, n]), 1.0)]
    b = Batch([(0, n), (n - 1, 1)], 4, 4, 64, "f32")
    for t in b.table:
        b.pool.put(t, k, v)
    b.q, b.scale = torch.cat([q, q[-1:]]), 1.0
    out = b.run()
    outs += [out[:n], out[n:]]
    for o, w in zip(outs, (v, v, v[-1:])):
        # the weight is a power of two and the others' are below 2^-180: the value's parts (2^-23) and a sum of two products
        err = (o.double() - w.double()) / w.double()
        assert err.abs().max() <= 2.0**-23 + 2 * 2.0**-24, float(err.abs().max())
        if o.numel() >= 512:  # truncation would keep all of them below zero
            assert (err > 0).double().mean() >= 0.1 and (err < 0).double().mean() >= 0.1


def put_wide_values(v, at=(5, 0.5, -1)):
    """Infinities and NaN in single places of v [n, 2, hd]."""
    n = v.shape[0]
    a, b, z = (int(x * n) if 0 < x < 1 else min(x, n - 1) if x > 0 else n + x for x in at)
    v[a, 0, 1] = float("inf")
    v[b, 1, 7] = -float("inf")
    v[z, 0, 9] = float("nan")
    v[a, 1, 20], v[b, 1, 20] = float("inf"), -float("inf")
    v[b, 0, 30] = v[z, 0, 30] = -float("inf")


def same_places(got, want, bound):
    """close() without its figure for the whole, which takes scores of up to 2^4; here they reach 2^7."""
    got = got.double()
    assert torch.equal(got.isnan(), want.isnan())
    fine = torch.isfinite(want)
    assert torch.equal(got[~fine & ~want.isnan()], want[~fine & ~want.isnan()])
    assert ((got - want)[fine].abs() <= bound[fine]).all(), float(((got - want)[fine].abs() / bound[fine]).max())


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("lens", [[(70, 60), (300, 1), (0, 200)], [(3000, 1), (1700, 1), (8, 1)],
                                  [(2000, 90), (300, 40), (700, 1)], [(4000, 130)]])
def test_what_is_not_finite_stays_in_its_place(rq, gpu, kv, lens):
    """Every element of rows that see infinities or NaN: those elements by their sum, the others as without them, in
    masked and unmasked tiles, with split and whole key ranges."""
    b = Batch(lens, 4, 2, 64, kv, seed=7)
    for i, (k, v) in enumerate(b.kv):
        put_wide_values(v)
        k[min(5, k.shape[0] - 1)] *= 30  # a weight of nearly 1 or of nothing
        b.pool.put(b.table[i], k, v)
    want, bound = b.want()
    for hints in ((None, None), (0, 0), (1, 1), (1, 100000), (1000, 64)):
        same_places(b.run(*hints)[:b.rows], want, bound)


@pytest.mark.parametrize("kv", ["f16", "f32"])
@pytest.mark.parametrize("lens", [[3, 40], [130, 64, 1, 700], [1500]])
def test_packed_what_is_not_finite_stays_in_its_place(rq, gpu, kv, lens):
    torch.manual_seed(8)
    starts = [0]
    for n in lens:
        starts.append(starts[-1] + n)
    q, k, v = torch.randn(3, starts[-1], 2, 64, device="cuda")
    k, v = k.to(KV[kv][0]), v.to(KV[kv][0])
    for a, z in zip(starts, starts[1:]):
        put_wide_values(v[a:z])
        k[min(a + 5, z - 1)] *= 30
    out = run_packed(q, k, v, ints(starts), 0.1, max(lens))
    for a, z in zip(starts, starts[1:]):
        same_places(out[a:z], *ref.attention(q[a:z], k[a:z], v[a:z], 0, 0.1))


@pytest.mark.parametrize("power", [112, 122])
@pytest.mark.parametrize("lens", [[(20000, 1), (70, 1)], [(9000, 40)], [(3000, 5), (1200, 200)]])
def test_f32_values_near_the_end_of_f32_over_split_keys(rq, gpu, lens, power):
    """Values up to 2^(power + 2): their weighted means are in range, and so is every step to them."""
    b = Batch(lens, 4, 2, 64, "f32")
    for i, (k, v) in enumerate(b.kv):
        v.copy_(v.abs().clamp(0.5, 4.0))
        b.pool.put(b.table[i], k, v)
    want, bound = b.want()
    close(b.run()[:b.rows], want, bound)
    for i, (k, v) in enumerate(b.kv):
        b.pool.put(b.table[i], k, v * 2.0**power)
    close(b.run()[:b.rows].double() * 2.0**-power, want, bound)


@pytest.mark.parametrize("n_seq,m", [(3, 2**21 + 1), (5000, 2**22 + 77)])
def test_plan_of_more_rows_than_its_workgroups_take_at_once(rq, gpu, n_seq, m):
    r = random.Random(m)
    new = [2 * m // n_seq // 2 - r.randrange(50) for _ in range(n_seq)]
    cached = [r.randrange(300) for _ in range(n_seq)]
    page, pad = 1024, m - sum(new)
    need = [-(-(c + n) // page) - -(-c // page) for c, n in zip(cached, new)]
    width = max(-(-(c + n) // page) for c, n in zip(cached, new))
    tables = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda")
    tables[:, 0] = torch.arange(n_seq, device="cuda") + sum(need)  # the pages of what is cached
    free = torch.randperm(sum(need), device="cuda").int()
    cd, nd = ints(cached), ints(new)
    rs, kl, sm = (torch.zeros(k, dtype=torch.int32, device="cuda") for k in (n_seq + 1, n_seq, 4))
    seq, pos, slot = (torch.full((m,), -7, dtype=torch.int32, device="cuda") for _ in range(3))
    A.plan_dev(cd.data_ptr(), nd.data_ptr(), n_seq, free.data_ptr(), free.numel(), page, tables.data_ptr(), width,
               rs.data_ptr(), kl.data_ptr(), m, seq.data_ptr(), pos.data_ptr(), slot.data_ptr(), sm.data_ptr(), stream())
    assert pad >= 0 and sm.tolist() == [sum(new), sum(need), 0, max(c + n for c, n in zip(cached, new))]
    ids = torch.repeat_interleave(torch.arange(n_seq, device="cuda"), nd)
    start = torch.cumsum(nd, 0) - nd
    want = cd[ids] + (torch.arange(sum(new), device="cuda") - start[ids])
    assert torch.equal(seq[:m - pad].long(), ids) and (seq[m - pad:] == -1).all()
    assert torch.equal(pos[:m - pad].long(), want) and (pos[m - pad:] == 0).all()
    # the new pages come off the free list in order; the table names them
    have = torch.tensor([-(-c // page) for c in cached], device="cuda")
    first = torch.cumsum(torch.tensor(need, device="cuda"), 0) - torch.tensor(need, device="cuda")
    p = want // page
    pages = torch.where(p < have[ids], tables[ids, 0].long(), free.long()[(first[ids] + p - have[ids]).clamp(0)])
    assert torch.equal(slot[:m - pad].long(), pages * page + want % page) and (slot[m - pad:] == -1).all()
    assert torch.equal(tables[ids, p].long(), pages)
