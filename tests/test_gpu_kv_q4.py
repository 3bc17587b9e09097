"""GPU tests of the head norms with the cache write, the 4-bit cache, forks
and page copies (include/rdl_attention.h) against plain implementations."""
import math
import random

import pytest
import torch

import attention_ref as ref
import kv_q4_ref as q4
from rdlquant import attention as A

pytestmark = pytest.mark.gpu
KV = {"f16": (torch.float16, A.DTYPE_F16), "f32": (torch.float32, A.DTYPE_F32), "q4": (torch.uint8, A.KV_Q4)}
STEP = 2.0 ** -24


def ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def stream():
    return torch.cuda.current_stream().cuda_stream


class Pool:
    """A pool of any type in one of the orders over memory filled with `fill` (bytes of 4-bit pools: 0xA5)."""

    def __init__(self, pages, page, kvh, hd, kv="f16", layout="heads", fill=float("nan")):
        dt, code = KV[kv]
        self.kv, self.page, self.hd, self.kvh, self.pages, self.dtype = kv, page, hd, kvh, pages, dt
        if kv == "q4":
            n = q4.run_bytes(page, hd)
            shape = {"heads": (pages, kvh, n), "positions": (kvh, pages, n), "padded": (pages, kvh, n + 32)}[layout]
            self.mem = [torch.full(shape, 0xA5, dtype=dt, device="cuda") for _ in range(2)]
            views = [t.transpose(0, 1) if layout == "positions" else t for t in self.mem]
            self.k, self.v = (q4.Runs(t, page, hd) for t in views)
            s = views[0].stride()
            self.c = A.KvPool(self.mem[0].data_ptr(), self.mem[1].data_ptr(), code, pages, page, kvh, hd, s[0], s[1], hd // 2)
            return
        shape = {"heads": (pages, kvh, page, hd), "positions": (pages, page, kvh, hd),
                 "padded": (pages, kvh, page + 1, hd + 8)}[layout]
        self.mem = [torch.full(shape, fill, dtype=dt, device="cuda") for _ in range(2)]
        view = {"heads": lambda t: t, "positions": lambda t: t.transpose(1, 2), "padded": lambda t: t[:, :, :page, :hd]}
        self.k, self.v = (view[layout](t) for t in self.mem)
        s = self.k.stride()
        self.c = A.KvPool(self.k.data_ptr(), self.v.data_ptr(), code, pages, page, kvh, hd, s[0], s[1], s[2])

    def both(self):
        """K and V [2, pages, kv heads, positions, hd] in 64 bits."""
        return torch.stack([x.values() if self.kv == "q4" else x.double() for x in (self.k, self.v)])

    def put(self, table, k, v):
        """Positions 0 .. len - 1 of a sequence."""
        pos = torch.arange(k.shape[0], device="cuda")
        ids, o = table[pos // self.page].long(), pos % self.page
        for x, y in ((self.k, k), (self.v, v)):
            if self.kv == "q4":
                x.put(ids, o, y)
            else:
                x[ids, :, o] = y.to(self.dtype)


# ---- norms, rotation, cache write ------------------------------------------------------------


def norm32(x, g, eps):
    """The documented arithmetic: the mean square in 64 bits, 1 / sqrt rounded to f32, then f32 products (on the CPU)."""
    mean = x.double().square().mean(-1, keepdim=True)
    r = (1 / (mean + eps).sqrt()).float()
    return x * r * g


def rope32(x, c, s):
    a, b = x.chunk(2, -1)
    return torch.cat([a * c - b * s, b * c + a * s], -1)


@pytest.mark.parametrize("kv,layout,hd", [
    (kv, layout, hd) for hd in (32, 64, 96, 128, 160, 256, 8, 40, 80)
    for kv, layout in (("q4", "heads"), ("f16", "padded"), ("f32", "positions"), ("q4", "padded"), ("q4", "positions"))
    if kv != "q4" or hd % 32 == 0])
@pytest.mark.parametrize("rope,in_place,norms", [(True, False, "qk"), (True, True, "k"), (False, False, "q"), (True, True, "")])
def test_store_norm(rq, gpu, hd, kv, layout, rope, in_place, norms):
    torch.manual_seed(hd)
    rows, heads, kvh, page, npos, eps = 37, 6, 2, 32, 90, 2.0 ** -17  # (f32 as 64 bits)
    pool = Pool(5, page, kvh, hd, kv, layout)
    before = [t.clone() for t in pool.mem]
    qkv = (torch.randn(rows, (heads + 2 * kvh) * hd + 4) * torch.logspace(-3, 3, rows)[:, None]).cuda()
    q, k, v = (qkv[:, a * hd:b * hd] for a, b in ((0, heads), (heads, heads + kvh), (heads + kvh, heads + 2 * kvh)))
    q0, k0, v0 = (x.cpu().reshape(rows, -1, hd) for x in (q, k, v))
    out = q if in_place else torch.full((rows, heads * hd), float("nan"), device="cuda")
    kept = out.clone()
    cap = 5 * page
    slots, pos = torch.randperm(cap)[:rows].int(), torch.randint(0, npos, (rows,)).int()
    slots[3], slots[5], slots[7] = -1, cap, -(2**31)
    skipped = {3, 5, 7}
    if rope:
        pos[9], pos[11] = -1, npos
        skipped |= {9, 11}
    ang = torch.rand(npos, hd // 2) * 6
    cos, sin = ang.cos(), ang.sin()
    g = [1 + 0.3 * torch.randn(hd) for _ in range(2)]
    dev = [x.cuda() for x in (pos, slots, cos, sin, *g)]
    ps, sl, cd, sd, gq, gk = (x.data_ptr() for x in dev)
    A.store_norm_dev(pool.c, rows, q.data_ptr(), q.stride(0), out.data_ptr(), out.stride(0), heads, k.data_ptr(), k.stride(0),
                     v.data_ptr(), v.stride(0), gq if "q" in norms else 0, gk if "k" in norms else 0, eps, ps, sl,
                     cd if rope else 0, sd if rope else 0, npos if rope else 0, stream())
    live = [r for r in range(rows) if r not in skipped]
    at = pos[live].long()
    want = []
    for x, n in ((q0[live], "q"), (k0[live], "k")):
        y = norm32(x, g[n == "k"], eps) if n in norms else x
        want.append(rope32(y, cos[at][:, None], sin[at][:, None]) if rope else y)
    # the same roundings in the same order: the same bits
    assert torch.equal(out[live].cpu().view(-1, heads, hd), want[0])
    for r in skipped:
        assert torch.equal(out[r].isnan(), kept[r].isnan()) and (not in_place or torch.equal(out[r], kept[r]))
    sel = slots[live].long()
    page_of, o = (sel // page).cuda(), (sel % page).cuda()
    for mem, x, y, was in ((pool.mem[0], pool.k, want[1], before[0]), (pool.mem[1], pool.v, v0[live], before[1])):
        if kv == "q4":
            d, c = q4.quantize(y)
            assert torch.equal(x.scales[page_of, :, o].cpu().view(torch.int16), d.view(torch.int16))
            assert torch.equal(x.codes[page_of, :, o].cpu(), q4.pack(c))
            x.scales[page_of, :, o], x.codes[page_of, :, o] = (
                t[page_of, :, o] for t in (lambda w: (w.scales, w.codes))(q4.Runs(was.transpose(0, 1) if layout == "positions" else was, page, hd)))
        else:
            assert torch.equal(x[page_of, :, o].cpu(), y.to(x.dtype))
            x[page_of, :, o] = float("nan")
        # every other element as it was
        assert torch.equal(mem.view(torch.uint8), was.view(torch.uint8))


@pytest.mark.parametrize("kv", ["f16", "q4"])
def test_more_rows_than_a_launch_has_workgroups(rq, gpu, kv):
    """Each workgroup then takes rows several times: one call, in place too, is bit for bit the calls of 499 and of 50000
    rows (which take one turn each)."""
    torch.manual_seed(4)
    rows, heads, hd, page, npos = 140001, 1, 32, 1024, 300
    q, k, v = torch.randn(3, rows, hd, device="cuda")
    g = 1 + 0.5 * torch.randn(hd, device="cuda")
    pos = torch.randint(-2, npos + 2, (rows,), device="cuda").int()
    slots = torch.randperm(140 * page, device="cuda")[:rows].int()
    slots[::1000] = -1
    ang = torch.rand(npos, hd // 2, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()

    def call(x, out, pool, r0, r1):
        A.store_norm_dev(pool.c, r1 - r0, x[r0:].data_ptr(), hd, out[r0:].data_ptr(), hd, heads, k[r0:].data_ptr(), hd,
                         v[r0:].data_ptr(), hd, g.data_ptr(), g.data_ptr(), 1e-6, pos[r0:].data_ptr(), slots[r0:].data_ptr(),
                         cos.data_ptr(), sin.data_ptr(), npos, stream())

    got = []
    for cuts in ([0, rows], [0, rows], [0, 499, 50499, 100499, rows]):
        pool = Pool(140, page, 1, hd, kv, fill=7.0)
        x = q.clone()
        out = x if len(got) == 1 else torch.full_like(q, 5.0)
        for r0, r1 in zip(cuts, cuts[1:]):
            call(x, out, pool, r0, r1)
        ok = (slots >= 0) & (pos >= 0) & (pos < npos)
        assert torch.equal(out[~ok], q[~ok] if len(got) == 1 else torch.full_like(q[~ok], 5.0))
        got.append([out[ok]] + [t.clone() for t in pool.mem])
    for other in got[1:]:
        assert all(torch.equal(a, b) for a, b in zip(got[0], other))


def test_norm_against_the_formula(rq, gpu):
    """Against 64 bits: r is off by half a step, two products and a rotation (two products and a sum) round once each."""
    torch.manual_seed(3)
    rows, heads, hd, eps = 65, 4, 128, 2.0 ** -20
    pool = Pool(5, 16, 1, hd, "f32")
    q = torch.randn(rows, heads, hd, device="cuda") * torch.logspace(-12, 12, rows, device="cuda")[:, None, None]
    k, v = torch.randn(2, rows, 1, hd, device="cuda")
    out = torch.empty_like(q)
    g = 1 + 0.5 * torch.randn(hd, device="cuda")
    pos, slots = ints(list(range(rows))), ints(list(range(rows)))
    ang = torch.rand(rows, hd // 2, device="cuda") * 6
    cos, sin = ang.cos(), ang.sin()
    A.store_norm_dev(pool.c, rows, q.data_ptr(), heads * hd, out.data_ptr(), heads * hd, heads, k.data_ptr(), hd, v.data_ptr(), hd,
                     g.data_ptr(), 0, eps, pos.data_ptr(), slots.data_ptr(), cos.data_ptr(), sin.data_ptr(), rows, stream())
    x = q.double()
    n = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * g.double()
    y, tol = ref.rope(n, cos, sin)
    # rope's bound is 2 steps of the products' sum; 3 more for r and the two products
    assert ((out.double() - y).abs() <= 2.5 * tol + 2.0 ** -140).all()


def test_rows_of_nothing_and_of_what_is_not_finite(rq, gpu):
    hd, eps = 64, 2.0 ** -20
    pool = Pool(1, 16, 1, hd, "q4")
    inf, nan = math.inf, math.nan
    rows = torch.randn(8, hd)
    rows[0] = 0
    rows[1, 5], rows[2, 40], rows[3, 3], rows[4] = nan, inf, -inf, 1e-42
    rows[5], rows[6] = 1e30, torch.linspace(-3e38, 3e38, hd)
    x = rows.cuda().view(8, 1, hd)
    out = torch.empty(8, hd, device="cuda")
    g, slots = torch.ones(hd, device="cuda"), ints(list(range(8)))
    A.store_norm_dev(pool.c, 8, x.data_ptr(), hd, out.data_ptr(), hd, 1, x.data_ptr(), hd, x.data_ptr(), hd, g.data_ptr(),
                     g.data_ptr(), eps, 0, slots.data_ptr(), 0, 0, 0, stream())
    want = norm32(rows, torch.ones(hd), eps)
    got = out.cpu()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.nan_to_num(7), want.nan_to_num(7))
    v = pool.v.values()[0, 0, :8].cpu()
    d, c = q4.quantize(rows)
    assert torch.equal(v.nan_to_num(9e9), q4.values(d, c).nan_to_num(9e9))
    assert v[1, :32].isnan().all() and not v[1, 32:].isnan().any()
    assert v[2, 32:].isnan().all() and v[3, :32].isnan().all() and (v[0] == 0).all() and (v[4] == 0).all()
    assert v[5].abs().amax() == 8 * 8160  # past the range: cut


# ---- page copies -----------------------------------------------------------------------------------


@pytest.mark.parametrize("hd,page,kvh", [(64, 16, 3), (128, 64, 2), (96, 32, 1), (256, 16, 2), (32, 1024, 1)])
@pytest.mark.parametrize("a", ["f16", "f32", "q4"])
@pytest.mark.parametrize("b", ["f16", "f32", "q4"])
def test_copy_pages(rq, gpu, a, b, hd, page, kvh):
    torch.manual_seed(hd)
    r = random.Random(page)
    layers = 3
    src = [Pool(7, page, kvh, hd, a, "heads") for _ in range(layers)]
    dst = [Pool(9, page, kvh, hd, b, "padded") for _ in range(layers)]
    for p in src:
        for m, x in zip(p.mem, (p.k, p.v)):
            y = torch.randn(7, kvh, page, hd) * 2.0 ** torch.randint(-12, 9, (7, kvh, page, 1))
            if a == "q4":
                d, c = q4.quantize(y)
                x.scales.copy_(d), x.codes.copy_(q4.pack(c))
            else:
                x.copy_(y)
    before = [[t.clone() for t in p.mem] for p in dst]
    pairs = [(r.randrange(7), p) for p in r.sample(range(9), 4)] + [(-1, 8), (7, 7), (2, -1), (3, 9), (2**31 - 1, 1)]
    pairs = [(x, y) for i, (x, y) in enumerate(pairs) if i < 4 or not (0 <= x < 7 and 0 <= y < 9)]
    f, t = ints([x for x, _ in pairs]), ints([y for _, y in pairs])
    A.copy_pages_dev([p.c for p in src], [p.c for p in dst], f.data_ptr(), t.data_ptr(), len(pairs), stream())
    done = pairs[:4]
    for s, d, was in zip(src, dst, before):
        for x, y, mem, w in ((s.k, d.k, d.mem[0], was[0]), (s.v, d.v, d.mem[1], was[1])):
            for i, j in done:
                if b == "q4":
                    if a == "q4":
                        ds, cs = x.scales[i].cpu(), x.codes[i].cpu()
                    else:
                        ds, cs = q4.quantize(x[i].float().cpu())
                        cs = q4.pack(cs)
                    assert torch.equal(y.scales[j].cpu().view(torch.int16), ds.view(torch.int16))
                    assert torch.equal(y.codes[j].cpu(), cs)
                else:
                    v = q4.values(x.scales[i], q4.unpack(x.codes[i])) if a == "q4" else x[i]
                    assert torch.equal(y[j], v.to(y.dtype))
            keep = [j for j in range(9) if j not in {j for _, j in done}]
            bits = lambda m: m.view(torch.uint8)[keep]  # noqa: E731
            assert torch.equal(bits(mem), bits(w))
            # the padding of written pages
            at = q4.run_bytes(page, hd) if b == "q4" else None
            for _, j in done:
                if at:
                    assert (mem[j][..., at:] == 0xA5).all()
                else:
                    assert mem[j][:, page:].isnan().all() and mem[j][..., hd:].isnan().all()


def test_copy_within_a_pool_and_many_layers(rq, gpu):
    torch.manual_seed(1)
    pools = [Pool(6, 16, 2, 64, "f16") for _ in range(70)]  # more than a launch takes
    for i, p in enumerate(pools):
        p.k.copy_(torch.randn(6, 2, 16, 64)), p.v.copy_(torch.randn(6, 2, 16, 64) + i)
    was = [(p.k.clone(), p.v.clone()) for p in pools]
    f, t = ints([0, 0, 3, 2]), ints([4, 5, 1, 2])  # one page twice, one onto itself
    c = [p.c for p in pools]
    A.copy_pages_dev(c, c, f.data_ptr(), t.data_ptr(), 4, stream())
    for p, (k, v) in zip(pools, was):
        for x, y in ((p.k, k), (p.v, v)):
            want = y.clone()
            want[4], want[5], want[1] = y[0], y[0], y[3]
            assert torch.equal(x, want)


def test_rounding_to_4_bits_at_its_borders(rq, gpu):
    """Halves between two codes, values beside them, both signs as large, smallest and largest scales: from f32 and through f16."""
    page, hd = 64, 32
    r = random.Random(5)
    rows = []
    for i in range(page):
        d = 2.0 ** r.choice([-24, -20, -14, -3, 0, 7, 12]) * r.choice([1, 255 / 128, 129 / 128, 1.5])
        row = [d * (k + 0.5) for k in range(-8, 7)] + [d * (k + 0.5) * (1 + s * 2.0 ** -23) for k in range(-4, 4) for s in (1, -1)]
        row = row[:31] + [r.choice([8, -8]) * d]
        if i % 5 == 0:
            row[3] = -row[31]
        rows.append(row)
    x = torch.tensor(rows, dtype=torch.float64).float().view(1, 1, page, hd)
    for kind in ("f32", "f16"):
        src, dst = Pool(1, page, 1, hd, kind), Pool(1, page, 1, hd, "q4")
        src.k.copy_(x), src.v.copy_(-x)
        z = ints([0])
        A.copy_pages_dev([src.c], [dst.c], z.data_ptr(), z.data_ptr(), 1, stream())
        for s, t in ((src.k, dst.k), (src.v, dst.v)):
            d, c = q4.quantize(s.float().cpu())
            assert torch.equal(t.scales.cpu().view(torch.int16), d.view(torch.int16))
            assert torch.equal(t.codes.cpu(), q4.pack(c))


# ---- forks --------------------------------------------------------------------------------------------


def plain_fork(tables, kv_len, page, parents, children, free):
    tables, kv_len = [list(r) for r in tables], list(kv_len)
    width = len(tables[0])
    src, dst, wanted, flags = [], [], 0, 0
    old, lens = [list(r) for r in tables], list(kv_len)
    for p, c in zip(parents, children):
        a = b = -1
        if not (0 <= p < len(kv_len) and 0 <= c < len(kv_len)) or p == c:
            flags |= 1
        else:
            n = max(0, min(lens[p], width * page))
            flags |= 2 if n != lens[p] else 0
            full = n // page
            tables[c][:full] = old[p][:full]
            if n % page:
                b = free[wanted] if wanted < len(free) else -1
                flags |= 4 if wanted >= len(free) else 0
                wanted += 1
                tables[c][full] = b
                a = old[p][full] if b >= 0 else -1
            kv_len[c] = n
        src.append(a), dst.append(b)
    return tables, kv_len, src, dst, [min(wanted, len(free)), flags]


def run_fork(tables, kv_len, page, parents, children, free):
    n = len(parents)
    t, k, f, c, fr = ints(tables), ints(kv_len), ints(parents or [0]), ints(children or [0]), ints(free or [0])
    out = [torch.full((s + 3,), -77, dtype=torch.int32, device="cuda") for s in (n, n, 2)]
    A.fork_dev(t.data_ptr(), t.shape[1], k.data_ptr(), len(kv_len), page, f.data_ptr(), c.data_ptr(), n, fr.data_ptr(), len(free),
               out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), stream())
    got = [o.tolist() for o in out]
    assert all(set(g[s:]) == {-77} for g, s in zip(got, (n, n, 2)))
    return t.tolist(), k.tolist(), got[0][:n], got[1][:n], got[2][:2]


@pytest.mark.parametrize("n,page,free", [(1, 64, 5), (40, 16, 100), (300, 16, 400), (2500, 32, 3000), (40, 16, 7), (9, 256, 0)])
def test_fork(rq, gpu, n, page, free):
    r = random.Random(n)
    parents_n = 1 + n // 3
    width = 11
    lens = [r.choice([0, 1, page - 1, page, page + 1, r.randrange(width * page), width * page]) for _ in range(parents_n)] + [-9] * n
    tables = [[r.randrange(10000) for _ in range(width)] for _ in lens]
    parents, children = [r.randrange(parents_n) for _ in range(n)], list(range(parents_n, parents_n + n))
    r.shuffle(children)
    pages = r.sample(range(20000, 40000), free)
    want = plain_fork(tables, lens, page, parents, children, pages)
    assert run_fork(tables, lens, page, parents, children, pages) == want


def test_fork_flags(rq, gpu):
    tables = [[1, 2, 3], [4, 5, 6], [0, 0, 0], [0, 0, 0], [0, 0, 0]]
    lens = [20, 2**31 - 1, -5, 7, 7]
    args = [([0, 1, -1, 0, 5, 2], [3, 4, 3, 9, 3, 2]), ([2], [3]), ([1], [3]), ([], []), ([0, 0], [3, 4])]
    for parents, children in args:
        for free in ([77], [77, 78, 79], []):
            assert run_fork(tables, lens, 16, parents, children, free) == plain_fork(tables, lens, 16, parents, children, free)


# ---- attention over 4 bits -------------------------------------------------------------------------------


def attend(pool, q, heads, lens, kv, tables, scale, out, max_rows=0, max_kv=0, m=None):
    start = [0]
    for n in lens:
        start.append(start[-1] + n)
    rs, kl = ints(start), ints(kv)
    A.attention_paged_dev(pool.c, q.data_ptr(), q.stride(0), heads, q.shape[0] if m is None else m, rs.data_ptr(), kl.data_ptr(),
                          len(lens), tables.data_ptr(), tables.shape[1], scale, out.data_ptr(), out.stride(0), max_rows, max_kv, stream())


def sequences(pool, kv, r, width=None, scale=1.0):
    """A table and k, v of sequences of kv[b] positions on shuffled pages."""
    need = [-(-n // pool.page) for n in kv]
    ids = list(range(pool.pages))
    r.shuffle(ids)
    tables, kvs = [], []
    for n, p in zip(kv, need):
        row = [ids.pop() for _ in range(p)]
        tables.append(row + [-1] * ((width or max(need + [1])) - p))
        k, v = (torch.randn(n, pool.kvh, pool.hd, device="cuda") * scale for _ in range(2))
        if n:
            pool.put(ints(tables[-1]), k, v)
        kvs.append((k, v))
    return ints(tables)


def floor_of_weights(v, n, heads, t):
    """What weights' smallest step adds to attention's bound: a weight is held as f16 parts, of whole steps of 2^-24, and
    cut toward zero, the largest between 2^11 and 2^15: each is off by at most 2^-35 of the largest, which the sum of
    weights is no less than, so row i's outputs by 2^-35 of the sum of the |v| that it sees.  Most 4-bit values are far
    above that, but a value is 0 in one of 16 cases, and where it has all the weight the others' are all there is."""
    sums = v.abs().nan_to_num(0, 0, 0).cumsum(0)[torch.arange(t - n, t, device="cuda").clamp(min=0)]
    return 2.0 ** -35 * sums.repeat_interleave(heads // v.shape[1], 1)


def check(pool, q, heads, lens, kv, tables, out, scale):
    """Each sequence's rows against 64 bits over the values that the pool stands for."""
    k, v = pool.both()
    r = 0
    for b, (n, t) in enumerate(zip(lens, kv)):
        kk, vv = (ref.gather(x, tables[b], t, pool.page) for x in (k, v))
        want, tol = ref.attention(q[r:r + n].view(n, heads, pool.hd), kk, vv, t - n, scale)
        got = out[r:r + n].view(n, heads, pool.hd).double()
        assert torch.equal(got.isnan(), want.isnan())
        f = torch.isfinite(want)
        assert torch.equal(got[~f].nan_to_num(5), want[~f].nan_to_num(5))
        off = (got - want).abs()[f]
        assert (off <= tol[f] + 1e-30).all(), (b, n, t, float((off / tol[f].clamp(min=1e-30)).max()))
        r += n


CASES = {
    "one": ([1], [1]), "decode": ([1] * 5, [1, 17, 64, 300, 1025]), "long": ([1, 1], [5000, 3]),
    "chunk": ([33], [33]), "chunks": ([5, 40, 1, 130, 0], [5, 300, 700, 131, 40]), "wide": ([300], [900]),
    "none": ([1, 3, 1], [0, 3, 2]),
}


@pytest.mark.parametrize("case", list(CASES))
@pytest.mark.parametrize("hd,heads,kvh,page", [(128, 8, 2, 64), (64, 4, 4, 16), (96, 6, 1, 32), (256, 4, 2, 16), (32, 16, 1, 128),
                                               (160, 3, 1, 64), (128, 7, 1, 1024)])
def test_attention(rq, gpu, case, hd, heads, kvh, page):
    lens, kv = CASES[case]
    torch.manual_seed(hd + len(kv))
    r = random.Random(hd)
    pool = Pool(sum(-(-n // page) for n in kv) + 3, page, kvh, hd, "q4", "padded")
    tables = sequences(pool, kv, r)
    m = sum(lens) + 2
    q = torch.randn(m, heads * hd + 8, device="cuda")[:, :heads * hd]
    for hint in (0, 1):
        out = torch.full((m, heads * hd), float("nan"), device="cuda")
        attend(pool, q, heads, lens, kv, tables, hd ** -0.5, out, max(lens) * hint, max(kv) * hint)
        check(pool, q[:m - 2], heads, lens, kv, tables, out, hd ** -0.5)
        assert out[m - 2:].isnan().all()  # rows behind the last sequence


@pytest.mark.parametrize("lens,kv,hd,heads,kvh,page", [
    ([1] * 48, [int(3000 * ((i * 37) % 48) / 47) + 1 for i in range(48)], 128, 8, 2, 64),  # dealt out over the launch
    ([1, 0, 1, 1, 0, 2], [5000, 300, 0, 1, 64, 2500], 64, 8, 2, 16),                       # sequences without rows or keys
    ([1] * 64, [700 + 13 * i for i in range(64)], 64, 4, 4, 32),                           # a lane each
    ([1] * 100, [300 + 7 * i for i in range(100)], 128, 4, 1, 128),                        # too many for a plan
    ([1], [40000], 128, 4, 1, 64),                                                          # more parts than are joined
    ([1, 2], [9000, 7000], 128, 8, 2, 64),                                                  # 4 and 8 pairs: packed
    ([1, 3], [9000, 7000], 128, 8, 2, 64),                                                  # 12 pairs: not
    ([1, 1], [9000, 7000], 256, 16, 1, 16),                                                 # 16 pairs, wide heads
    ([2, 1], [4000, 3000], 32, 3, 1, 16),
    ([1] * 5 + [40], [3000, 10, 700, 1500, 64, 900], 128, 8, 2, 32)])                       # single rows beside a chunk
def test_attention_of_split_keys(rq, gpu, lens, kv, hd, heads, kvh, page):
    torch.manual_seed(len(kv) + hd)
    pool = Pool(sum(-(-n // page) for n in kv) + 3, page, kvh, hd, "q4")
    tables = sequences(pool, kv, random.Random(hd))
    q = torch.randn(sum(lens), heads * hd, device="cuda")
    last = None
    for rows, keys in ((max(lens), max(kv)), (0, 0), (1, max(kv)), (1, 129)):  # the last two: less than there is
        out = torch.full_like(q, float("nan"))
        attend(pool, q, heads, lens, kv, tables, hd ** -0.5, out, rows, keys)
        check(pool, q, heads, lens, kv, tables, out, hd ** -0.5)
        again = torch.full_like(q, float("nan"))
        attend(pool, q, heads, lens, kv, tables, hd ** -0.5, again, rows, keys)
        assert torch.equal(out, again)  # whichever part arrives last
        last = out if last is None else last
        assert (out - last).abs().max() < 1e-4


def test_two_streams(rq, gpu):
    torch.manual_seed(5)
    hd, heads, kvh, page = 128, 8, 2, 64
    lens, kv = [1] * 20, [200 + 190 * i for i in range(20)]
    pool = Pool(sum(-(-n // page) for n in kv), page, kvh, hd, "q4")
    tables = sequences(pool, kv, random.Random(7))
    qs = [torch.randn(20, heads * hd, device="cuda") for _ in range(2)]
    want = [torch.empty_like(q) for q in qs]
    rs, kl = ints(list(range(21))), ints(kv)

    def call(q, out, s):
        A.attention_paged_dev(pool.c, q.data_ptr(), heads * hd, heads, 20, rs.data_ptr(), kl.data_ptr(), 20, tables.data_ptr(),
                              tables.shape[1], 0.1, out.data_ptr(), heads * hd, 1, max(kv), s)

    for q, w in zip(qs, want):
        call(q, w, stream())
    torch.cuda.synchronize()
    got, streams = [torch.empty_like(q) for q in qs], [torch.cuda.Stream() for _ in range(2)]
    for _ in range(30):
        for q, o, s in zip(qs, got, streams):
            call(q, o, s.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for o, w in zip(got, want))


def test_offsets_past_32_bits(rq, gpu):
    """Pages 3 GB apart: stored, attended to, copied."""
    torch.manual_seed(6)
    hd, heads, kvh, page, far = 64, 4, 1, 16, 3 << 30
    n = q4.run_bytes(page, hd)
    mem = [torch.empty(2 * far + n, dtype=torch.uint8, device="cuda") for _ in range(2)]
    runs = [torch.as_strided(t, (3, kvh, n), (far, n, 1)) for t in mem]
    pool = Pool(1, page, kvh, hd, "q4")
    pool.k, pool.v = (q4.Runs(t, page, hd) for t in runs)
    pool.pages = 3
    pool.c = A.KvPool(mem[0].data_ptr(), mem[1].data_ptr(), A.KV_Q4, 3, page, kvh, hd, far, n, hd // 2)
    rows = 40
    x = torch.randn(rows, (heads + 2) * hd, device="cuda")
    q, k, v = x[:, :heads * hd], x[:, heads * hd:(heads + 1) * hd], x[:, (heads + 1) * hd:]
    tables = ints([[2, 0, 1]])
    slots = ints([[2, 0, 1][i // page] * page + i % page for i in range(rows)])
    w = x.shape[1]
    out = torch.empty(rows, heads * hd, device="cuda")
    A.store_dev(pool.c, rows, q.data_ptr(), w, out.data_ptr(), heads * hd, heads, k.data_ptr(), w, v.data_ptr(), w, 0, slots.data_ptr(), 0,
                0, 0, stream())
    d, c = q4.quantize(k.cpu().view(rows, 1, hd))
    sl = slots.long()
    assert torch.equal(pool.k.codes[sl // page, :, sl % page].cpu(), q4.pack(c))
    got = torch.full((rows, heads * hd), float("nan"), device="cuda")
    for lens in ([rows], [1]):
        m = lens[0]
        attend(pool, q[rows - m:], heads, lens, [rows], tables, 0.125, got[rows - m:])
        check(pool, q[rows - m:].contiguous(), heads, lens, [rows], tables, got[rows - m:], 0.125)
    dst = Pool(2, page, kvh, hd, "f16")
    f, t = ints([2, 1]), ints([0, 1])
    A.copy_pages_dev([pool.c], [dst.c], f.data_ptr(), t.data_ptr(), 2, stream())
    both = pool.both()
    assert torch.equal(dst.k[0].double(), both[0, 2]) and torch.equal(dst.v[0].double(), both[1, 2])


@pytest.mark.parametrize("lens,kv", [([1, 1], [200, 130]), ([40, 70], [200, 130])])
def test_attention_of_blocks_without_finite_values(rq, gpu, lens, kv):
    """Masked blocks of NaN have no effect; seen ones are NaN in their own dims only, K's in the rows that see them."""
    torch.manual_seed(4)
    hd, heads, kvh, page = 128, 4, 2, 16
    for where in ("masked", "value", "key"):
        pool = Pool(40, page, kvh, hd, "q4")
        tables = sequences(pool, kv, random.Random(2))
        q = torch.randn(sum(lens), heads * hd, device="cuda")
        plain = torch.full_like(q, float("nan"))
        attend(pool, q, heads, lens, kv, tables, 0.09, plain)
        check(pool, q, heads, lens, kv, tables, plain, 0.09)
        for b, n in enumerate(kv):  # past the end of each sequence, on its last page
            if n % page:
                for x in (pool.k, pool.v):
                    x.scales[tables[b, n // page].long(), :, n % page:] = float("nan")
        out = torch.full_like(q, float("nan"))
        seen = kv[0] - 20  # of sequence 0: the last rows of a chunk see it, the single row does
        at = (tables[0, seen // page].long(), 1, seen % page, 2)
        if where == "value":
            pool.v.scales[at] = float("nan")
        if where == "key":
            pool.k.scales[at] = float("inf")
        attend(pool, q, heads, lens, kv, tables, 0.09, out)
        rows = torch.arange(lens[0], device="cuda") + kv[0] - lens[0] >= seen
        o, p = out.view(-1, heads, hd), plain.view(-1, heads, hd)
        if where == "masked":
            assert torch.equal(o, p)
        elif where == "value":
            bad = torch.zeros_like(o, dtype=torch.bool)
            bad[:lens[0], 2:, 64:96] = rows[:, None, None]
            assert torch.equal(o.isnan(), bad)
            same = torch.where(bad, 0.0, (o - p).abs())
            assert (same <= 2.0 ** -20 * (1 + p.abs())).all()
        else:  # rows that do not see the key, the other heads and the other sequence are as before
            assert torch.equal(o[lens[0]:], p[lens[0]:]) and torch.equal(o[:, :2], p[:, :2])
            assert torch.equal(o[:lens[0]][~rows], p[:lens[0]][~rows])


def test_attention_pages_outside_the_pool(rq, gpu):
    torch.manual_seed(9)
    hd, heads, kvh, page = 64, 4, 1, 16
    lens, kv = [1, 50], [100, 90]
    pool = Pool(20, page, kvh, hd, "q4")
    tables = sequences(pool, kv, random.Random(3))
    bad = tables.clone()
    bad[0, 2], bad[1, 1], bad[1, 4] = -1, 20, 2**31 - 1
    q, out = torch.randn(51, heads * hd, device="cuda"), torch.full((51, heads * hd), float("nan"), device="cuda")
    attend(pool, q, heads, lens, kv, bad, 0.125, out)
    k, v = pool.both()
    r = 0
    for b, (n, t) in enumerate(zip(lens, kv)):
        kk, vv = (ref.gather(x, tables[b], t, page) for x in (k, v))
        inside = torch.tensor([0 <= int(bad[b, j // page]) < 20 for j in range(t)], device="cuda")
        for i in range(n):
            see = inside & (torch.arange(t, device="cuda") <= t - n + i)
            want, tol = ref.attention(q[r + i:r + i + 1].view(1, heads, hd), kk[see], vv[see], int(see.sum()) - 1, 0.125)
            assert ((out[r + i].view(1, heads, hd).double() - want).abs() <= tol + 1e-30).all()
        r += n


def test_scales_of_more_bits_and_large_scores(rq, gpu):
    """Scales of a whole f16 number: values are rounded to f16.  Scores of hundreds: one key takes all the weight."""
    torch.manual_seed(8)
    hd, heads, kvh, page = 128, 8, 2, 64
    lens, kv = [1, 35], [500, 300]
    pool = Pool(15, page, kvh, hd, "q4")
    tables = sequences(pool, kv, random.Random(1))
    for x in (pool.k, pool.v):
        x.scales.copy_((x.scales.float() * (1 + torch.rand_like(x.scales.float()) / 64)).half())
    q = torch.randn(36, heads * hd, device="cuda") * torch.logspace(-1, 2.5, 36, device="cuda")[:, None]
    out = torch.full_like(q, float("nan"))
    attend(pool, q, heads, lens, kv, tables, 1.0, out)
    both = pool.both().half().double()
    r = 0
    for b, (n, t) in enumerate(zip(lens, kv)):
        kk, vv = (ref.gather(x, tables[b], t, page) for x in both)
        want, tol = ref.attention(q[r:r + n].view(n, heads, hd), kk, vv, t - n, 1.0)
        assert ((out[r:r + n].view(n, heads, hd).double() - want).abs() <= tol + floor_of_weights(vv, n, heads, t)).all()
        r += n


# ---- together -------------------------------------------------------------------------------------------------


def test_steps_forks_and_graphs(rq, gpu):
    """Two prompts into a 4-bit cache, forked, and a step of all continuations; then the step captured and replayed
    with the program's own work between the replays."""
    torch.manual_seed(12)
    hd, heads, kvh, page, layers, npos = 128, 8, 2, 16, 2, 200
    pools = [Pool(40, page, kvh, hd, "q4") for _ in range(layers)]
    side = torch.cuda.Stream()
    ang = torch.rand(npos, hd // 2, device="cuda") * 6
    cos, sin, g = ang.cos(), ang.sin(), 1 + 0.2 * torch.randn(hd, device="cuda")
    n_seq, width, m = 5, 12, 80
    tables = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda")
    cached, new = ints([0] * n_seq), ints([37, 32, 0, 0, 0])
    free = ints(random.Random(1).sample(range(40), 40))
    start, kl = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (n_seq + 1, n_seq))
    seq, pos, slots = (torch.zeros(m, dtype=torch.int32, device="cuda") for _ in range(3))
    summary = torch.zeros(4, dtype=torch.int32, device="cuda")
    qkv = torch.randn(layers, m, (heads + 2 * kvh) * hd, device="cuda")
    out = torch.zeros(layers, m, heads * hd, device="cuda")

    def step(taken, s):
        A.plan_dev(cached.data_ptr(), new.data_ptr(), n_seq, free.data_ptr() + 4 * taken, 40 - taken, page, tables.data_ptr(), width,
                   start.data_ptr(), kl.data_ptr(), m, seq.data_ptr(), pos.data_ptr(), slots.data_ptr(), summary.data_ptr(), s)
        for l, p in enumerate(pools):
            x = qkv[l].data_ptr()
            w = qkv.shape[2]
            A.store_norm_dev(p.c, m, x, w, out[l].data_ptr(), heads * hd, heads, x + heads * hd * 4, w, x + (heads + kvh) * hd * 4, w,
                             g.data_ptr(), g.data_ptr(), 1e-6, pos.data_ptr(), slots.data_ptr(), cos.data_ptr(), sin.data_ptr(), npos, s)
            # the normed queries are read from `out`, the attention's result goes into q's place
            A.attention_paged_dev(p.c, out[l].data_ptr(), heads * hd, heads, m, start.data_ptr(), kl.data_ptr(), n_seq,
                                  tables.data_ptr(), width, hd ** -0.5, x, w, 0, 0, s)

    def verify():
        lens = (start[1:] - start[:-1]).tolist()
        for l, p in enumerate(pools):
            q, got = out[l], qkv[l][:, :heads * hd]
            check(p, q[:sum(lens)], heads, lens, kl.tolist(), tables, got, hd ** -0.5)

    with torch.cuda.stream(side):
        step(0, side.cuda_stream)
    side.synchronize()
    verify()
    # three continuations: two of the first (whose last page is copied), one of the second (whose pages are full)
    f, c = ints([0, 0, 1]), ints([2, 3, 4])
    src, dst, taken = (torch.zeros(n, dtype=torch.int32, device="cuda") for n in (3, 3, 2))
    A.fork_dev(tables.data_ptr(), width, kl.data_ptr(), n_seq, page, f.data_ptr(), c.data_ptr(), 3, free.data_ptr() + 4 * 5, 35,
               src.data_ptr(), dst.data_ptr(), taken.data_ptr(), stream())
    ps = [p.c for p in pools]
    A.copy_pages_dev(ps, ps, src.data_ptr(), dst.data_ptr(), 3, stream())
    assert taken.tolist() == [2, 0] and kl.tolist() == [37, 32, 37, 37, 32]
    assert dst.tolist()[2] == -1 and len({*dst.tolist()}) == 3
    for p in pools:
        both = p.both()
        for b in (2, 3):
            assert torch.equal(ref.gather(both[0], tables[b], 37, page), ref.gather(both[0], tables[0], 37, page))
            assert tables[b, 2] != tables[0, 2] and torch.equal(tables[b, :2], tables[0, :2])
    cached.copy_(kl)
    new.copy_(ints([1, 2, 1, 3, 1]))
    qkv.normal_()
    keep = qkv.clone(), tables.clone(), [[t.clone() for t in p.mem] for p in pools]
    step(7, stream())
    verify()
    want = [qkv.clone(), out.clone(), tables.clone()] + [t.clone() for p in pools for t in p.mem]

    def restore():
        qkv.copy_(keep[0]), tables.copy_(keep[1]), out.fill_(-1.0)
        for p, mem in zip(pools, keep[2]):
            for t, x in zip(p.mem, mem):
                t.copy_(x)

    restore()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side), torch.cuda.graph(graph, stream=side):
        step(7, side.cuda_stream)
    rows = int(start[-1])
    for _ in range(4):
        restore()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [qkv, out, tables] + [t for p in pools for t in p.mem]
        for x, y in zip(got, want):
            if x.dim() == 3 and x.dtype == torch.float32:
                x, y = x[:, :rows], y[:, :rows]
            assert torch.equal(x, y)
        (torch.randn(512, 512, device="cuda") @ torch.randn(512, 512, device="cuda")).sum().item()
