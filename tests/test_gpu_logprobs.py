"""GPU tests of rdl_logprobs_dev (include/rdl_llama.h) against 64 bits."""
import math

import pytest
import torch

from rdlquant import llama as L

pytestmark = pytest.mark.gpu


def run(x, tokens, top, vocab=None, entropy=True):
    m = x.shape[0]
    vocab = vocab or x.shape[1]
    lp, en = (torch.full((m + 2,), 77.0, device="cuda") for _ in range(2))
    ids = torch.full((m + 1, max(top, 1)), -77, dtype=torch.int32, device="cuda")
    tl = torch.full((m + 1, max(top, 1)), 77.0, device="cuda")
    L.logprobs_dev(x.data_ptr(), x.stride(0), m, vocab, 0 if tokens is None else tokens.data_ptr(),
                   0 if tokens is None else lp.data_ptr(), en.data_ptr() if entropy else 0, top, ids.data_ptr() if top else 0,
                   tl.data_ptr() if top else 0, torch.cuda.current_stream().cuda_stream)
    assert (lp[m:] == 77).all() and (en[m:] == 77).all() and (ids[m:] == -77).all() and (tl[m:] == 77).all()
    if tokens is None:
        assert (lp == 77).all()
    if not entropy:
        assert (en == 77).all()
    return lp[:m], en[:m], ids[:m, :top], tl[:m, :top]


def check(x, tokens, top):
    """Bounds: d = x - M rounds once and by log2(e) once more, so e^d is off by (2 |d| + 2) 2^-24 of itself; a lane sums at
    most n = vocab / 64 of them and 64 lanes, 4 waves and 64 parts join in 14 more steps.  S and T = sum e^d d are
    off by that, their logarithm, quotient and the differences behind them round once or twice each."""
    lp, en, ids, tl = run(x, tokens, top)
    y = x.double()
    M = y.amax(1, keepdim=True)
    d = y - M
    p = torch.softmax(y, 1)
    logp = torch.log_softmax(y, 1)
    fin = torch.where(p > 0, d, 0.0)
    a1, a2 = (p * fin.abs()).sum(1), (p * fin * fin).sum(1)
    n = -(-x.shape[1] // 64) + 20
    e_s = 2.0 ** -24 * (2 * a1 + 2 + n)
    log_s = torch.log_softmax(y, 1).amax(1).neg()
    tol = e_s + 2.0 ** -23 * (log_s + 1)
    want = logp.gather(1, tokens.long()[:, None])[:, 0]
    here = want > -math.inf
    assert torch.equal(lp == -math.inf, ~here)
    off = (lp.double() - want).abs()[here]
    assert (off <= (tol + 2.0 ** -23 * want.abs())[here]).all(), float(off.max())
    want = -(p * torch.where(p > 0, logp, 0.0)).sum(1)
    e_t = 2.0 ** -24 * (2 * a2 + (2 + n) * a1) + e_s * a1 + 2.0 ** -23 * a1
    assert ((en.double() - want).abs() <= tol + e_t + 2.0 ** -23 * want).all(), float((en.double() - want).abs().max())
    if top:
        best, at = torch.sort(y, dim=1, descending=True, stable=True)
        assert torch.equal(ids.long(), at[:, :top])
        w = logp.gather(1, at[:, :top])
        assert torch.equal(tl == -math.inf, w == -math.inf)
        f = w > -math.inf
        assert ((tl.double() - w).abs()[f] <= (tol[:, None] + 2.0 ** -23 * w.abs())[f]).all()


@pytest.mark.parametrize("m,vocab,top,pad", [
    (1, 1, 1, 0), (1, 2, 2, 3), (3, 63, 20, 1), (2, 64, 64, 0), (5, 65, 64, 0), (4, 1023, 5, 1), (3, 1024, 1, 0),
    (2, 1025, 5, 2), (1, 4097, 64, 0), (7, 5000, 0, 1), (1, 32000, 5, 0), (16, 32003, 20, 1), (1, 262147, 64, 0),
    (1, 300000, 0, 0), (1100, 997, 3, 0), (600, 9001, 20, 2), (1030, 4100, 64, 0)])
def test_rows(rq, gpu, m, vocab, top, pad):
    torch.manual_seed(vocab)
    mem = torch.full((m, vocab + pad), 1e30, device="cuda")  # what is between the rows is not read as theirs
    x = mem[:, :vocab]
    x.copy_(torch.randn(m, vocab, device="cuda") * (0.1 + 8 * torch.rand(m, 1, device="cuda")))
    check(x, torch.randint(0, vocab, (m,), device="cuda").int(), top)


@pytest.mark.parametrize("m,vocab", [(1, 6000), (40, 3000), (1500, 1400)])
def test_equal_values_go_to_the_lower_index(rq, gpu, m, vocab):
    torch.manual_seed(m)
    for levels in (1, 2, 5):
        x = torch.randint(0, levels, (m, vocab), device="cuda").float() - 2
        x = torch.where((x == -2) & (torch.rand_like(x) < 0.5), -0.0 * x, x)
        x = torch.where(x == 0, torch.where(torch.rand_like(x) < 0.5, -0.0, 0.0), x)
        check(x, torch.randint(0, vocab, (m,), device="cuda").int(), 20)


@pytest.mark.parametrize("order", ["up", "down", "one lane"])
def test_orders_that_fill_the_list_again_and_again(rq, gpu, order):
    vocab = 20000
    x = torch.arange(vocab, device="cuda").float() / 500
    if order == "down":
        x = x.flip(0)
    if order == "one lane":
        x = torch.where(torch.arange(vocab, device="cuda") % 256 < 4, x + 40, x)
    x = torch.stack([x, x + 1, -x])
    check(x.contiguous(), torch.tensor([0, vocab - 1, 7], dtype=torch.int32, device="cuda"), 64)


@pytest.mark.parametrize("m", [2, 1200])
def test_masked_logits(rq, gpu, m):
    torch.manual_seed(m)
    vocab = 2500
    x = torch.randn(m, vocab, device="cuda") * 3
    x.masked_fill_(torch.rand(m, vocab, device="cuda") < 0.5, -math.inf)
    x[0, 5:] = -math.inf   # fewer tokens than alternatives
    x[0, :5] = torch.tensor([1.0, -math.inf, 3.0, 2.0, -math.inf])
    x[1, :] = -math.inf
    x[1, 2222] = -5.0      # one token left
    tokens = torch.randint(0, vocab, (m,), device="cuda").int()
    tokens[0], tokens[1] = 2, 2222
    check(x, tokens, 20)
    lp, en, ids, _ = run(x, tokens, 20)
    assert lp[1] == 0 and en[1] == 0 and ids[1].tolist()[:3] == [2222, 0, 1]


@pytest.mark.parametrize("m,vocab", [(4, 9000), (1027, 700)])
def test_rows_without_probabilities(rq, gpu, m, vocab):
    torch.manual_seed(2)
    x = torch.randn(m, vocab, device="cuda")
    good = x.clone()
    x[0, vocab - 1], x[1, 3] = math.nan, math.inf
    x[2] = -math.inf
    tokens = torch.zeros(m, dtype=torch.int32, device="cuda")
    tokens[3] = -1
    lp, en, ids, tl = run(x, tokens, 5)
    assert lp[:4].isnan().all() and en[:3].isnan().all() and (ids[:3] == -1).all() and tl[:3].isnan().all()
    assert torch.isfinite(en[3:]).all()
    check(good[3:], torch.full((m - 3,), vocab - 1, dtype=torch.int32, device="cuda"), 5)
    assert torch.equal(run(good, tokens, 5)[2][3:], ids[3:])


def test_far_values(rq, gpu):
    """Logits far from 0, differences that f32 holds: what matters is their distance from the largest."""
    torch.manual_seed(7)
    x = (torch.randn(5, 3000, device="cuda") * 30).round()
    for shift in (2.0 ** 20, -2.0 ** 20):
        check(x + shift, torch.zeros(5, dtype=torch.int32, device="cuda"), 5)
    y = torch.full((2, 700), -3.0e38, device="cuda")
    y[:, 9] = 3.0e38
    lp, en, ids, tl = run(y, torch.full((2,), 9, dtype=torch.int32, device="cuda"), 2)
    assert (lp == 0).all() and (en == 0).all() and (ids[:, 0] == 9).all() and (ids[:, 1] == 0).all()


def test_parts_of_the_outputs(rq, gpu):
    torch.manual_seed(0)
    x = torch.randn(3, 5000, device="cuda")
    t = torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda")
    whole = run(x, t, 4)
    assert torch.equal(run(x, None, 4)[2], whole[2]) and torch.equal(run(x, t, 0)[0], whole[0])
    assert torch.equal(run(x, t, 4, entropy=False)[3], whole[3]) and torch.equal(run(x, None, 0)[1], whole[1])


def test_streams_and_graphs(rq, gpu):
    """Two streams at once, each with work memory of its own, and a captured call replayed with other logits."""
    torch.manual_seed(1)
    x = [torch.randn(6, 20000, device="cuda") * 4 for _ in range(2)]
    t = torch.arange(6, device="cuda").int()
    want = [[o.clone() for o in run(v, t, 7)] for v in x]
    out = [[torch.zeros_like(o) for o in w] for w in want]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def call(v, o, s):
        L.logprobs_dev(v.data_ptr(), 20000, 6, 20000, t.data_ptr(), o[0].data_ptr(), o[1].data_ptr(), 7, o[2].data_ptr(),
                       o[3].data_ptr(), s)

    torch.cuda.synchronize()
    for _ in range(20):
        for v, o, s in zip(x, out, streams):
            call(v, o, s.cuda_stream)
    torch.cuda.synchronize()
    for o, w in zip(out, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
    buf, o = x[0].clone(), out[0]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(streams[0]), torch.cuda.graph(graph, stream=streams[0]):
        call(buf, o, streams[0].cuda_stream)
        call(buf, o, streams[0].cuda_stream)
    for i in (1, 0, 1, 1, 0):
        buf.copy_(x[i])
        for a in o:
            a.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(o, want[i]))
        run(x[1 - i], t, 7)
