"""Steps of several sequences through the decoder (rdl_llama_batch_*) against
the CPU restatement, one LlamaRef a sequence."""
import numpy as np
import pytest

from oracle.llama_ref import LlamaRef
from parity import assert_close

from llama_fixtures import tiny_config, tiny_weights

pytestmark = pytest.mark.gpu


def build(cfg, types=None):
    from rdlquant.llama import LlamaModel
    slots, ref_w = tiny_weights(cfg, 1234, types=types, centered=True)
    m = LlamaModel(cfg, types)
    for slot, layer, arr in slots:
        m.set_weight(slot, layer, arr)
    return m, lambda: LlamaRef(cfg, ref_w, kv_f16=bool(cfg.kv_f16))


def check_step(m, refs, tokens):
    before = m.batch_positions()
    got = m.batch_forward(tokens)
    for b, t in enumerate(tokens):
        if t:
            assert_close(got[b], refs[b].forward_with_cache(t))
        else:
            assert np.isnan(got[b]).all()
    assert m.batch_positions() == [p + len(t) for p, t in zip(before, tokens)]


@pytest.mark.parametrize("kw", [dict(), dict(kv_f16=True), dict(n_heads=2, n_kv_heads=2, head_dim=128),
                                dict(n_heads=8, n_kv_heads=1, head_dim=32, max_batch=100)])
def test_steps_of_several_sequences(rq, gpu, kw):
    cfg = tiny_config(max_seq=512, **{"max_batch": 48, **kw})
    m, new = build(cfg)
    m.batch_begin(4)
    refs = [new() for _ in range(4)]
    r = np.random.default_rng(5)

    def toks(n):
        return r.integers(0, cfg.vocab, n).tolist()

    check_step(m, refs, [toks(9), [], toks(30), toks(1)])       # prompts, one still without rows
    check_step(m, refs, [toks(1), toks(20), toks(1), toks(1)])  # single tokens beside a prompt
    for _ in range(3):
        check_step(m, refs, [toks(1) for _ in range(4)])
    check_step(m, refs, [toks(1), [], [], toks(1)])
    for _ in range(3):
        check_step(m, refs, [[], toks(40), [], toks(1)])        # past the first page
    m.batch_drop(1)                                            # its pages go to others
    refs[1] = new()
    check_step(m, refs, [toks(1), toks(3), toks(40), []])
    check_step(m, refs, [toks(2), toks(2), toks(40), toks(1)])
    # a reset gives the cache back to one sequence
    m.reset()
    ref = new()
    t = toks(7)
    assert_close(m.forward_with_cache(t), ref.forward_with_cache(t))


@pytest.mark.parametrize("native", [False, True])
def test_mixed_types(rq, gpu, native):
    from rdlquant import llama as L
    cfg = tiny_config(max_seq=256, max_batch=40, kv_f16=True, output_dtype=14)
    types = {(L.WQ, 0): 12, (L.WK, 0): 12, (L.WV, 0): 14, (L.W_DOWN, 0): 14, (L.WQ, 1): 8, (L.WK, 1): 8,
             (L.WV, 1): 8, (L.W_GATE, 1): 3}
    m, new = build(cfg, types)
    m.set_native_q4_matmul(native)
    m.batch_begin(3)
    # the same steps one sequence at a time: other kernels for other row counts, so in tolerance of one another
    one, _ = build(cfg, types)
    one.set_native_q4_matmul(native)
    steps = [[[5, 6, 7], [9] * 20, [1]], [[3], [4], [200]], [[8], [2, 2], [1, 5, 9]]]
    got = [m.batch_forward(s) for s in steps]
    for b in range(3):
        one.reset()
        for s, g in zip(steps, got):
            want = one.forward_with_cache(s[b])
            if native:  # a Q8_0 code at a border may round the other way: bounded by the codes' own step
                assert np.abs(g[b] - want).max() <= 0.02 * np.abs(want).max()
            else:
                assert_close(g[b], want)


def test_more_sequences_than_four_and_the_cache_full(rq, gpu):
    cfg = tiny_config(max_seq=640, max_batch=128, kv_f16=True)  # 10 pages
    m, new = build(cfg)
    m.batch_begin(9)
    refs = [new() for _ in range(9)]
    r = np.random.default_rng(6)
    check_step(m, refs, [r.integers(0, cfg.vocab, 3 + b).tolist() for b in range(9)])
    # sequence 0 grows past its page: one page is left, two are not
    with pytest.raises(rq.InvalidData) as e:
        m.batch_forward([[1] * 126] + [[]] * 8)
    assert "full" in str(e.value)
    assert m.batch_positions() == [3 + b for b in range(9)]
    check_step(m, refs, [r.integers(0, cfg.vocab, 100).tolist()] + [[2]] * 8)
    m.batch_drop(8)
    check_step(m, refs[:8] + [new()], [[1] * 60] + [[3]] * 7 + [[]])


def test_refusals(rq, gpu):
    cfg = tiny_config()
    m, new = build(cfg)
    for call in (lambda: m.batch_forward([[1]]), lambda: m.batch_drop(0)):
        with pytest.raises(rq.InvalidData):
            call()
    m.forward_with_cache([1, 2])
    with pytest.raises(rq.InvalidData):
        m.batch_begin(2)  # the cache is not empty
    m.reset()
    for n in (0, 5000):
        with pytest.raises(rq.InvalidData):
            m.batch_begin(n)
    m.batch_begin(2)
    with pytest.raises(rq.InvalidData):
        m.batch_begin(2)
    with pytest.raises(rq.InvalidData):
        m.forward_with_cache([1])
    with pytest.raises(rq.InvalidData):
        m.generate_greedy([1], 3)
    with pytest.raises(rq.InvalidData):
        m.batch_drop(2)
    for bad, kind in (([[1]], rq.ShapeMismatch), ([[], []], rq.ShapeMismatch), ([[1] * 17, []], rq.ShapeMismatch),
                      ([[1], [cfg.vocab]], rq.InvalidData), ([[-1], [1]], rq.InvalidData)):
        with pytest.raises(kind):
            m.batch_forward(bad)
    for _ in range(4):
        m.batch_forward([[1] * 16, []])
    with pytest.raises(rq.InvalidData):
        m.batch_forward([[1], []])  # past max_seq
    assert m.batch_positions() == [64, 0]
    m.reset()
    with pytest.raises(rq.InvalidData):
        m.batch_positions()
    m.batch_begin(3)  # more than before
    refs = [new() for _ in range(3)]
    with pytest.raises(rq.InvalidData):
        m.batch_forward([[3], [], [4, 5]])  # one page, two sequences
    check_step(m, refs, [[], [], [4, 5]])
    bad = tiny_config(dim=96, n_heads=8, n_kv_heads=4, head_dim=12)
    from rdlquant.llama import LlamaModel
    with pytest.raises(rq.DeviceError) as e:
        LlamaModel(bad).batch_begin(2)
    assert e.value.status == rq.ERR_UNSUPPORTED


def test_memory_of_a_batch(rq, gpu):
    """Logits are kept of the rows that a step can have, not of every sequence, and a larger batch takes the smaller
    one's place."""
    import torch
    cfg = tiny_config(vocab=32000, max_seq=64 * 8, max_batch=16)
    m, new = build(cfg)
    used = lambda: -torch.cuda.mem_get_info()[0]  # noqa: E731
    m.batch_begin(2)
    check_step(m, [new(), new()], [[1, 2], [3]])
    m.reset()
    before = used()
    for n in (600, 1200, 2400, 4096):
        m.batch_begin(n)
        m.reset()
        # 16 rows of logits (2 MB), 4096 page tables of 8 and a few ints a sequence
        assert used() - before <= 16 << 20, n
    m.batch_begin(4096)
    refs = [new() for _ in range(3)]
    toks = [[]] * 4096
    toks[5], toks[2000], toks[4095] = [1, 2, 3], [7], [9, 9]
    got = m.batch_forward(toks)
    for r, b in zip(refs, (5, 2000, 4095)):
        assert_close(got[b], r.forward_with_cache(toks[b]))
