"""The batch decoder's forks, log probabilities and 4-bit cache
(rdl_llama_batch_fork, rdl_llama_batch_logprobs, RDL_LLAMA_KV_Q4)."""
import numpy as np
import pytest
import torch

import kv_q4_ref as q4
from oracle import llama_ref
from oracle.llama_ref import LlamaRef
from parity import assert_close

from llama_fixtures import tiny_config, tiny_weights
from test_gpu_llama_batch import build

pytestmark = pytest.mark.gpu


def toks(r, cfg, n):
    return r.integers(0, cfg.vocab, n).tolist()


@pytest.mark.parametrize("kv", [False, True])
def test_forks_go_on_as_their_parents_would(rq, gpu, kv):
    cfg = tiny_config(max_seq=640, max_batch=150, kv_f16=kv)
    m, new = build(cfg)
    r = np.random.default_rng(3)
    m.batch_begin(6)
    prompts = [toks(r, cfg, 70), toks(r, cfg, 64), [], [], [], []]
    m.batch_forward(prompts)
    m.batch_fork([0, 0, 1], [2, 4, 5])
    assert m.batch_positions() == [70, 64, 70, 0, 70, 64]
    history = [prompts[0], prompts[1], prompts[0], [], prompts[0], prompts[1]]
    refs = []
    for h in history:
        refs.append(new())
        if h:
            refs[-1].forward_with_cache(h)
    for step in range(3):  # every copy goes its own way, past its own page's end
        t = [toks(r, cfg, 1 + 20 * (b == step)) if history[b] else [] for b in range(6)]
        got = m.batch_forward(t)
        for b in range(6):
            if t[b]:
                assert_close(got[b], refs[b].forward_with_cache(t[b]))
    # pages that are shared outlive their first holder
    m.batch_drop(0)
    m.batch_drop(1)
    t = [toks(r, cfg, 80), [], [7], [], [8], [9]]
    got = m.batch_forward(t)
    refs[0] = new()
    for b in (0, 2, 4, 5):
        assert_close(got[b], refs[b].forward_with_cache(t[b]))


def test_pages_are_counted(rq, gpu):
    cfg = tiny_config(max_seq=256, max_batch=150, kv_f16=True)  # four pages
    m, _ = build(cfg)
    m.batch_begin(5)
    m.batch_forward([[1] * 128, [], [], [], []])
    m.batch_fork([0, 0, 0], [1, 2, 3])  # full pages alone: none is taken
    m.batch_forward([[1], [2], [], [], []])
    with pytest.raises(rq.InvalidData):
        m.batch_forward([[], [], [3], [], []])
    with pytest.raises(rq.InvalidData):  # a part page needs one
        m.batch_fork([0], [4])
    assert m.batch_positions() == [129, 129, 128, 128, 0]
    for b in (0, 2, 3):
        m.batch_drop(b)
    m.batch_fork([1], [4])  # the page of 0's last position
    with pytest.raises(rq.InvalidData):
        m.batch_forward([[5], [], [], [], []])
    m.batch_drop(1), m.batch_drop(4)
    m.batch_forward([[1] * 150, [], [], [], []])
    m.batch_forward([[1] * 106, [], [], [], []])  # all four pages again
    assert m.batch_positions()[0] == 256


def test_fork_refusals(rq, gpu):
    cfg = tiny_config(max_seq=512, max_batch=40)
    m, _ = build(cfg)
    with pytest.raises(rq.InvalidData):
        m.batch_fork([0], [1])  # no sequences
    m.batch_begin(4)
    m.batch_forward([[1, 2], [3], [], []])
    for p, c in (([0], [1]), ([0], [0]), ([0], [4]), ([-1], [2]), ([4], [2]), ([0, 1], [2, 2]), ([0, 2], [2, 3]),
                 ([0] * 5, [2] * 5)):
        with pytest.raises(rq.InvalidData):
            m.batch_fork(p, c)
    assert m.batch_positions() == [2, 1, 0, 0]
    m.batch_fork([], [])
    m.batch_fork([3], [2])  # an empty one's copy is empty
    m.batch_fork([0, 1], [2, 3])
    assert m.batch_positions() == [2, 1, 2, 1]


def test_logprobs_of_a_step(rq, gpu):
    cfg = tiny_config(max_seq=512, max_batch=60)
    m, _ = build(cfg)
    one, _ = build(cfg)
    r = np.random.default_rng(4)
    m.batch_begin(4), one.batch_begin(4)
    for t in ([toks(r, cfg, 9), [], toks(r, cfg, 30), toks(r, cfg, 1)], [[1], [2, 3], [], [4]]):
        targets = [5, 6, 7, 8]
        logits = one.batch_forward(t)
        lp, en, ids, tl = m.batch_logprobs(t, targets, 5)
        assert m.batch_positions() == one.batch_positions()
        for b in range(4):
            if not t[b]:
                assert np.isnan(lp[b]) and np.isnan(en[b]) and (ids[b] == -1).all() and np.isnan(tl[b]).all()
                continue
            want = torch.log_softmax(torch.from_numpy(logits[b]).double(), 0).numpy()
            # f32 sums of cfg.vocab terms, a difference and a logarithm
            tol = (cfg.vocab / 64 + 40) * 2.0 ** -23 * (1 + np.abs(want).max())
            order = np.argsort(-logits[b], kind="stable")[:5]
            assert (ids[b] == order).all()
            assert abs(lp[b] - want[targets[b]]) <= tol and (np.abs(tl[b] - want[order]) <= tol).all()
            assert abs(en[b] + (np.exp(want) * want).sum()) <= tol * (1 + np.abs(want).max())
    lp, en, ids, tl = m.batch_logprobs([[1], [], [], []])
    assert lp is None and ids.shape == (4, 0) and np.isfinite(en[0])
    before = m.batch_positions()
    for kw in (dict(n_top=65), dict(n_top=cfg.vocab + 1)):
        with pytest.raises(rq.DeviceError):
            m.batch_logprobs([[1], [], [], []], **kw)
    with pytest.raises(rq.InvalidData):
        m.batch_logprobs([[cfg.vocab], [], [], []], [1, 1, 1, 1])
    assert m.batch_positions() == before


class FourBitRef(LlamaRef):
    """The CPU restatement whose cache keeps what 4 bits keep of each position."""

    @staticmethod
    def kept(x):
        d, c = q4.quantize(torch.from_numpy(np.ascontiguousarray(x, dtype=np.float32)))
        return q4.values(d, c).numpy().astype(np.float32)


def test_decoder_over_a_4_bit_cache(rq, gpu, monkeypatch):
    from rdlquant.llama import KV_Q4
    cfg = tiny_config(max_seq=512, max_batch=90, kv_f16=KV_Q4)
    m, _ = build(cfg)
    _, ref_w = tiny_weights(cfg, 1234, types=None, centered=True)
    ref32 = LlamaRef(cfg, ref_w, kv_f16=False)
    # the plain restatement over the same cache: keys and values pass through 4 bits before the attention reads them
    plain = llama_ref.attention

    def over_4_bits(q, kc, vc, start):
        return plain(q, FourBitRef.kept(kc), FourBitRef.kept(vc), start)

    r = np.random.default_rng(9)
    m.batch_begin(3)
    steps = [[toks(r, cfg, 70), [], toks(r, cfg, 3)], [[5], toks(r, cfg, 10), [6]], [[7], [8], [9]]]
    refs = [LlamaRef(cfg, ref_w, kv_f16=False) for _ in range(3)]
    monkeypatch.setattr(llama_ref, "attention", over_4_bits)
    for t in steps:
        got = m.batch_forward(t)
        for b in range(3):
            if t[b]:
                want = refs[b].forward_with_cache(t[b])
                # The two sides' keys and values differ by some 2^-20 of themselves, so one in 2^16 lies on the two
                # sides of a border of two codes and takes another one: none or one of the 36000 here, an eighth of its
                # block's largest in one value of 64, with its position's weight (1 / 70 and up): 1 / 8 / 8 / 70 and
                # up, 2^-12 .. 2^-9.  Rounding itself moves the logits by some 2^-4.
                off = np.linalg.norm(got[b] - want) / np.linalg.norm(want)
                assert off < 2e-3, off
    monkeypatch.undo()
    exact = ref32.forward_with_cache(steps[0][0])
    assert np.linalg.norm(exact) > 0
    m.batch_drop(1)
    m.batch_fork([0], [1])
    a = m.batch_forward([[11], [11], []])
    assert np.array_equal(a[0], a[1])
    m.reset()
    for call in (lambda: m.forward_with_cache([1]), lambda: m.generate_greedy([1, 2], 3)):
        with pytest.raises(rq.DeviceError) as e:
            call()
        assert e.value.status == rq.ERR_UNSUPPORTED


def test_4_bit_decoders_need_whole_blocks(rq, gpu):
    from rdlquant.llama import KV_Q4, LlamaModel
    with pytest.raises(rq.InvalidData):
        LlamaModel(tiny_config(kv_f16=KV_Q4, n_heads=16, n_kv_heads=16, head_dim=16))
