"""The batch decoder's page bookkeeping and uploads (rdl_llama_batch_*)."""
import numpy as np
import pytest

from llama_fixtures import tiny_config
from parity import assert_close
from test_gpu_llama_batch import build

pytestmark = pytest.mark.gpu


def test_steps_in_a_row_gather_their_own_last_rows(rq, gpu):
    """40 sequences of which another part has tokens in each step, against steps of one sequence at a time."""
    cfg = tiny_config(max_seq=4096, max_batch=100, kv_f16=True)
    a, _ = build(cfg)
    b, _ = build(cfg)
    n = 40
    a.batch_begin(n), b.batch_begin(n)
    r = np.random.default_rng(1)
    for step in range(6):
        t = [r.integers(0, cfg.vocab, int(r.integers(0, 3))).tolist() for _ in range(n)]
        t[step] = r.integers(0, cfg.vocab, 7).tolist()
        if step % 2:
            got = a.batch_forward(t)
        else:  # the tokens that one at a time finds likeliest
            _, _, ids, _ = a.batch_logprobs(t, n_top=1)
        for s in range(n):
            if t[s]:
                one = b.batch_forward([t[s] if k == s else [] for k in range(n)])[s]
                if step % 2:
                    assert_close(got[s], one)
                else:
                    assert one[ids[s, 0]] >= one.max() - 1e-3 * np.abs(one).max()
    assert a.batch_positions() == b.batch_positions()


# 12, 8, 7 and 3 pages: enough, too few at times, too few mostly.  least: how often each call at least comes about
@pytest.mark.parametrize("max_seq,least", [(768, dict(step=20, fork=5, drop=5)), (512, dict(step=20, fork=5, drop=5, full=5)),
                                           (448, dict(step=15, fork=5, drop=5, full=15)), (192, dict(drop=2, full=40))])
def test_forks_and_drops_at_random(rq, gpu, max_seq, least):
    """Sequences forked, dropped and continued, against a decoder that runs each history alone."""
    cfg = tiny_config(max_seq=max_seq, max_batch=130, kv_f16=False)
    m, _ = build(cfg)
    alone, _ = build(cfg)
    n, r = 7, np.random.default_rng(8)
    m.batch_begin(n)
    history = [[] for _ in range(n)]
    done = dict(step=0, fork=0, drop=0, full=0)
    for _ in range(60):
        what = r.random()
        busy, empty = [s for s in range(n) if history[s]], [s for s in range(n) if not history[s]]
        if what < 0.5 or not busy:
            t = [r.integers(0, cfg.vocab, int(r.choice([0, 1, 2, 18]))).tolist() for _ in range(n)]
            if not any(t):
                continue
            try:
                got = m.batch_forward(t)
            except rq.InvalidData as e:
                assert "full" in str(e)
                done["full"] += 1
                continue
            for s in range(n):
                history[s] = history[s] + t[s]
            s = int(r.choice([s for s in range(n) if t[s]]))
            alone.reset()
            alone.batch_begin(1)
            for i in range(0, len(history[s]), 130):
                want = alone.batch_forward([history[s][i:i + 130]])
            assert_close(got[s], want[0])
            done["step"] += 1
        elif what < 0.75 and empty:
            c = [int(x) for x in r.permutation(empty)[:int(r.integers(1, len(empty) + 1))]]
            p = [int(r.choice(busy)) for _ in c]
            try:
                m.batch_fork(p, c)
            except rq.InvalidData as e:
                assert "full" in str(e)
                done["full"] += 1
                continue
            for a, b in zip(p, c):
                history[b] = list(history[a])
            done["fork"] += 1
        else:
            s = int(r.integers(0, n))
            m.batch_drop(s)
            history[s] = []
            done["drop"] += 1
        assert m.batch_positions() == [len(h) for h in history]
    assert all(done[k] >= v for k, v in least.items()), done
