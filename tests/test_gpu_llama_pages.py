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
