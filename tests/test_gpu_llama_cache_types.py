"""What rdl_llama_config's kv_f16 stands for."""
import numpy as np
import pytest

from llama_fixtures import tiny_config
from test_gpu_llama_batch import build

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", [2, 3, -1, 4])
def test_any_other_number_is_an_f16_cache(rq, gpu, kv):
    a, _ = build(tiny_config(kv_f16=kv))
    b, _ = build(tiny_config(kv_f16=True))
    for t in ([1, 2, 3, 4, 5], [6], [7]):
        assert np.array_equal(a.forward_with_cache(t), b.forward_with_cache(t))
    assert np.array_equal(a.generate_greedy([8], 4), b.generate_greedy([8], 4))


def test_the_4_bit_cache_is_a_number_of_its_own(rq, gpu):
    from rdlquant.attention import KV_Q4 as pool_type
    from rdlquant.llama import KV_Q4
    assert KV_Q4 == pool_type
    m, _ = build(tiny_config(kv_f16=KV_Q4))
    with pytest.raises(rq.DeviceError):
        m.forward_with_cache([1])
    m.batch_begin(1)
    assert np.isfinite(m.batch_forward([[1, 2, 3]])).all()
