"""Refusals of the head norms with the cache write, 4-bit pools, forks, page
copies and log probabilities: bad arguments end in the documented status
before anything is launched, so no device is needed."""
import pytest
import torch

import kv_q4_ref as q4
from rdlquant import attention as A
from rdlquant import llama as L

HALF = dict(k_dev=1 << 20, v_dev=1 << 21, dtype=1, n_pages=4, page_positions=64, n_kv_heads=2, head_dim=64,
            page_stride=2 * 64 * 64, head_stride=64 * 64, position_stride=64)
RUN = 64 * (32 + 4)
FOUR = dict(HALF, dtype=A.KV_Q4, page_stride=2 * RUN, head_stride=RUN, position_stride=32)
Q, K, V, OUT, INTS, G = 1 << 22, 1 << 23, 1 << 24, 1 << 25, 1 << 26, 1 << 27  # addresses nothing reads


def pool(base=FOUR, **kw):
    return A.KvPool(*[{**base, **kw}[n] for n, _ in A.KvPool._fields_])


def store(p, m=4, q=Q, qs=256, qo=OUT, qos=256, heads=4, k=K, ks=128, v=V, vs=128, gq=G, gk=G, eps=1e-6, pos=INTS, slots=INTS,
          cos=INTS, sin=INTS, n=10):
    A.store_norm_dev(p, m, q, qs, qo, qos, heads, k, ks, v, vs, gq, gk, eps, pos, slots, cos, sin, n, 0)


def paged(p, scale=0.125, rs=INTS):
    A.attention_paged_dev(p, Q, 256, 4, 4, rs, INTS, 2, INTS, 4, scale, OUT, 256, 0, 0, 0)


def test_block_format_round_trip():
    x = torch.randn(3, 2, 96) * 5
    d, c = q4.quantize(x)
    assert torch.equal(q4.unpack(q4.pack(c)), c) and q4.pack(c).shape[-1] == 48
    v = q4.values(d, c)
    assert torch.equal(v, v.half().double())  # values are f16 numbers
    assert ((v - x).abs().unflatten(-1, (-1, 32)) <= d.double().abs()[..., None] * (0.5 + 0.55)).all()
    assert torch.equal(q4.pack(torch.tensor([[0, 1, 2, 3, 4, 5, 6, 7]])), torch.tensor([[0x20, 0x64, 0x31, 0x75]], dtype=torch.uint8))


@pytest.mark.parametrize("change,kind", [
    (dict(head_dim=48, position_stride=24), "DeviceError"), (dict(head_dim=72), "DeviceError"),
    (dict(position_stride=64), "ShapeMismatch"), (dict(position_stride=0), "ShapeMismatch"),
    (dict(head_stride=RUN + 8), "InvalidData"), (dict(page_stride=2 * RUN + 4), "InvalidData"),
    (dict(head_stride=RUN - 16), "ShapeMismatch"), (dict(page_stride=2 * RUN - 16), "ShapeMismatch"),
    (dict(page_stride=RUN // 2 // 16 * 16), "ShapeMismatch"), (dict(page_stride=-2 * RUN), "ShapeMismatch"),
    (dict(k_dev=8), "InvalidData"), (dict(v_dev=0), "DeviceError"), (dict(page_positions=8), "DeviceError"),
    (dict(dtype=0x105), "DTypeMismatch"), (dict(dtype=2), "DTypeMismatch"),
])
def test_4_bit_pool_refusals(rq, change, kind):
    for call in (store, paged, lambda p: A.store_dev(p, 4, Q, 256, OUT, 256, 4, K, 128, V, 128, INTS, INTS, INTS, INTS, 10, 0),
                 lambda p: A.copy_pages_dev([pool(), p], [pool(), p], INTS, INTS, 3, 0)):
        with pytest.raises(getattr(rq, kind)):
            call(pool(**change))


def test_4_bit_pools_pass_the_checks(rq):
    for call in (lambda: store(pool(), slots=0), lambda: paged(pool(), rs=0),
                 lambda: paged(pool(page_stride=RUN, head_stride=4 * RUN), rs=0)):
        with pytest.raises(rq.DeviceError) as e:
            call()
        assert e.value.status == rq.ERR_NULL_POINTER


def test_packed_rows_are_not_4_bits(rq):
    with pytest.raises(rq.DTypeMismatch):
        A.attention_packed_dev(Q, 256, 4, K, 128, V, 128, A.KV_Q4, 2, 64, 4, INTS, 2, 0.1, OUT, 256, 0, 0)


@pytest.mark.parametrize("kw,kind", [
    (dict(eps=-1e-6), "InvalidData"), (dict(eps=float("nan")), "InvalidData"), (dict(eps=float("inf")), "InvalidData"),
    (dict(gq=G + 4), "InvalidData"), (dict(gk=G + 8), "InvalidData"), (dict(q=0), "DeviceError"), (dict(qs=252), "ShapeMismatch"),
    (dict(qo=Q + 64), "InvalidData"), (dict(qo=K), "InvalidData"), (dict(ks=64), "ShapeMismatch"), (dict(v=V + 4), "InvalidData"),
    (dict(slots=0), "DeviceError"), (dict(pos=0), "DeviceError"), (dict(sin=0), "DeviceError"), (dict(m=1 << 32), "DeviceError"),
])
@pytest.mark.parametrize("base", [HALF, FOUR])
def test_store_norm_refusals(rq, base, kw, kind):
    with pytest.raises(getattr(rq, kind)):
        store(pool(base), **kw)


def copy(src, dst, f=INTS, t=INTS, n=3):
    A.copy_pages_dev(src, dst, f, t, n, 0)


def test_copy_refusals(rq):
    a, b = pool(), pool(HALF)
    for src, dst, kind in (([a], [pool(HALF, head_dim=32)], "ShapeMismatch"),
                           ([a], [pool(HALF, page_positions=32)], "ShapeMismatch"),
                           ([a], [pool(HALF, n_kv_heads=1)], "ShapeMismatch"),
                           ([a, pool(n_pages=3)], [b, b], "InvalidData"), ([a, a], [b, a], "InvalidData"),
                           ([b, pool(HALF, page_stride=3 * 64 * 64)], [a, a], "InvalidData")):
        with pytest.raises(getattr(rq, kind)):
            copy(src, dst)
    for f, t in ((0, INTS), (INTS, 0)):
        with pytest.raises(rq.DeviceError) as e:
            copy([a], [b], f or None, t or None)
        assert e.value.status == rq.ERR_NULL_POINTER
    with pytest.raises(rq.DeviceError):
        copy([a], [b], n=1 << 32)
    with pytest.raises(ValueError):
        copy([a], [a, a])
    assert rq.lib.rdl_kv_copy_pages_dev(None, None, 1, INTS, INTS, 1, None) == rq.ERR_NULL_POINTER


def test_empty_calls_need_no_device(rq):
    store(pool(), m=0)
    copy([pool()], [pool(HALF)], n=0)
    copy([], [], n=5)
    L.logprobs_dev(Q, 100, 0, 100, INTS, OUT, OUT, 0, 0, 0, 0)


@pytest.mark.parametrize("page", [0, 8, 24, 2048])
def test_fork_page_refusals(rq, page):
    with pytest.raises(rq.DeviceError) as e:
        A.fork_dev(INTS, 4, INTS, 3, page, INTS, INTS, 2, INTS, 5, INTS, INTS, INTS, 0)
    assert e.value.status == rq.ERR_UNSUPPORTED


@pytest.mark.parametrize("at", [0, 2, 5, 6, 8, 10, 11, 12])
def test_fork_null_pointers(rq, at):
    args = [INTS, 4, INTS, 3, 64, INTS, INTS, 2, INTS, 5, INTS, INTS, INTS]
    args[at] = None
    with pytest.raises(rq.DeviceError) as e:
        A.fork_dev(*args, 0)
    assert e.value.status == rq.ERR_NULL_POINTER


@pytest.mark.parametrize("at", [1, 3, 7, 9])
def test_fork_sizes(rq, at):
    args = [INTS, 4, INTS, 3, 64, INTS, INTS, 2, INTS, 5, INTS, INTS, INTS]
    args[at] = 1 << 40
    with pytest.raises(rq.DeviceError) as e:
        A.fork_dev(*args, 0)
    assert e.value.status == rq.ERR_UNSUPPORTED


@pytest.mark.parametrize("kw,kind", [
    (dict(vocab=0), "DeviceError"), (dict(vocab=1 << 29, stride=1 << 29), "DeviceError"), (dict(stride=99), "ShapeMismatch"),
    (dict(top=65), "DeviceError"), (dict(top=3, vocab=2), "DeviceError"), (dict(m=1 << 24), "DeviceError"),
    (dict(stride=1 << 33), "DeviceError"), (dict(tokens=0), "DeviceError"), (dict(lp=0), "DeviceError"),
    (dict(ids=0), "DeviceError"), (dict(tl=0), "DeviceError"), (dict(x=0), "DeviceError"), (dict(x=Q + 2), "InvalidData"),
])
def test_logprobs_refusals(rq, kw, kind):
    a = {**dict(x=Q, stride=100, m=2, vocab=100, tokens=INTS, lp=OUT, en=OUT, top=5, ids=INTS, tl=OUT), **kw}
    with pytest.raises(getattr(rq, kind)):
        L.logprobs_dev(a["x"] or None, a["stride"], a["m"], a["vocab"], a["tokens"], a["lp"], a["en"], a["top"], a["ids"], a["tl"], 0)
