"""The several-sequence operators' refusals (include/rdl_attention.h): bad
arguments end in the documented status before anything is launched, so no
device is needed."""
import ctypes as C

import pytest

from rdlquant import attention as A

GOOD = dict(k_dev=1 << 20, v_dev=1 << 21, dtype=1, n_pages=4, page_positions=64, n_kv_heads=2, head_dim=64,
            page_stride=2 * 64 * 64, head_stride=64 * 64, position_stride=64)
Q, K, V, OUT, INTS = 1 << 22, 1 << 23, 1 << 24, 1 << 25, 1 << 26  # addresses nothing reads


def pool(**kw):
    return A.KvPool(*[{**GOOD, **kw}[n] for n, _ in A.KvPool._fields_])


def store(p, m=4, q=Q, qs=256, qo=OUT, qos=256, heads=4, k=K, ks=128, v=V, vs=128, pos=INTS, slots=INTS, cos=INTS,
          sin=INTS, n=10):
    A.store_dev(p, m, q, qs, qo, qos, heads, k, ks, v, vs, pos, slots, cos, sin, n, 0)


def paged(p, q=Q, qs=256, heads=4, m=4, rs=INTS, kv=INTS, n_seq=2, tables=INTS, width=4, scale=0.125, out=OUT,
          os=256):
    A.attention_paged_dev(p, q, qs, heads, m, rs, kv, n_seq, tables, width, scale, out, os, 0, 0, 0)


def packed(q=Q, qs=256, heads=4, k=K, ks=128, v=V, vs=128, dtype=0, kvh=2, hd=64, m=4, rs=INTS, n_seq=2, scale=0.125,
           out=OUT, os=256):
    A.attention_packed_dev(q, qs, heads, k, ks, v, vs, dtype, kvh, hd, m, rs, n_seq, scale, out, os, 0, 0)


@pytest.mark.parametrize("change,kind", [
    (dict(dtype=2), "DTypeMismatch"), (dict(page_positions=8), "DeviceError"),
    (dict(page_positions=48), "DeviceError"), (dict(page_positions=2048), "DeviceError"),
    (dict(page_positions=-64), "DeviceError"), (dict(head_dim=0), "DeviceError"), (dict(head_dim=-64), "DeviceError"),
    (dict(head_dim=60), "DeviceError"), (dict(head_dim=264), "DeviceError"), (dict(n_kv_heads=0), "InvalidData"),
    (dict(n_pages=-1), "InvalidData"), (dict(k_dev=0), "DeviceError"), (dict(v_dev=8), "InvalidData"),
    (dict(position_stride=68), "InvalidData"), (dict(position_stride=56), "ShapeMismatch"),
    (dict(head_stride=64 * 64 - 8), "ShapeMismatch"), (dict(page_stride=64 * 64), "ShapeMismatch"),
    (dict(page_stride=-2 * 64 * 64), "ShapeMismatch"), (dict(page_stride=1 << 62), "ShapeMismatch"),
])
def test_pool_refusals(rq, change, kind):
    with pytest.raises(getattr(rq, kind)):
        store(pool(**change))
    with pytest.raises(getattr(rq, kind)):
        paged(pool(**change))


def test_null_pool_is_an_error(rq):
    assert rq.lib.rdl_kv_store_dev(None, 1, Q, 256, OUT, 256, 4, K, 128, V, 128, INTS, INTS, None, None, 0,
                                   None) == rq.ERR_NULL_POINTER


@pytest.mark.parametrize("kw,kind", [
    (dict(q=0), "DeviceError"), (dict(qs=252), "ShapeMismatch"), (dict(qs=258), "InvalidData"),
    (dict(q=Q + 4), "InvalidData"), (dict(qo=Q + 64), "InvalidData"), (dict(qo=Q, qos=260), "InvalidData"),
    (dict(ks=124), "ShapeMismatch"), (dict(v=0), "DeviceError"), (dict(vs=130), "InvalidData"),
    (dict(slots=0), "DeviceError"), (dict(pos=0), "DeviceError"), (dict(sin=0), "DeviceError"),
    (dict(cos=0), "DeviceError"), (dict(cos=INTS + 8), "InvalidData"), (dict(heads=1 << 20), "DeviceError"),
    (dict(m=1 << 32), "DeviceError"), (dict(qs=1 << 60), "DeviceError"),
])
def test_store_refusals(rq, kw, kind):
    with pytest.raises(getattr(rq, kind)):
        store(pool(), **kw)


@pytest.mark.parametrize("kw,kind", [
    (dict(heads=3), "InvalidData"), (dict(heads=0), "InvalidData"), (dict(scale=0.0), "InvalidData"),
    (dict(scale=-1.0), "InvalidData"), (dict(scale=float("nan")), "InvalidData"),
    (dict(scale=float("inf")), "InvalidData"), (dict(q=0), "DeviceError"), (dict(qs=128), "ShapeMismatch"),
    (dict(os=254), "ShapeMismatch"), (dict(os=257), "InvalidData"), (dict(out=OUT + 8), "InvalidData"),
    (dict(out=Q), "InvalidData"), (dict(out=Q + 512), "InvalidData"), (dict(rs=0), "DeviceError"),
    (dict(n_seq=1 << 30), "DeviceError"), (dict(m=1 << 40), "DeviceError"),
])
def test_attention_refusals(rq, kw, kind):
    with pytest.raises(getattr(rq, kind)):
        paged(pool(), **kw)
    with pytest.raises(getattr(rq, kind)):
        packed(**kw)


@pytest.mark.parametrize("kw,kind", [(dict(kv=0), "DeviceError"), (dict(tables=0), "DeviceError"),
                                     (dict(width=1 << 31), "DeviceError")])
def test_paged_refusals(rq, kw, kind):
    with pytest.raises(getattr(rq, kind)):
        paged(pool(), **kw)


@pytest.mark.parametrize("kw,kind", [
    (dict(dtype=3), "DTypeMismatch"), (dict(hd=12), "DeviceError"), (dict(kvh=0), "InvalidData"),
    (dict(k=0), "DeviceError"), (dict(ks=64), "ShapeMismatch"), (dict(vs=132, dtype=1), "InvalidData"),
    (dict(v=V + 4), "InvalidData"),
])
def test_packed_refusals(rq, kw, kind):
    with pytest.raises(getattr(rq, kind)):
        packed(**kw)


@pytest.mark.parametrize("page", [0, 1, 8, 24, 63, 2048])
def test_plan_page_refusals(rq, page):
    with pytest.raises(rq.DeviceError) as e:
        A.plan_dev(INTS, INTS, 1, INTS, 1, page, INTS, 1, INTS, INTS, 1, INTS, INTS, INTS, INTS, 0)
    assert e.value.status == rq.ERR_UNSUPPORTED


@pytest.mark.parametrize("missing", [0, 1, 3, 6, 8, 9, 11, 12, 13, 14])
def test_plan_null_pointers(rq, missing):
    args = [INTS, INTS, 2, INTS, 3, 64, INTS, 4, INTS, INTS, 5, INTS, INTS, INTS, INTS]
    args[missing] = None
    with pytest.raises(rq.DeviceError) as e:
        A.plan_dev(*args, 0)
    assert e.value.status == rq.ERR_NULL_POINTER


def test_empty_calls_need_no_device(rq):
    store(pool(), m=0)
    paged(pool(), m=0)
    paged(pool(), n_seq=0)
    packed(m=0)
    packed(n_seq=0)


def test_columns_of_the_same_rows_do_not_overlap(rq):
    # q and out as two parts of the same row buffer pass the overlap check (and then reach the null check)
    with pytest.raises(rq.DeviceError) as e:
        paged(pool(), q=Q, qs=512, out=Q + 1024, os=512, rs=0)
    assert e.value.status == rq.ERR_NULL_POINTER
    with pytest.raises(rq.InvalidData):
        paged(pool(), q=Q, qs=512, out=Q + 1008, os=512, rs=0)
    assert C.sizeof(A.KvPool) == 64


@pytest.mark.parametrize("n_seq,kvh,m", [(1 << 24, 1, 1 << 24), (1 << 23, 2, 1 << 23), (1 << 24, 2, 8), (1 << 22, 16, 1 << 22)])
def test_more_workgroups_than_a_launch_has(rq, n_seq, kvh, m):
    far = dict(q=1 << 40, out=1 << 50)
    w = kvh * 8
    one = pool(n_kv_heads=kvh, head_dim=8, position_stride=8, head_stride=512, page_stride=512 * kvh)
    for call in (lambda: paged(one, qs=w, os=w, heads=kvh, m=m, n_seq=n_seq, **far),
                 lambda: A.attention_paged_dev(one, far["q"], w, kvh, m, INTS, INTS, n_seq, INTS, 4, 0.1, far["out"], w, 1,
                                               4, 0),
                 lambda: packed(qs=w, os=w, heads=kvh, ks=w, vs=w, kvh=kvh, hd=8, m=m, n_seq=n_seq, **far)):
        with pytest.raises(rq.DeviceError) as e:
            call()
        assert e.value.status == rq.ERR_UNSUPPORTED, e.value


@pytest.mark.parametrize("kw", [dict(qo=K), dict(qo=V + 16), dict(qo=K - 256 * 4 * 4 + 16), dict(k=OUT + 512),
                                dict(q=Q, qs=512, qo=Q, qos=512, k=Q + 1008, ks=512),
                                dict(q=Q, qs=512, qo=Q, qos=512, k=Q + 1024, ks=512, v=Q + 1008, vs=512)])
def test_store_refuses_q_out_over_k_or_v(rq, kw):
    with pytest.raises(rq.InvalidData) as e:
        store(pool(), **kw)
    assert "q_out overlaps k or v" in str(e.value)


def test_store_takes_parts_of_the_same_rows(rq):
    # q in place, k and v behind it in rows of one stride: past the overlap checks, up to the null check
    with pytest.raises(rq.DeviceError) as e:
        store(pool(), q=Q, qs=512, qo=Q, qos=512, k=Q + 1024, ks=512, v=Q + 1536, vs=512, slots=0)
    assert e.value.status == rq.ERR_NULL_POINTER
    with pytest.raises(rq.DeviceError) as e:
        store(pool(), heads=0, q=0, qo=K, slots=0)  # no q: no q_out
    assert e.value.status == rq.ERR_NULL_POINTER


@pytest.mark.parametrize("kw", [dict(out=K), dict(out=V + 16), dict(out=K, dtype=1, ks=512), dict(k=OUT + 512),
                                dict(q=Q, qs=1024, out=Q + 1024, os=1024, k=Q + 2032, ks=1024)])
def test_packed_refuses_out_over_k_or_v(rq, kw):
    with pytest.raises(rq.InvalidData) as e:
        packed(**kw)
    assert "out overlaps k or v" in str(e.value)
