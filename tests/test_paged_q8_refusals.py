"""What the entry points over 8-bit pages refuse, before anything is launched
(no GPU needed: every call here returns RQMV_EINVAL from its checks)."""
import ctypes

import pytest

import rqmv
from tests.test_paged_refusals import A, BAD_BATCHES, BAD_CACHES, BAD_TABLES, At, batch, plan, refused


def cache(blocks=10, block=16, kv=2, hd=64, k=A, v=A, ks=At(3), vs=At(5)):
    return rqmv.PagedCacheQ8(k, v, ks, vs, blocks, block, kv, hd)


SHAPES = [dict(kv=0), dict(hd=32), dict(hd=96), dict(k=None), dict(v=None), dict(k=At(8)), dict(v=At(24)), dict(ks=None),
          dict(vs=None)]


def qk(b=None, c=None, **kw):
    a = dict(qkv=At(1 << 24), x_dtype=0, ld=512, q_heads=4, table=A, rope_rows=8, q_out=At(1 << 30), q_dtype=0, ldq=256)
    a.update(kw)
    rqmv.qk_norm_rope_q8(b or batch(), c or cache(), **a)


def attend(b=None, c=None, **kw):
    a = dict(q=A, dtype=0, ldq=256, q_heads=4, out=A, ldo=256, workspace=A)
    a.update(kw)
    rqmv.paged_attention_q8(b or batch(), c or cache(), **a)


@pytest.mark.parametrize("kw", BAD_CACHES + SHAPES)
def test_caches(kw):
    refused(qk, c=cache(**kw))
    refused(attend, c=cache(**kw))
    refused(rqmv.paged_attention_q8_workspace_size, batch(), cache(**kw), 4)
    refused(rqmv.paged_values_q8, cache(**kw), rqmv.PagedCache(At(1 << 28), At(1 << 29), 10, 16, 2, 64))


@pytest.mark.parametrize("kw", BAD_BATCHES)
def test_batches(kw):
    refused(qk, b=batch(**kw))
    refused(attend, b=batch(**kw))
    refused(rqmv.paged_attention_q8_workspace_size, batch(**kw), cache(), 4)


@pytest.mark.parametrize("kw", BAD_TABLES + [dict(q_start=None), dict(kv_len=None), dict(block_table=None)])
def test_tables(kw):
    refused(attend, b=batch(**kw))


@pytest.mark.parametrize("kw", [dict(positions=None), dict(slots=None)])
def test_missing_rows(kw):
    refused(qk, b=batch(**kw))


@pytest.mark.parametrize("kw", [
    dict(x_dtype=2), dict(q_dtype=-1), dict(ld=508), dict(ld=514), dict(ldq=252), dict(ld=1 << 41), dict(q_heads=0),
    dict(q_heads=1025), dict(rope_rows=0), dict(rot_dim=0), dict(rot_dim=12), dict(rot_dim=72), dict(q_norm=A),
    dict(q_norm=A, k_norm=A, eps=float("nan")), dict(table=At(4)), dict(qkv=At(20)), dict(q_out=At(None)),
    dict(q_out=At((1 << 24) + 1024)), dict(q_out=At(1 << 24), q_dtype=1)])
def test_append_arguments(kw):
    refused(qk, **kw)


@pytest.mark.parametrize("kw", [
    dict(q=At(None)), dict(out=At(None)), dict(dtype=2), dict(scale=0.0), dict(scale=float("nan")), dict(window=-1),
    dict(q_heads=3), dict(q_heads=0), dict(out=At(A.ptr + 512)), dict(ldo=512), dict(ldq=250)])
def test_attention_arguments(kw):
    refused(attend, **kw)


def test_values_arguments():
    big = 10 * 16 * 2 * 64
    k, v, ks, vs = At(1 << 20), At(1 << 21), At(1 << 22), At(1 << 23)
    c = cache(k=k, v=v, ks=ks, vs=vs)

    def to(k=At(1 << 28), v=At(1 << 29), blocks=10, block=16, kv=2, hd=64):
        return rqmv.PagedCache(k, v, blocks, block, kv, hd)

    for kw in (dict(blocks=9), dict(block=32), dict(kv=1), dict(hd=128), dict(k=None), dict(v=At(8)),
               dict(k=k), dict(v=At(v.ptr + big - 16)), dict(k=At(ks.ptr - 2 * big + 16)), dict(v=vs),
               dict(v=At((1 << 28) + 2 * big - 16))):
        refused(rqmv.paged_values_q8, c, to(**kw))


def test_the_last_error_names_the_call():
    with pytest.raises(rqmv.RqmvError, match="paged_attention_q8: block_size must be"):
        attend(c=cache(block=24))
    with pytest.raises(rqmv.RqmvError, match="qk_norm_rope_q8: the scales must not be NULL"):
        qk(c=cache(ks=None))
    with pytest.raises(rqmv.RqmvError, match="qk_norm_rope_q8: cache is NULL"):
        rqmv._check(rqmv.lib().lib.rqmv_qk_norm_rope_q8(batch().ref, None, *([None, 0, 0, 0, None, None, 0.0, None, 0, 0,
                                                        None, 0, 0, None])), "rqmv_qk_norm_rope_q8")


def test_a_plan_takes_these_pages_too():
    """rqmv_paged_cache_q8 begins with its rqmv_paged_cache: a plan reads blocks and block_size through the same
    reference."""
    refused(plan, c=cache(block=24))
    refused(plan, c=cache(blocks=0))
    fields = dict((n, getattr(rqmv._CacheQ8Struct, n).offset) for n, _ in rqmv._CacheQ8Struct._fields_)
    plain = dict((n, getattr(rqmv._CacheStruct, n).offset) for n, _ in rqmv._CacheStruct._fields_)
    assert all(fields[n] == at for n, at in plain.items())
    assert fields["k_scale"] == ctypes.sizeof(rqmv._CacheStruct) and fields["v_scale"] == fields["k_scale"] + 8


def test_assigned_buffers_are_what_calls_pass():
    c = cache()
    c.k_scale = None
    assert c.struct.k_scale is None
    refused(qk, c=c)
    c.k_scale = A
    assert c.struct.k_scale == A.ptr


def test_each_kind_of_pages_has_its_calls():
    """Codes read as fp16 would end past their memory, and fp16 pages have no scales."""
    from tests.test_paged_refusals import attend as attend16, cache as cache16, qk as qk16

    for call, c in ((qk, cache16()), (attend, cache16()), (qk16, cache()), (attend16, cache())):
        with pytest.raises(TypeError, match="pages of"):
            call(c=c)
    for args in ((cache16(), cache16()), (cache(), cache())):
        with pytest.raises(TypeError, match="pages of"):
            rqmv.paged_values_q8(*args)
    with pytest.raises(TypeError):
        rqmv.paged_attention_workspace_size(batch(), cache(), 4)
    with pytest.raises(TypeError):
        rqmv.paged_attention_q8_workspace_size(batch(), cache16(), 4)
