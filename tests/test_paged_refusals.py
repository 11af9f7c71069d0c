"""What the paged serving entry points refuse, before anything is launched (no
GPU needed: every call here returns RQMV_EINVAL from its checks)."""
import numpy as np
import pytest

import rqmv


class At:
    """Stands for a device address; nothing is read through it."""

    def __init__(self, ptr=1 << 20, nbytes=1 << 30):
        self.ptr, self.nbytes = ptr, nbytes


A = At()


def batch(seqs=2, tokens=4, max_blocks=3, stride=None, **none):
    names = ("q_start", "kv_len", "block_table", "positions", "slots")
    return rqmv.PagedBatch(seqs, tokens, max_blocks, table_stride=stride,
                           **{n: none.get(n, A) for n in names})


def cache(blocks=10, block=16, kv=2, hd=64, k=A, v=A):
    return rqmv.PagedCache(k, v, blocks, block, kv, hd)


BAD_CACHES = [dict(block=8), dict(block=48), dict(block=512), dict(block=0), dict(blocks=0), dict(blocks=-1),
              dict(blocks=1 << 27)]
BAD_BATCHES = [dict(seqs=0), dict(seqs=8193), dict(tokens=0), dict(tokens=(1 << 20) + 1)]
BAD_TABLES = [dict(max_blocks=0), dict(max_blocks=5, stride=4), dict(stride=1 << 41), dict(max_blocks=(1 << 26) + 1)]


def refused(call, *args, **kw):
    with pytest.raises(rqmv.RqmvError, match=r"\(-1\)"):
        call(*args, **kw)


def plan(b=None, c=None, **kw):
    a = dict(cached_len=A, new_len=A, free_list=A, free_count=3, free_head=A, free_head_out=A, status=A)
    a.update(kw)
    rqmv.paged_plan(b or batch(), c or cache(), **a)


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_plan_refuses_caches(kw):
    refused(plan, c=cache(**kw))


@pytest.mark.parametrize("kw", BAD_BATCHES + BAD_TABLES)
def test_plan_refuses_batches(kw):
    refused(plan, b=batch(**kw))


@pytest.mark.parametrize("name", ["q_start", "kv_len", "block_table", "positions", "slots"])
def test_plan_refuses_missing_tables(name):
    refused(plan, b=batch(**{name: None}))


@pytest.mark.parametrize("kw", [dict(cached_len=At(None)), dict(new_len=At(None)), dict(free_head=At(None)),
                                dict(free_head_out=At(None)), dict(status=At(None)), dict(free_list=None),
                                dict(free_count=-1)])
def test_plan_refuses_arguments(kw):
    refused(plan, **kw)


def qk(b=None, c=None, **kw):
    a = dict(qkv=At(1 << 24), x_dtype=0, ld=512, q_heads=4, table=A, rope_rows=8, q_out=At(1 << 30), q_dtype=0, ldq=256)
    a.update(kw)
    rqmv.qk_norm_rope(b or batch(), c or cache(), **a)


@pytest.mark.parametrize("kw", BAD_CACHES + [dict(kv=0), dict(kv=1025), dict(hd=32), dict(hd=96), dict(k=None),
                                             dict(v=None), dict(k=At(8)), dict(v=At(24))])
def test_qk_norm_rope_refuses_caches(kw):
    refused(qk, c=cache(**kw))


@pytest.mark.parametrize("kw", BAD_BATCHES + [dict(positions=None), dict(slots=None)])
def test_qk_norm_rope_refuses_batches(kw):
    refused(qk, b=batch(**kw))


@pytest.mark.parametrize("kw", [
    dict(x_dtype=2), dict(q_dtype=-1), dict(ld=508), dict(ld=514), dict(ldq=252), dict(ldq=258), dict(ld=1 << 41),
    dict(x_dtype=1, ld=516), dict(q_heads=0), dict(q_heads=1025), dict(rope_rows=0), dict(rot_dim=0), dict(rot_dim=12),
    dict(rot_dim=72), dict(q_norm=A), dict(k_norm=A), dict(q_norm=A, k_norm=At(8)), dict(q_norm=A, k_norm=A, eps=-1.0),
    dict(q_norm=A, k_norm=A, eps=float("nan")), dict(table=At(4)), dict(qkv=At(20)), dict(q_out=At(40)),
    dict(qkv=At(None)), dict(q_out=At(None)), dict(table=At(None)),
    # q_out inside qkv's span, or qkv itself with another type or stride
    dict(q_out=At((1 << 24) + 1024)), dict(q_out=At(1 << 24), q_dtype=1), dict(q_out=At(1 << 24))])
def test_qk_norm_rope_refuses_arguments(kw):
    refused(qk, **kw)


def test_the_last_error_names_the_call():
    with pytest.raises(rqmv.RqmvError, match="paged_plan: block_size must be"):
        plan(c=cache(block=24))
    with pytest.raises(rqmv.RqmvError, match="qk_norm_rope: batch is NULL"):
        rqmv._check(rqmv.lib().lib.rqmv_qk_norm_rope(None, rqmv.byref(cache().struct), *([None, 0, 0, 0, None, None, 0.0,
                                                     None, 0, 0, None, 0, 0, None])), "rqmv_qk_norm_rope")
    assert np.int32(rqmv.PLAN_LENGTH | rqmv.PLAN_TOKENS | rqmv.PLAN_POOL) == 7


def attend(b=None, c=None, **kw):
    a = dict(q=A, dtype=0, ldq=256, q_heads=4, out=A, ldo=256, workspace=A)
    a.update(kw)
    rqmv.paged_attention(b or batch(), c or cache(), **a)


@pytest.mark.parametrize("kw", BAD_CACHES + [dict(kv=0), dict(hd=32), dict(hd=96), dict(k=None), dict(v=At(24))])
def test_paged_attention_refuses_caches(kw):
    refused(attend, c=cache(**kw))
    refused(rqmv.paged_attention_workspace_size, batch(), cache(**kw), 4)


@pytest.mark.parametrize("kw", BAD_BATCHES + BAD_TABLES)
def test_paged_attention_refuses_batches(kw):
    refused(attend, b=batch(**kw))
    refused(rqmv.paged_attention_workspace_size, batch(**kw), cache(), 4)


@pytest.mark.parametrize("kw", [
    dict(q=At(None)), dict(out=At(None)), dict(dtype=2), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
    dict(scale=float("inf")), dict(window=-1), dict(q_heads=3), dict(q_heads=0), dict(q_heads=1026)])
def test_paged_attention_refuses_arguments(kw):
    refused(attend, **kw)


@pytest.mark.parametrize("kw", [dict(out=At(A.ptr + 512)), dict(q=At(A.ptr + 16)), dict(ldo=512), dict(dtype=1, ldq=512)])
def test_paged_attention_refuses_overlapping_outputs(kw):
    refused(attend, **kw)


def test_paged_attention_refuses_grids_it_cannot_launch():
    refused(attend, b=batch(tokens=1 << 20), q_heads=512, ldq=512 * 64, ldo=512 * 64)
    refused(rqmv.paged_attention_workspace_size, batch(tokens=1 << 20, seqs=8192), cache(kv=1024), 1024)


def test_a_call_without_a_device_is_an_error():
    """Past the checks of its arguments the call needs a device that rqmv_init has prepared."""
    import subprocess
    import sys

    code = ("import sys; sys.path[:0] = %r\n"
            "import rqmv, tests.test_paged_refusals as t\n"
            "try:\n    rqmv.paged_attention_workspace_size(t.batch(), t.cache(), 4)\n"
            "except rqmv.RqmvError as e:\n    print('raised', e)\n" % sys.path)
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=120,
                         env={**__import__("os").environ, "HIP_VISIBLE_DEVICES": ""})
    assert "raised" in out.stdout and "(-1)" not in out.stdout, out.stdout + out.stderr


@pytest.mark.parametrize("kw", [dict(logits=At(None)), dict(u=At(None)), dict(tokens=At(None)), dict(rows=0),
                                dict(rows=(1 << 20) + 1), dict(n=0), dict(n=(1 << 20) + 1), dict(ld=99), dict(rows=-1),
                                dict(ld=1 << 41)])
def test_sample_refuses_arguments(kw):
    a = dict(logits=A, rows=2, n=100, ld=100, u=A, tokens=A, workspace=A)
    a.update(kw)
    refused(rqmv.sample, **a)
    if set(kw) & {"rows", "n"}:
        refused(rqmv.sample_workspace_size, a["rows"], a["n"])


@pytest.mark.parametrize("name", ["q_start", "kv_len", "block_table", "positions", "slots"])
def test_assigned_buffers_are_what_calls_pass(name):
    b = batch()
    setattr(b, name, None)
    assert getattr(b, name) is None and getattr(b.struct, name) is None
    refused(plan, b=b)
    other = At(1 << 22)
    setattr(b, name, other)
    assert getattr(b, name) is other and getattr(b.struct, name) == 1 << 22


def test_assigned_counts_are_what_calls_pass():
    for name, bad in (("seqs", 8193), ("tokens", 0), ("max_blocks", 1 << 27), ("table_stride", 2)):
        b = batch()
        was = getattr(b, name)
        setattr(b, name, bad)
        assert getattr(b, name) == getattr(b.struct, name) == bad
        refused(plan, b=b)
        setattr(b, name, was)
        assert getattr(b.struct, name) == was
    for name, bad in (("k", None), ("v", At(24)), ("blocks", 0), ("block_size", 24), ("kv_heads", 0), ("head_dim", 96)):
        c = cache()
        setattr(c, name, bad)
        assert getattr(c.struct, name) == (bad if isinstance(bad, int) else rqmv._p(bad))
        refused(attend, c=c)
    assert cache().k is A and batch(stride=7).table_stride == 7 and batch().table_stride == 3
    c = cache()
    with pytest.raises(TypeError):
        c.blocks = 2.5
    assert c.blocks == 10  # as the calls pass it
