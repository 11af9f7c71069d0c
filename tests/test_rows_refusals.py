"""What rqmv_logprobs and rqmv_block_norm refuse, before anything is launched
(no GPU needed: every call here returns RQMV_EINVAL from its checks)."""
import pytest

import rqmv
from tests.test_paged_refusals import A, At, refused


@pytest.mark.parametrize("kw", [
    dict(logits=At(None)), dict(tokens=None), dict(logprob=None), dict(rows=0), dict(rows=-1), dict(rows=(1 << 20) + 1),
    dict(n=0), dict(n=(1 << 20) + 1), dict(ld=99), dict(ld=1 << 41), dict(top=-1), dict(top=33), dict(top=101, n=100),
    dict(top=5, n=4, ld=4), dict(top_tokens=None, top_logprobs=None),
    dict(tokens=None, logprob=None, entropy=None, top=0)])
def test_logprobs(kw):
    a = dict(logits=A, rows=2, n=100, ld=100, tokens=A, logprob=A, entropy=A, top=3, top_tokens=A, top_logprobs=A, workspace=A)
    a.update(kw)
    refused(rqmv.logprobs, **a)
    if set(kw) & {"rows", "n", "top"} and "tokens" not in kw:
        refused(rqmv.logprobs_workspace_size, a["rows"], a["n"], a["top"])


X, D, G, P, Q, U, O = (At(k << 24) for k in range(1, 8))


def norm(**kw):
    a = dict(x=X, rows=3, n=64, delta=D, post_norm=P, gate=G, pre_norm=Q, x_out=U, out=O)
    a.update(kw)
    rqmv.block_norm(**a)


@pytest.mark.parametrize("kw", [
    dict(x=At(None)), dict(x_out=None, out=None, pre_norm=None), dict(out=None), dict(pre_norm=None), dict(delta=None),
    dict(delta=None, gate=None), dict(delta=None, post_norm=None), dict(rows=0), dict(rows=(1 << 20) + 1), dict(n=0),
    dict(n=62), dict(n=32772), dict(n=-4), dict(out_dtype=2), dict(eps=-1.0), dict(eps=float("nan")),
    dict(scale=float("nan")), dict(ldx=60), dict(ldd=66), dict(ldg=60), dict(ldxo=62), dict(ldo=63), dict(out_dtype=1, ldo=66),
    dict(ldx=1 << 41), dict(x=At(X.ptr + 4)), dict(delta=At(8)), dict(gate=At(4)), dict(post_norm=At(12)),
    dict(pre_norm=At(20)), dict(x_out=At(24)), dict(out=At(8))])
def test_block_norm(kw):
    refused(norm, **kw)


@pytest.mark.parametrize("kw", [
    dict(x_out=At(X.ptr + 256)), dict(x_out=X, ldxo=128), dict(x_out=D), dict(out=X), dict(out=D), dict(out=U),
    dict(out=At(U.ptr + 2 * 256 + 240)), dict(out=At(P.ptr - 2 * 256)), dict(x_out=G), dict(out=Q), dict(x_out=At(D.ptr - 256)),
    dict(out=At(G.ptr + 2 * 64 * 4), ldg=64)])
def test_block_norm_refuses_overlapping_outputs(kw):
    refused(norm, **kw)


def test_the_last_error_names_the_call():
    with pytest.raises(rqmv.RqmvError, match="block_norm: rows must be 1"):
        norm(rows=0)
    with pytest.raises(rqmv.RqmvError, match="logprobs: top must be 0..32"):
        rqmv.logprobs_workspace_size(1, 100, 40)
