"""GPU parity of rqmv_block_norm against oracle/paged.py.

Bars, in roundings of 2^-24: a sum of squares takes at most 32 additions in a thread, 6 in a wave and 16 of
waves, all of one sign, and the mean, the root and its reciprocal 4: a factor of a row is off by
(54 / 2 + 5) = 32. f = factor * weight * scale * gate: 4 more, so f d is off by 36 of itself and u by that
and 1 of itself. out is off by what u is, by what this does to the root mean square (its own root mean square, relative),
and by 32 + 3 of itself; fp16 outputs by half a step (2^-11 relative, 2^-25 at least).
"""
import numpy as np
import pytest

from oracle import paged as ref

pytestmark = pytest.mark.gpu
R = 2.0 ** -24


def wide(gpu, a, pad, fill=3.0):
    """Rows with `pad` values between them; (buffer, stride)."""
    rows, n = a.shape
    h = np.full((rows, n + pad), fill, a.dtype)
    h[:, :n] = a
    return gpu.DeviceBuffer.from_array(h), n + pad


def run(gpu, x, delta=None, post=None, gate=None, scale=1.0, pre=None, eps=1e-6, f16=False, u_too=True, in_place=False,
        pad=0, stream=None):
    rows, n = x.shape
    X, ldx = wide(gpu, x, pad)
    kw = {"ldx": ldx, "scale": scale, "eps": eps, "stream": stream}
    if delta is not None:
        kw["delta"], kw["ldd"] = wide(gpu, delta, 2 * pad)
    for name, w in (("post_norm", post), ("pre_norm", pre)):
        if w is not None:
            kw[name] = gpu.DeviceBuffer.from_array(w)
    if gate is not None:
        kw["gate"], ldg = wide(gpu, gate, pad)
        kw["ldg"] = 0 if len(gate) == 1 else ldg
    if u_too:
        U, kw["ldxo"] = (X, ldx) if in_place else wide(gpu, np.full_like(x, 7), pad, 7)
        kw["x_out"] = U
    if pre is not None:
        dt = np.float16 if f16 else np.float32
        O, kw["ldo"] = wide(gpu, np.full((rows, n), 7, dt), 2 * pad, 7)
        kw["out"], kw["out_dtype"] = O, gpu.DTYPE_F16 if f16 else gpu.DTYPE_F32
    gpu.block_norm(X, rows, n, **kw)
    gpu.synchronize()
    u = out = None
    if u_too:
        u = U.download(np.float32).reshape(rows, -1)
        assert np.all(u[:, n:] == (3 if in_place else 7))
        u = u[:, :n].astype(np.float64)
    if pre is not None:
        out = O.download(np.uint16 if f16 else np.uint32).view(dt).reshape(rows, -1)
        assert np.all(out[:, n:] == 7)
        out = out[:, :n].astype(np.float64)
    return u, out


def check(gpu, x, delta=None, post=None, gate=None, scale=1.0, pre=None, eps=1e-6, f16=False, **kw):
    got_u, got = run(gpu, x, delta, post, gate, scale, pre, eps, f16, **kw)
    eps = float(np.float32(eps))
    scale = float(np.float32(scale))
    u, out = ref.block_norm(x, delta, post, gate, scale, pre, eps)
    off = 36 * R * np.abs(u - x) + R * np.abs(u)
    if got_u is not None:
        assert np.all(np.abs(got_u - u) <= off)
    if pre is not None:
        r = 1 / np.sqrt((u ** 2).mean(-1, keepdims=True) + eps)
        bar = np.abs(pre) * r * (off + np.abs(u) * np.sqrt((off ** 2).mean(-1, keepdims=True)) * r) + 35 * R * np.abs(out)
        if f16:
            bar = bar + np.maximum(np.abs(out) * 2.0 ** -11, 2.0 ** -25)
        assert np.all(np.abs(got - out) <= bar * 1.01)


def inputs(rows, n, seed=0):
    rng = np.random.default_rng(seed + n)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    return (f(rows, n) * 3, f(rows, n) * np.float32(0.5), 1 + f(n) * np.float32(0.2), 1 + f(n) * np.float32(0.2), rng)


@pytest.mark.parametrize("n", [4, 64, 252, 256, 260, 1024, 1028, 2880, 4096, 4100, 5120, 8192, 8196, 16384, 16388, 32768])
@pytest.mark.parametrize("rows", [1, 3, 70])
@pytest.mark.parametrize("f16", [False, True])
def test_sizes(gpu, n, rows, f16):
    x, d, post, pre, rng = inputs(rows, n)
    gate = np.tanh(rng.standard_normal((1, n))).astype(np.float32)
    check(gpu, x, d, post, gate, 0.22, pre, f16=f16)


@pytest.mark.parametrize("rows,n", [(1100, 4096), (1101, 8192), (1100, 1028), (1100, 5120), (2050, 256), (5000, 64)])
@pytest.mark.parametrize("f16", [False, True])
def test_many_rows(gpu, rows, n, f16):
    x, d, post, pre, rng = inputs(rows, n, 1)
    check(gpu, x, d, post, None, 1.0, pre, f16=f16)


@pytest.mark.parametrize("n", [128, 4096, 9000])
@pytest.mark.parametrize("has_post", [False, True])
@pytest.mark.parametrize("gates", [0, 1, 5])
@pytest.mark.parametrize("has_pre", [False, True])
def test_parts(gpu, n, has_post, gates, has_pre):
    """Each norm, gate and output with and without the others, rows with gaps between them."""
    x, d, post, pre, rng = inputs(5, n, 2)
    gate = rng.standard_normal((gates, n)).astype(np.float32) if gates else None
    kw = dict(post=post if has_post else None, gate=gate, scale=-1.5, pre=pre if has_pre else None, pad=8)
    check(gpu, x, d, **kw)
    check(gpu, x, d, in_place=True, **kw)
    if has_pre:
        check(gpu, x, d, u_too=False, f16=True, **kw)


@pytest.mark.parametrize("rows,n", [(1, 4096), (9, 260)])
def test_without_a_block(gpu, rows, n):
    x, _, _, pre, _ = inputs(rows, n, 3)
    check(gpu, x, pre=pre, u_too=False)
    check(gpu, x, pre=pre, eps=0.5)


def test_zeros_and_sizes_of_rows(gpu):
    x, d, post, pre, _ = inputs(6, 512, 4)
    x[0], d[0] = 0, 0
    x[1], d[1] = x[1] * np.float32(1e15), d[1] * np.float32(1e15)
    x[2], d[2] = x[2] * np.float32(1e-15), d[2] * np.float32(1e-15)
    d[3] = 0
    x[4] = 0
    check(gpu, x, d, post, None, 1.0, pre, eps=1e-6)
    u, out = run(gpu, x, d, post, None, 1.0, pre, eps=1e-6)
    assert not u[0].any() and not out[0].any()


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("n", [64, 1000, 4096, 20000])
def test_non_finite_values_stay_in_their_row(gpu, bad, n):
    x, d, post, pre, _ = inputs(7, n, 5)
    clean = run(gpu, x, d, post, None, 1.0, pre)
    x[2, n // 2] = bad
    d[5, 3] = bad
    got = run(gpu, x, d, post, None, 1.0, pre)
    rest = [0, 1, 3, 4, 6]
    for a, b in zip(got, clean):
        assert np.array_equal(a[rest], b[rest])
        assert not np.isfinite(a[2]).all() and not np.isfinite(a[5]).all()


def test_one_row_is_add_rmsnorm(gpu):
    x, d, _, pre, _ = inputs(1, 4096, 6)
    X, D, W, O = (gpu.DeviceBuffer.from_array(a) for a in (x, d, pre, x))
    gpu.add_rmsnorm(X, D, W, 4096, 1e-6, O)
    gpu.synchronize()
    u, out = run(gpu, x, d, None, None, 1.0, pre, 1e-6)
    assert np.array_equal(X.download(np.float32).astype(np.float64), u[0])
    assert np.all(np.abs(O.download(np.float32) - out[0]) <= 2 * 40 * R * np.abs(out[0]))


def test_replayed_from_a_graph(gpu):
    rows, n = 33, 5120
    x, d, post, pre, rng = inputs(rows, n, 7)
    bufs = [gpu.DeviceBuffer.from_array(a) for a in (x, d, post, pre)]
    O, stream = gpu.DeviceBuffer(4 * rows * n), gpu.Stream()
    gpu.synchronize()
    graph = gpu.Graph(stream, lambda: gpu.block_norm(bufs[0], rows, n, delta=bufs[1], post_norm=bufs[2], pre_norm=bufs[3],
                                                     scale=0.5, eps=1e-6, x_out=bufs[0], out=O, stream=stream))
    for _ in range(3):  # the residual stream goes on in place
        graph.launch(stream)
        stream.synchronize()
        u, out = run(gpu, x, d, post, None, 0.5, pre)
        assert np.array_equal(bufs[0].download(np.float32).reshape(rows, n), u)
        assert np.array_equal(O.download(np.float32).reshape(rows, n), out)
        x = u.astype(np.float32)
    graph.close()
