"""Norms around a block (ops.block_norm) against the formulas in 64 bits.

Tolerance, from the arithmetic: a mean of n squares summed in 32 bits by t threads errs by at most (n/t + 10) 2^-24
relative, half of that after the root; rsqrt, the sigmoid (|gate| < 8) and the products add less than 2.5e-6.  With at
least 32 values a thread at the widths below that is under 5e-6 of the terms' magnitudes.  A bf16 result adds its
rounding, 2^-9 of the value.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

F32, BF16 = torch.float32, torch.bfloat16
REL = 5e-6


@pytest.fixture()
def dev():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    return torch.device("cuda:0")


def make(rng, shape, dtype, dev, scale=1.0, stride=None):
    v = torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * scale).to(dtype)
    if stride is None:
        return v.to(dev)
    wide = torch.full((shape[0], stride), float("nan"), dtype=dtype)
    wide[:, :shape[1]] = v
    return wide.to(dev)[:, :shape[1]]


def want(y, r, post, nxt, gate, act, eps, off, rs, bs):
    d = lambda t: t.double().cpu()
    u = d(y)
    if post is not None:
        u = u / torch.sqrt((u * u).mean(1, keepdim=True) + eps) * (off + d(post))
    if gate is not None:
        g = d(gate)
        u = u * (1.0 / (1.0 + torch.exp(-g)) if act == "sigmoid" else g)
    u = bs * u
    a = rs * d(r) if r is not None else torch.zeros_like(u)
    h = a + u
    size = a.abs() + u.abs()
    if nxt is None:
        return h, size, None, None
    f = (off + d(nxt)) / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return h, size, h * f, size * f.abs() + (h * f).abs()


def close(got, ref, size):
    err = (got.double().cpu() - ref).abs()
    tol = REL * size + (2.0 ** -8 * ref.abs() if got.dtype == BF16 else 0.0) + 1e-30
    bad = err > tol
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: worst {float((err / tol).max()):.2f} of the tolerance"


def check(dev, m, n, yt=F32, rt=BF16, gt=BF16, wt=BF16, ht=None, zt=BF16, gate="none", act="none", post=True, nxt=True, off=0.0, res=True,
          pad=0, seed=0):
    from weightstream_b200 import ops
    rng = np.random.default_rng(seed + 7 * m + n)
    stride = n + pad if pad else None
    y = make(rng, (m, n), yt, dev, 2.0, stride)
    r = make(rng, (m, n), rt, dev, 3.0, stride) if res else None
    w = [make(rng, (n,), wt, dev, 0.2) + (1.0 - off) if on else None for on in (post, nxt)]
    shape = {"none": None, "channel": (n,), "token": (m, 1), "full": (m, n)}[gate]
    g = make(rng, shape, gt, dev, 1.5, stride if gate == "full" else None) if shape else None
    h, z = ops.block_norm(y, r, post_weight=w[0], next_weight=w[1], gate=g, gate_act=act, eps=1e-5, weight_offset=off, residual_scale=0.75,
                          block_scale=1.5, out_dtype=ht, normed_dtype=zt)
    assert h.dtype == (ht or (rt if res else BF16)) and (z is None) == (not nxt)
    hr, hs, zr, zs = want(y, r, w[0], w[1], g, act, 1e-5, off, 0.75, 1.5)
    close(h, hr, hs)
    if nxt:
        assert z.dtype == zt
        close(z, zr, zs)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 2, 7, 149, 700])
@pytest.mark.parametrize("n", [1, 8, 31, 128, 2304, 2307, 5120, 7168, 16384])
def test_sizes(dev, m, n):
    check(dev, m, n, gate="full" if (m + n) % 2 else "token", act="sigmoid")


@pytest.mark.gpu
@pytest.mark.parametrize("n", [33000, 65543])
def test_wide_rows(dev, n):
    check(dev, 3, n, gate="channel")


@pytest.mark.gpu
@pytest.mark.parametrize("yt", [F32, BF16])
@pytest.mark.parametrize("rt", [F32, BF16])
@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("m", [3, 400])
def test_types_and_gates(dev, yt, rt, gate, m):
    for gt, wt, zt in ((F32, F32, F32), (BF16, F32, BF16), (F32, BF16, F32)):
        check(dev, m, 520, yt=yt, rt=rt, gt=gt, wt=wt, zt=zt, gate=gate, act="sigmoid" if gt == F32 else "none")


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 4, 8, 56])
@pytest.mark.parametrize("m", [5, 333])
def test_strides(dev, pad, m):
    check(dev, m, 1024, pad=pad, gate="full")
    check(dev, m, 1024, yt=BF16, rt=F32, pad=pad, gate="full", zt=F32)


@pytest.mark.gpu
def test_parts_that_are_left_out(dev):
    for m in (2, 300):
        check(dev, m, 512, post=False)
        check(dev, m, 512, nxt=False)
        check(dev, m, 512, post=False, nxt=False)
        check(dev, m, 512, res=False)
        check(dev, m, 512, res=False, ht=F32, off=1.0)
        check(dev, m, 512, ht=F32, rt=BF16)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(4, 7168), (300, 5120), (3, 77)])
def test_in_place_is_the_same(dev, m, n):
    from weightstream_b200 import ops
    rng = np.random.default_rng(3)
    for t in (F32, BF16):
        y, r = make(rng, (m, n), F32, dev), make(rng, (m, n), t, dev)
        w = make(rng, (n,), BF16, dev)
        h, z = ops.block_norm(y, r, post_weight=w, next_weight=w)
        h2, z2 = ops.block_norm(y, r, post_weight=w, next_weight=w, out=r)
        assert h2 is r and torch.equal(h2, h) and torch.equal(z2, z)


@pytest.mark.gpu
def test_zero_rows_and_zero_values(dev):
    from weightstream_b200 import ops
    w = torch.ones(64, dtype=BF16, device=dev)
    h, z = ops.block_norm(torch.zeros((0, 64), device=dev), torch.zeros((0, 64), dtype=BF16, device=dev), next_weight=w)
    assert h.shape == (0, 64) and z.shape == (0, 64)
    h, z = ops.block_norm(torch.zeros((3, 64), device=dev), torch.zeros((3, 64), dtype=BF16, device=dev), post_weight=w, next_weight=w)
    assert not h.any() and not z.any()
    for v in (float("inf"), float("nan")):  # a broken value breaks its own row only
        y = torch.ones((3, 64), device=dev)
        y[1, 5] = v
        h, z = ops.block_norm(y, torch.zeros((3, 64), dtype=BF16, device=dev), next_weight=w)
        assert torch.isfinite(z[0]).all() and torch.isfinite(z[2]).all() and not torch.isfinite(z[1]).all()


@pytest.mark.gpu
def test_another_stream_and_a_graph(dev):
    from weightstream_b200 import ops
    rng = np.random.default_rng(9)
    y, r, w = make(rng, (40, 2048), F32, dev), make(rng, (40, 2048), BF16, dev), make(rng, (2048,), BF16, dev)
    h, z = ops.block_norm(y, r, post_weight=w, next_weight=w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    h2, z2 = ops.block_norm(y, r, post_weight=w, next_weight=w, stream=s)
    s.synchronize()
    assert torch.equal(h, h2) and torch.equal(z, z2)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        h3, z3 = ops.block_norm(y, r, post_weight=w, next_weight=w)
    y.mul_(-1.0)
    g.replay()
    h, z = ops.block_norm(y, r, post_weight=w, next_weight=w)
    torch.cuda.synchronize()
    assert torch.equal(h, h3) and torch.equal(z, z3)


BAD = [
    (ValueError, dict(y=torch.zeros(256))),
    (TypeError, dict(y=torch.zeros((3, 256), dtype=torch.float64))),
    (ValueError, dict(y=torch.zeros((3, 512))[:, ::2])),
    (ValueError, dict(residual=torch.zeros((3, 255)))),
    (ValueError, dict(residual=torch.zeros((1, 256)).expand(3, 256))),
    (ValueError, dict(post_weight=torch.zeros(255))),
    (TypeError, dict(post_weight=torch.zeros(256, dtype=torch.bfloat16))),
    (ValueError, dict(next_weight=torch.zeros(512)[::2])),
    (ValueError, dict(gate=torch.zeros((2, 256)))),
    (ValueError, dict(gate=torch.zeros((3, 512))[:, ::2])),
    (TypeError, dict(gate=torch.zeros((3, 256), dtype=torch.float16))),
    (ValueError, dict(gate=torch.zeros(256), gate_act="relu")),
    (ValueError, dict(eps=-1.0)),
    (ValueError, dict(eps=float("nan"))),
    (TypeError, dict(normed_dtype=torch.float16)),
    (ValueError, dict(out=torch.zeros((3, 128)))),
    (TypeError, dict(out=torch.zeros((3, 256), dtype=torch.int32))),
]


def plain():
    return dict(y=torch.zeros((3, 256)), residual=torch.zeros((3, 256), dtype=torch.bfloat16), post_weight=torch.zeros(256),
                next_weight=torch.zeros(256), gate=None, gate_act="none", eps=1e-6, out=None, normed_dtype=torch.bfloat16)


@pytest.mark.parametrize("error,change", BAD)
def test_refuses(error, change):
    from weightstream_b200 import ops
    rest = dict(weight_offset=0.0, residual_scale=1.0, block_scale=1.0, out_dtype=None)
    ops._block_norm_args(**plain(), **rest)
    with pytest.raises(error):
        ops._block_norm_args(**{**plain(), **change}, **rest)


@pytest.mark.gpu
def test_calls_refuse(dev):
    """The same through the call itself, whose native front end looks first."""
    from weightstream_b200 import ops

    def move(d):  # with the same strides
        put = lambda t: torch.zeros(t.untyped_storage().nbytes() // t.element_size(), dtype=t.dtype, device=dev).as_strided(t.size(), t.stride())
        return {k: put(v) if isinstance(v, torch.Tensor) else v for k, v in d.items()}

    ops.block_norm(**move(plain()))
    for error, change in BAD:
        with pytest.raises(error):
            ops.block_norm(**{**move(plain()), **move(change)})
    with pytest.raises(ValueError):
        ops.block_norm(**plain())  # tensors of the host
    with pytest.raises(ValueError):
        ops.block_norm(**{**move(plain()), "residual": plain()["residual"]})


@pytest.mark.parametrize("n", [2 ** 31 - 1, 2 ** 31 - 4096, 0, -1])
def test_c_entry_refuses_widths_that_its_counters_do_not_hold(n):
    """A row is counted in 32 bits, up to a block's step past its end.  (No rows, so that nothing could be launched.)"""
    import ctypes as C
    from weightstream_b200 import _lib
    L, err = _lib.load(), C.create_string_buffer(256)
    a = _lib.BlockNormArgs(m=0, n=n, eps=1e-6)
    assert L.ws_block_norm(C.byref(a), None, err, len(err)) == _lib.WS_ERR_INVALID and b"out of range" in err.value
    a.n = 2 ** 31 - 4097
    assert L.ws_block_norm(C.byref(a), None, err, len(err)) == _lib.WS_OK


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,pad", [(400, 5121, 0), (400, 5120, 1), (297, 2561, 0), (300, 8191, 0), (3, 8193, 0), (3, 9001, 0), (3, 16383, 0),
                                     (3, 16384, 1), (2, 16385, 0), (3, 16640, 8)])
def test_values_one_by_one_at_every_width(dev, m, n, pad):
    """Rows that no vector fits, with eight, sixteen and thirty-two values a thread and with any number of them."""
    check(dev, m, n, gate="full", act="sigmoid", rt=F32, pad=pad)
    check(dev, m, n, yt=BF16, rt=BF16, gt=F32, wt=F32, ht=F32, zt=F32, gate="channel", pad=pad)
    check(dev, m, n, gate="token", post=False, pad=pad)
    check(dev, m, n, res=False, nxt=False, gate="full", pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n", [(400, 5121), (3, 9001), (3, 16383), (2, 20001)])
def test_values_one_by_one_in_place(dev, m, n):
    from weightstream_b200 import ops
    rng = np.random.default_rng(m + n)
    for t in (F32, BF16):
        y, r, g = make(rng, (m, n), F32, dev), make(rng, (m, n), t, dev), make(rng, (m, n), BF16, dev)
        w = make(rng, (n,), BF16, dev)
        h, z = ops.block_norm(y, r, post_weight=w, next_weight=w, gate=g)
        h2, z2 = ops.block_norm(y, r, post_weight=w, next_weight=w, gate=g, out=r)
        assert h2 is r and torch.equal(h2, h) and torch.equal(z2, z)
