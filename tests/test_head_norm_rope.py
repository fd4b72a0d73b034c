"""Norms of heads with their rotation (ops.head_norm_rope) against the definition in 64 bits.

Tolerance (u = 2^-24): a sum of d squares is added in chains of at most d / 16 + 16 terms and six levels, so mean and its
root err by (d / 16 + 24) / 2 u, the reciprocal root by 4 u more, the products by 3 u: (d / 32 + 19) u relative of a value.
A cosine errs by 2 u of its argument's rounding (half an ulp of at most one half turn: pi 2^-25), 2 ulp of its own and one
rounding with the scale: 8 u; a' = a cos - b sin adds two roundings.  The 64-bit angle adds 2 u up to positions of 2^31.
Then the result's own rounding.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


@pytest.fixture()
def dev():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    return torch.device("cuda:0")


def made(rng, shape, dtype, dev, scale=1.0):
    return torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * scale).to(dtype).to(dev)


def definition(x, w, positions, inv_freq, *, norm=True, eps=1e-6, weight_offset=0.0, rotary_start=0, interleaved=False, rope_scale=1.0):
    """Values and what they may be off by, before the rounding to x's type."""
    v = x.double().cpu()
    d = v.shape[2]
    if norm:
        v = v / torch.sqrt((v * v).mean(2, keepdim=True) + eps)
    if w is not None:
        v = v * (weight_offset + w.double().cpu())
    off = (d / 32 + 19) * U * v.abs()
    if positions is not None:
        f = inv_freq.shape[0]
        angle = positions.double().cpu()[:, None] * inv_freq.double().cpu()
        c, s = torch.cos(angle)[:, None] * rope_scale, torch.sin(angle)[:, None] * rope_scale
        i = torch.arange(f)
        ia, ib = (rotary_start + 2 * i, rotary_start + 2 * i + 1) if interleaved else (rotary_start + i, rotary_start + f + i)
        a, b = v[:, :, ia], v[:, :, ib]
        both = (d / 32 + 19 + 8 + 2 + 2) * U * abs(rope_scale) * (a.abs() + b.abs())
        v, off = v.clone(), off.clone()
        v[:, :, ia], v[:, :, ib] = a * c - b * s, a * s + b * c
        off[:, :, ia] = off[:, :, ib] = both
    return v, off


def check(q, k, wq, wk, positions, inv_freq, q_out=None, k_out=None, stream=None, **how):
    from weightstream_b200 import ops
    want = [definition(t, w, positions, inv_freq, **how) for t, w in ((q, wq), (k, wk)) if t is not None]
    got = ops.head_norm_rope(q, k, positions=positions, inv_freq=inv_freq, q_weight=wq, k_weight=wk, q_out=q_out, k_out=k_out,
                             stream=stream, **how)
    if stream is not None:
        stream.synchronize()
    assert (got[1] is None) == (k is None)
    for g, t, (v, off) in zip(got, (q, k), want):
        assert g.dtype == t.dtype and g.shape == t.shape
        tol = off + torch.finfo(t.dtype).eps / 2 * (v.abs() + off)
        bad = (g.double().cpu() - v).abs() > tol
        assert not bad.any(), ((g.double().cpu() - v).abs() / tol).max()
    return got


def frequencies(f, dev, theta=1e4):
    return torch.tensor([theta ** (-i / f) for i in range(f)], dtype=F32, device=dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot,start", [(128, 128, 0), (64, 64, 0), (512, 64, 448), (576, 64, 512), (192, 64, 128), (96, 48, 0), (80, 80, 0), (72, 16, 8),
                                         (256, 128, 64), (2048, 1024, 512), (8, 8, 0), (16, 8, 8), (1, 0, 0), (2, 2, 0), (7, 4, 2), (100, 50, 25),
                                         (130, 126, 3), (2056, 2048, 8), (24, 16, 8), (1032, 16, 1016)])
@pytest.mark.parametrize("m,hq,hk", [(1, 5, 1), (9, 17, 3)])
def test_shapes(dev, dtype, interleaved, d, rot, start, m, hq, hk):
    rng = np.random.default_rng(d + m)
    positions = torch.from_numpy(rng.integers(0, 5000, m)).to(dev) if rot else None
    inv = frequencies(rot // 2, dev) if rot else None
    check(made(rng, (m, hq, d), dtype, dev), made(rng, (m, hk, d), dtype, dev), made(rng, (d,), BF16, dev), made(rng, (d,), BF16, dev), positions, inv,
          rotary_start=start if rot else 0, interleaved=interleaved)


@pytest.mark.gpu
@pytest.mark.parametrize("how", [dict(norm=False), dict(weight_offset=1.0), dict(rope_scale=0.7), dict(eps=0.5), dict(eps=0.0)])
@pytest.mark.parametrize("weights", [None, F32, BF16])
@pytest.mark.parametrize("d", [128, 90])
def test_forms(dev, how, weights, d):
    rng = np.random.default_rng(d)
    w = [None if weights is None else made(rng, (d,), weights, dev) for _ in range(2)]
    q, k = made(rng, (6, 4, d), BF16, dev), made(rng, (6, 2, d), BF16, dev)
    positions = torch.arange(6, dtype=torch.int32, device=dev)
    check(q, k, *w, positions, frequencies(d // 2, dev), **how)
    check(q, None, w[0], None, positions, frequencies(d // 2, dev), **how)
    check(q, k, None, w[1], None, None, **how)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [300, 1111])
@pytest.mark.parametrize("hq,hk", [(64, 8), (3, 70), (1, 1)])
def test_many_tokens(dev, m, hq, hk):
    rng = np.random.default_rng(m)
    check(made(rng, (m, hq, 64), BF16, dev), made(rng, (m, hk, 64), BF16, dev), made(rng, (64,), F32, dev), None,
          torch.from_numpy(rng.integers(0, 1 << 20, m)).to(dev), frequencies(16, dev), rotary_start=32)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rot,start,hq,hk", [(128, 128, 0, 9, 2), (512, 64, 448, 3, 1), (96, 32, 64, 5, 5), (64, 64, 0, 1, 17)])
def test_blocks_of_several_tokens(dev, dtype, interleaved, d, rot, start, hq, hk):
    rng = np.random.default_rng(d + hq)
    row = made(rng, (1187, (hq + hk) * d), dtype, dev)
    q, k = row[:, :hq * d].unflatten(1, (hq, d)), row[:, hq * d:].unflatten(1, (hk, d))
    check(q, k, made(rng, (d,), BF16, dev), made(rng, (d,), BF16, dev), torch.from_numpy(rng.integers(0, 1 << 20, 1187)).to(dev), frequencies(rot // 2, dev),
          rotary_start=start, interleaved=interleaved, q_out=q, k_out=k)


@pytest.mark.gpu
@pytest.mark.parametrize("positions", [[0, 1, 2 ** 20, 2 ** 24 + 1, 2 ** 31 - 1], [-1, -4097, 10 ** 6 + 1, 2 ** 30 + 3, 77]])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_far_positions(dev, positions, dtype):
    rng = np.random.default_rng(1)
    check(made(rng, (5, 2, 64), F32, dev), None, None, None, torch.tensor(positions, dtype=dtype, device=dev), frequencies(32, dev, 5e5))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("d,pad", [(64, 8), (64, 3), (128, 128), (30, 1)])
def test_strides_offsets_and_results_in_place(dev, dtype, d, pad):
    rng = np.random.default_rng(d + pad)
    row = made(rng, (11, 9 * d + pad), dtype, dev)
    inv, pos = frequencies(d // 2, dev), torch.arange(100, 111, device=dev)
    q, k = row[:, :6 * d].unflatten(1, (6, d)), row[:, 6 * d:8 * d].unflatten(1, (2, d))
    check(q, k, None, None, pos, inv)                                   # slices of a fused row
    check(q.transpose(0, 1).contiguous().transpose(0, 1), k, None, None, pos, inv)  # heads outside
    check(k[:, :1].expand(11, 5, d), k, None, None, pos, inv)           # one head read by several
    check(row[:, pad:pad + 2 * d].unflatten(1, (2, d))[3:], None, None, None, pos[3:], inv)
    rest = row[:, 8 * d:].clone()
    check(q, k, None, None, pos, inv, q_out=q, k_out=k)                 # the slices themselves
    assert torch.equal(row[:, 8 * d:], rest)
    wide = torch.full((11, 7, d + pad), 3.0, dtype=dtype, device=dev)
    check(q, None, None, None, pos, inv, q_out=wide[:, :6, :d])
    assert (wide[:, 6] == 3.0).all() and (wide[:, :, d:] == 3.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("d", [64, 66])
def test_values_that_are_not_finite_stay_in_their_head(dev, d):
    from weightstream_b200 import ops
    rng = np.random.default_rng(2)
    q = made(rng, (4, 4, d), F32, dev)
    q[0, 1, 3], q[1, 2, 0], q[2, 0] = float("nan"), float("inf"), 0.0
    pos, inv = torch.arange(4, device=dev), frequencies(d // 2, dev)
    got, _ = ops.head_norm_rope(q, positions=pos, inv_freq=inv)
    assert torch.isnan(got[0, 1]).all() and torch.isnan(got[1, 2]).any()
    assert (got[2, 0] == 0).all()                                       # a head of zeros
    keep = torch.ones((4, 4), dtype=torch.bool, device=dev)
    keep[0, 1] = keep[1, 2] = False
    assert torch.isfinite(got[keep]).all()


@pytest.mark.gpu
def test_nothing_to_do(dev):
    from weightstream_b200 import ops
    q, k = ops.head_norm_rope(torch.empty((0, 4, 64), device=dev), torch.empty((0, 2, 64), device=dev))
    assert q.shape == (0, 4, 64) and k.shape == (0, 2, 64)
    q, k = ops.head_norm_rope(torch.ones((3, 0, 64), device=dev), torch.ones((3, 2, 64), device=dev))
    assert q.shape == (3, 0, 64) and (k - 1).abs().max() < 1e-6
    q, k = ops.head_norm_rope(torch.ones((3, 2, 64), device=dev), torch.ones((3, 0, 64), device=dev))
    assert k.shape == (3, 0, 64) and (q - 1).abs().max() < 1e-6


@pytest.mark.gpu
def test_stream_and_graph(dev):
    from weightstream_b200 import ops
    rng = np.random.default_rng(3)
    q, k = made(rng, (7, 8, 128), BF16, dev), made(rng, (7, 2, 128), BF16, dev)
    pos, inv = torch.arange(7, device=dev), frequencies(64, dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    check(q, k, None, None, pos, inv, stream=s)
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = ops.head_norm_rope(q, k, positions=pos, inv_freq=inv)
    torch.cuda.current_stream().wait_stream(s)
    for seed in (4, 5):
        q.copy_(made(np.random.default_rng(seed), q.shape, BF16, dev))
        pos.add_(1000)
        graph.replay()
        want = ops.head_norm_rope(q, k, positions=pos, inv_freq=inv)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def arguments():
    return dict(q=torch.zeros((3, 4, 16)), k=torch.zeros((3, 2, 16)), positions=torch.zeros(3, dtype=torch.int64), inv_freq=torch.ones(8),
                q_weight=torch.ones(16), k_weight=torch.ones(16))


@pytest.mark.parametrize("change,error", [
    (dict(q=torch.zeros((3, 64))), ValueError), (dict(q=torch.zeros((3, 4, 0))), ValueError), (dict(q=torch.zeros((3, 4, 16), dtype=torch.float16)), TypeError),
    (dict(k=torch.zeros((2, 2, 16))), ValueError), (dict(k=torch.zeros((3, 2, 8))), ValueError), (dict(k=torch.zeros((3, 2, 16), dtype=BF16)), TypeError),
    (dict(q=torch.zeros((3, 4, 32))[:, :, ::2]), ValueError), (dict(positions=None), ValueError), (dict(inv_freq=None), ValueError),
    (dict(positions=torch.zeros(2, dtype=torch.int64)), ValueError), (dict(positions=torch.zeros(3)), TypeError),
    (dict(positions=torch.zeros(6, dtype=torch.int64)[::2]), ValueError), (dict(inv_freq=torch.ones(9)), ValueError), (dict(inv_freq=torch.ones(0)), ValueError),
    (dict(inv_freq=torch.ones(8, dtype=torch.float64)), TypeError), (dict(rotary_start=1), ValueError), (dict(rotary_start=-1), ValueError),
    (dict(q_weight=torch.ones(15)), ValueError), (dict(k_weight=torch.ones(16, dtype=BF16)), TypeError), (dict(q_weight=torch.ones(16, dtype=torch.float64)), TypeError),
    (dict(eps=-1.0), ValueError), (dict(eps=float("nan")), ValueError), (dict(q_out=torch.zeros((3, 4, 8))), ValueError), (dict(q_out=torch.zeros((3, 4, 16), dtype=BF16)), TypeError),
    (dict(q_out=torch.zeros((3, 1, 16)).expand(3, 4, 16)), ValueError), (dict(k_out=torch.zeros((1, 2, 16)).expand(3, 2, 16)), ValueError),
    (dict(k=None), ValueError), (dict(q=[1.0]), TypeError), (dict(k=3), TypeError), (dict(inv_freq=2.0), TypeError),
])
def test_refusals(change, error):
    from weightstream_b200 import ops
    with pytest.raises(error):
        ops.head_norm_rope(**{**arguments(), **change})


def test_host_tensors_are_refused():
    from weightstream_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.head_norm_rope(**arguments())


@pytest.mark.gpu
@pytest.mark.parametrize("start", [2 ** 31, 2 ** 32, -2 ** 32, 2 ** 32 + 8, 2 ** 62, 2 ** 70, -2 ** 70])
def test_starts_beyond_32_bits_are_refused(dev, start):
    from weightstream_b200 import ops
    a = {k: v.to(dev) for k, v in arguments().items()}
    with pytest.raises(ValueError, match="not within"):
        ops.head_norm_rope(**{**a, "inv_freq": torch.ones(4, device=dev)}, rotary_start=start)
    q, _ = ops.head_norm_rope(torch.ones((3, 2, 16), device=dev), rotary_start=start)      # (without positions there is no part)
    assert (q - 1).abs().max() < 1e-6


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,far", [(torch.int32, 2 ** 31), (torch.int64, 2 ** 31), (torch.int64, 2 ** 40), (torch.int64, 2 ** 53)])
@pytest.mark.parametrize("d", [16, 14])
def test_angles_of_far_positions(dev, dtype, far, d):
    """Cosines and sines by themselves: heads of (1, 0) without a norm.  An argument of half a turn at most is rounded to 32 bits
    (pi 2^-25, less than 2 u), cosine and sine err by 2 u, the products and the sum with zeros add a rounding each: 6 u.  The angle
    itself is the oracle's to 2^-60: a rational number reduced by a pi of 75 digits."""
    from fractions import Fraction

    from weightstream_b200 import ops
    rng = np.random.default_rng(far.bit_length() + d)
    f, m = d // 2, 200
    two_pi = 2 * Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628")
    positions = rng.integers(far - far // 4, far, m) * rng.choice([-1, 1], m)
    inv = np.concatenate([[1.0, 0.5], 1.0 - rng.random(f - 2) * 0.9]).astype(np.float32)
    q = torch.zeros((m, 1, d), device=dev)
    q[:, :, :f] = 1.0
    got, _ = ops.head_norm_rope(q, positions=torch.from_numpy(positions).to(dtype).to(dev), inv_freq=torch.from_numpy(inv).to(dev), norm=False)
    got = got.double().cpu().numpy()[:, 0]
    for t in range(m):
        for i in range(f):
            turn = int(positions[t]) * Fraction(float(inv[i])) / two_pi
            angle = float((turn - round(turn)) * two_pi)
            assert abs(got[t, i] - np.cos(angle)) <= 6 * U and abs(got[t, f + i] - np.sin(angle)) <= 6 * U, (positions[t], inv[i])
