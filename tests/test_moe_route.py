"""Choice of experts (ops.moe_route) against the definition in 64 bits.

Ids are exact: the oracle compares scores in 64 bits.  Weights (u = 2^-24): an exponential errs by 2 ulp and by |argument| u,
a logarithm, root and quotient by 2 ulp each, a sum of n terms by n u: 16 u + (2 |argument| + n) u relative.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
SCORES = ["softmax", "sigmoid", "sqrtsoftplus"]


@pytest.fixture()
def dev():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    return torch.device("cuda:0")


def definition(row, top_k, score, bias, renormalize, scale):
    """Ids, weights and the weights' relative tolerance of one row (float64)."""
    good = row > -math.inf
    s = np.zeros(row.shape)
    x = row[good]
    if score == "softmax":
        e = np.exp(x - x.max()) if x.size else x
        s[good] = e / e.sum()
    elif score == "sigmoid":
        s[good] = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
    else:
        s[good] = np.sqrt(np.maximum(x, 0) + np.log1p(np.exp(-np.abs(x))))
    # without a bias the order is the logits' (a score may saturate, even here)
    key = row if bias is None else s + bias
    order = np.lexsort((np.arange(row.size), -np.where(good, key, -np.inf)))
    ids = [i for i in order if good[i] and key[i] == key[i]][:top_k]
    w = s[ids]
    if renormalize and len(ids):
        w = w / w.sum()
    far = np.abs(row[ids] - (x.max() if score == "softmax" and x.size else 0.0))
    tol = (16 + 2 * far.max() + (top_k if renormalize else 0) + (row.size / 32 + 6 if score == "softmax" and not renormalize else 0)) * U if len(ids) else 0.0
    return ids, scale * w, 2 * tol


def check(logits, top_k, **how):
    from weightstream_b200 import ops
    ids, w = ops.moe_route(logits, top_k, **how)
    m = logits.shape[0]
    assert ids.shape == w.shape == (m, top_k) and ids.dtype == torch.int32 and w.dtype == F32
    x, bias = logits.double().cpu().numpy(), how.get("bias")
    bias = None if bias is None else bias.double().cpu().numpy()
    ids, w = ids.cpu().numpy(), w.double().cpu().numpy()
    for t in range(m):
        want, ww, tol = definition(x[t], top_k, how.get("score", "softmax"), bias, how.get("renormalize", True), how.get("scale", 1.0))
        assert list(ids[t, :len(want)]) == list(want), (t, ids[t], want)
        assert (ids[t, len(want):] == -1).all() and (w[t, len(want):] == 0).all()
        assert (np.abs(w[t, :len(want)] - ww) <= tol * np.abs(ww) + 2.0 ** -126).all(), (t, w[t], ww)


def rows_of(seed, m, experts, dtype, dev, scale=2.0, pad=0):
    v = np.random.default_rng(seed).standard_normal((m, experts + pad)).astype(np.float32) * scale
    return torch.from_numpy(v).to(dtype).to(dev)[:, :experts]


def biases(seed, experts, dev, scale=0.2):
    return torch.from_numpy(np.random.default_rng(seed + 99).standard_normal(experts).astype(np.float32) * scale).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("experts,top_k", [(1, 1), (2, 2), (8, 2), (31, 5), (33, 33 - 1), (64, 8), (65, 6), (128, 32), (129, 1), (256, 8), (384, 6), (385, 8), (512, 8), (1000, 7), (1024, 32)])
def test_sizes(dev, score, biased, experts, top_k):
    for m in (1, 5):
        check(rows_of(experts, m, experts, F32, dev), top_k, score=score, bias=biases(experts, experts, dev) if biased else None, scale=2.5)


@pytest.mark.gpu
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_forms(dev, score, renormalize, dtype):
    for bias in (None, biases(1, 96, dev)):
        check(rows_of(2, 333, 96, dtype, dev, pad=3), 4, score=score, renormalize=renormalize, bias=bias, scale=0.5)      # (strided rows, many equal logits in bf16)


@pytest.mark.gpu
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("biased", [False, True])
def test_equal_and_near_keys(dev, score, biased):
    """Equal keys go by index; keys that 32 bits cannot tell apart go by the definition."""
    base = np.zeros((6, 200), dtype=np.float32)
    base[1] = np.repeat(np.arange(50), 4)[::-1] * 0.125
    base[2] = 1.0 + np.arange(200) * 2.0 ** -23             # neighbouring floats
    base[3] = np.random.default_rng(0).permutation(200).astype(np.float32) * 2.0 ** -22 - 3.0
    base[4] = 20.0 + np.random.default_rng(1).permutation(200).astype(np.float32) * 2.0 ** -19     # scores next to their limit
    base[5] = np.random.default_rng(2).permutation(200).astype(np.float32) - 100.0
    x = torch.from_numpy(base).to(dev)
    bias = torch.full((200,), 0.3, device=dev) if biased else None
    if score == "sigmoid" and biased:
        x = x[[0, 1, 2, 3, 5]]                              # (near 1 the oracle's own 64 bits tie)
    if score == "softmax" and biased:
        x = x[:5]                                           # (scores below 64 bits of the bias tie in the oracle too)
    check(x, 8, score=score, bias=bias)
    if biased:      # a bias that makes up for the score's difference, up to its rounding
        l = rows_of(3, 1, 200, F32, dev)
        s = {"softmax": torch.softmax, "sigmoid": lambda v, _: torch.sigmoid(v), "sqrtsoftplus": lambda v, _: torch.sqrt(torch.log1p(torch.exp(v)))}[score](l.double(), 1)
        check(l, 8, score=score, bias=(2.0 - s[0]).float())


@pytest.mark.gpu
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("biased", [False, True])
def test_masked_and_nan_experts(dev, score, biased):
    x = rows_of(4, 7, 40, F32, dev)
    x[0, 3:] = -math.inf                # fewer than are wanted
    x[1] = -math.inf                    # none
    x[2, ::2] = float("nan")
    x[3] = float("nan")
    x[4, 5:] = torch.finfo(F32).min     # the type's lowest value is a value
    x[5] = -200.0 if score != "sqrtsoftplus" else -150.0        # scores that 32 bits do not hold: their ratios are
    x[5, 7] = x[5, 0] + 1.0
    bias = biases(4, 40, dev) if biased else None
    if biased:
        bias[20] = float("nan")
        x = x[[0, 1, 2, 3, 6]]
    else:
        from weightstream_b200 import ops
        ids, w = ops.moe_route(x, 6, score=score)
        # the row of lowest values has five of weight zero or, where they are all there is, equal ones
        assert ids[4].tolist()[:5] == sorted(range(5), key=lambda i: -float(x[4, i])) and int(ids[4, 5]) == 5
        x = x[[0, 1, 2, 3, 5, 6]]
    check(x, 6, score=score, bias=bias)


@pytest.mark.gpu
@pytest.mark.parametrize("score", SCORES)
def test_many_tokens(dev, score):
    check(rows_of(8, 3001, 128, F32, dev), 8, score=score, bias=biases(8, 128, dev))


@pytest.mark.gpu
def test_no_rows(dev):
    from weightstream_b200 import ops
    ids, w = ops.moe_route(torch.empty((0, 8), device=dev), 3)
    assert ids.shape == w.shape == (0, 3)


@pytest.mark.gpu
def test_stream_and_graph(dev):
    from weightstream_b200 import ops
    x, bias = rows_of(6, 20, 64, F32, dev), biases(6, 64, dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    a = ops.moe_route(x, 4, bias=bias, stream=s)
    s.synchronize()
    b = ops.moe_route(x, 4, bias=bias)
    assert all(torch.equal(i, j) for i, j in zip(a, b))
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = ops.moe_route(x, 4, bias=bias)
    torch.cuda.current_stream().wait_stream(s)
    x.copy_(rows_of(7, 20, 64, F32, dev))
    graph.replay()
    assert all(torch.equal(i, j) for i, j in zip(got, ops.moe_route(x, 4, bias=bias)))


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(8)), ValueError), (dict(logits=torch.zeros((3, 0))), ValueError), (dict(logits=torch.zeros((3, 8), dtype=torch.float16)), TypeError),
    (dict(logits=torch.zeros((3, 16))[:, ::2]), ValueError), (dict(top_k=0), ValueError), (dict(top_k=9), ValueError), (dict(score="relu"), ValueError),
    (dict(bias=torch.zeros(7)), ValueError), (dict(bias=torch.zeros(8, dtype=BF16)), TypeError), (dict(logits=None), TypeError), (dict(bias=0.5), TypeError),
])
def test_refusals(change, error):
    from weightstream_b200 import ops
    with pytest.raises(error):
        ops.moe_route(**{**dict(logits=torch.zeros((3, 8)), top_k=2, bias=torch.zeros(8)), **change})


@pytest.mark.gpu
@pytest.mark.parametrize("experts,top_k", [(1025, 2), (64, 33)])
def test_too_many(dev, experts, top_k):
    from weightstream_b200 import ops
    with pytest.raises(ops.WsError, match="CAPACITY"):
        ops.moe_route(torch.zeros((3, experts), device=dev), top_k)


@pytest.mark.gpu
@pytest.mark.parametrize("size", [900.0, 1e4, 1e6, 1e9])
@pytest.mark.parametrize("top_k", [1, 8])
def test_biases_that_cancel_large_scores(dev, size, top_k):
    """Keys near zero of scores whose own rounding in 32 bits is larger than what the keys differ by.  Weights: a root of
    a value above 1 errs by 4 u, the others' arguments are 4 at most: (16 + 2 * 4 + top_k) u."""
    from weightstream_b200 import ops
    rng = np.random.default_rng(int(size) + top_k)
    x = np.where(np.arange(80) < 64, size * (1 + rng.random(80)), -4 + rng.random(80)).astype(np.float32)
    exact = lambda v: np.sqrt(np.maximum(v, 0) + np.log1p(np.exp(-np.abs(v))))  # noqa: E731
    step = np.where(np.arange(80) < 64, np.spacing(x), 2e-5)
    x = (x + rng.integers(-8, 9, (60, 80)) * step).astype(np.float32)
    bias = (-exact(x.astype(np.float64)).mean(0)).astype(np.float32)
    ids, w = ops.moe_route(torch.from_numpy(x).to(dev), top_k, score="sqrtsoftplus", bias=torch.from_numpy(bias).to(dev))
    s = exact(x.astype(np.float64))
    for t in range(60):
        want = np.lexsort((np.arange(80), -(s[t] + bias.astype(np.float64))))[:top_k]
        assert ids[t].tolist() == want.tolist(), t
        ww = s[t, want] / s[t, want].sum()
        assert (np.abs(w[t].double().cpu().numpy() - ww) <= (24 + top_k) * U * ww).all(), t


@pytest.mark.gpu
def test_one_large_score_among_small_ones(dev):
    """The first expert's key is the second largest, whichever way its score's root is rounded to 32 bits."""
    from weightstream_b200 import ops
    x = torch.tensor([[1000000.0625, -4.0, -4.0]], device=dev)
    bias = torch.tensor([-1000.0, -0.13467541, -0.13470542], device=dev)
    for top_k in (1, 2, 3):
        ids, _ = ops.moe_route(x, top_k, score="sqrtsoftplus", bias=bias)
        assert ids[0].tolist() == [1, 0, 2][:top_k]


@pytest.mark.gpu
@pytest.mark.parametrize("biased", [False, True])
@pytest.mark.parametrize("renormalize", [False, True])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_softmax_that_is_no_number_chooses_none(dev, biased, renormalize, dtype):
    """With a logit of +inf every score of the row is NaN."""
    from weightstream_b200 import ops
    x = rows_of(9, 4, 40, dtype, dev)
    x[1, 7] = x[3, 0] = x[3, 39] = math.inf
    how = dict(score="softmax", bias=biases(9, 40, dev) if biased else None, renormalize=renormalize)
    ids, w = ops.moe_route(x, 6, **how)
    assert (ids[[1, 3]] == -1).all() and (w[[1, 3]] == 0).all()
    check(x[[0, 2]], 6, **how)
