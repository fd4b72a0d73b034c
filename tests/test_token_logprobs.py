"""Scores of given tokens (ops.token_logprobs) against the definition in 64 bits.

Tolerance, from the arithmetic (u = 2^-24): a term exp(x - M) errs by 4 u (its exponential) and 2 u |x - M| (the argument);
a thread adds up to vocab / 512 + 4 of them one by one, 14 more levels join the threads.  So the sum s errs by at most
(vocab / 512 + 22 + 4 D) u relative, D = sum p |x - M|, and ln s, at most as much absolutely, adds its rounding.
logprob = (x - M) - ln s adds 2 u (|x - M| + |ln s|); the entropy ln s - t / s has t's error too, (1 + D) times that of s.
Ids, ranks and counts are exact.
"""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
LOWEST = {F32: torch.finfo(F32).min, BF16: torch.finfo(BF16).min}


@pytest.fixture()
def dev():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    return torch.device("cuda:0")


def rows_of(rng, m, vocab, dtype, dev, pad=0, scale=2.5):
    v = torch.from_numpy(rng.standard_normal((m, vocab + pad)).astype(np.float32) * scale)
    return v.to(dtype).to(dev)[:, :vocab]


def compare(x, tok, top, r):
    """One result against numpy, row by row."""
    m, vocab = x.shape
    assert r.logprobs.shape == r.entropy.shape == r.rank.shape == (m,) and r.rank.dtype == torch.int32
    assert (r.top_ids is None) == (top == 0)
    xs, ts = x.float().cpu().numpy(), tok.cpu().numpy()
    lp, en, rk = r.logprobs.cpu().numpy(), r.entropy.cpu().numpy(), r.rank.cpu().numpy()
    ids, tl = (r.top_ids.cpu().numpy(), r.top_logprobs.cpu().numpy()) if top else (None, None)
    for i in range(m):
        row = xs[i].astype(np.float64)
        good = row > -math.inf
        order = np.lexsort((np.arange(vocab), -np.where(good, xs[i], -np.inf)))  # by value, then by index
        t = int(ts[i])
        has = 0 <= t < vocab
        if top:
            k = min(top, int(good.sum()))
            assert (ids[i, :k] == order[:k]).all(), (i, ids[i], order[:top])
            assert (ids[i, k:] == -1).all() and (tl[i, k:] == -math.inf).all()
        want_rank = int(((row > row[t]) | ((row == row[t]) & (np.arange(vocab) < t))).sum()) if has and row[t] == row[t] else -1
        assert rk[i] == want_rank, (i, rk[i], want_rank)
        if np.isnan(row).any() or (row == math.inf).any():
            assert math.isnan(en[i]) and (math.isnan(lp[i]) if has else lp[i] == 0)
            if top:
                assert np.isnan(tl[i, :k]).all()
            continue
        if not good.any():
            assert lp[i] == (-math.inf if has else 0.0) and en[i] == 0.0
            continue
        big = row[good].max()
        d = row[good] - big
        e = np.exp(d)
        s = e.sum()
        spread = float((e * -d).sum() / s)
        tol = U * (vocab / 512 + 22 + 4 * spread) + 2 * U
        assert abs(en[i] - (math.log(s) + spread)) <= tol * (2 + spread) + 2 * U * (math.log(s) + spread), (i, en[i], math.log(s) + spread)
        for got, j in [(lp[i], t)] * has + [(tl[i, j], order[j]) for j in range(k if top else 0)]:
            if row[j] == -math.inf:
                assert got == -math.inf
            else:
                ref = row[j] - big - math.log(s)
                assert abs(got - ref) <= tol + 2 * U * (abs(row[j] - big) + math.log(s) + abs(ref)), (i, j, got, ref)
        if not has:
            assert lp[i] == 0.0


def check(x, tok, top):
    from weightstream_b200 import ops
    compare(x, tok, top, ops.token_logprobs(x, tok, top=top))


def tokens(rng, m, vocab, dev, dtype=torch.int32):
    return torch.from_numpy(rng.integers(0, vocab, m)).to(dtype).to(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 31, 513, 4099, 20000, 50257, 129280, 160001])
@pytest.mark.parametrize("m,top", [(1, 20), (3, 0), (19, 5)])
def test_sizes(dev, dtype, vocab, m, top):
    rng = np.random.default_rng(vocab + m)
    check(rows_of(rng, m, vocab, dtype, dev), tokens(rng, m, vocab, dev), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m", [40, 100, 301])
@pytest.mark.parametrize("top", [0, 1, 32])
def test_many_rows(dev, dtype, m, top):
    rng = np.random.default_rng(m)
    check(rows_of(rng, m, 9001, dtype, dev), tokens(rng, m, 9001, dev, torch.int64), top)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad", [1, 2, 3, 5, 8])
def test_row_strides_and_offsets(dev, dtype, pad):
    rng = np.random.default_rng(pad)
    for vocab in (5, 30011):
        x = rows_of(rng, 9, vocab, dtype, dev, pad)
        check(x, tokens(rng, 9, vocab, dev), 8)
        check(x[2:, 1:], tokens(rng, 7, vocab - 1, dev), 8)


def patterns(vocab, dtype):
    i = np.arange(vocab)
    yield "equal", np.zeros(vocab)
    yield "ascending", i / 4.0
    yield "descending", -i / 4.0
    yield "few values", (i * 7919 % 11).astype(np.float64)
    yield "signed zeros", np.where(i % 2, 0.0, -0.0)
    for step in (512, 2048, 4096):  # all large values on one thread
        yield f"every {step}", np.where(i % step < 3, 10.0 + i / vocab, -i % 7 * 1.0)
        yield f"every {step} but low", np.where(i % step == 1, 1.0, 2.0)
    yield "last", np.where(i == vocab - 1, 5.0, 0.0)
    yield "block", np.where(i < 4000, 3.0, 0.0)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab,lead", [(40, 0), (33000, 0), (129280, 3)])
@pytest.mark.parametrize("m", [1, 160])
def test_ties_and_orders(dev, dtype, vocab, lead, m):
    rng = np.random.default_rng(4)
    rows = [p for _, p in patterns(vocab, dtype)]
    pick = range(len(rows)) if m == 1 else [j % len(rows) for j in range(m)]
    buf = torch.zeros((len(rows), vocab + lead), dtype=dtype)
    buf[:, lead:] = torch.from_numpy(np.stack(rows).astype(np.float32)).to(dtype)
    base = buf.to(dev)[:, lead:]
    if m == 1:
        for j in pick:
            for top in (1, 20, 32):
                check(base[j:j + 1], tokens(rng, 1, vocab, dev), top)
    else:
        x = torch.cat([base[j:j + 1] for j in pick])
        r = None
        from weightstream_b200 import ops
        tok = tokens(rng, m, vocab, dev)
        r = ops.token_logprobs(x, tok, top=20)
        some = list(range(len(rows))) + [m - 1]
        compare(x[some], tok[some], 20, ops.TokenLogprobs(*(t[some] for t in r)))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [100, 33001])
def test_masks(dev, dtype, vocab):
    rng = np.random.default_rng(8)
    x = rows_of(rng, 12, vocab, dtype, dev).clone()
    x[0] = -math.inf                            # nothing left
    x[1] = -math.inf
    x[1, vocab // 2] = 1.5                      # one entry left
    x[2, rng.random(vocab) < 0.9] = -math.inf
    x[3] = LOWEST[dtype]                        # masked by the type's lowest value: all equal
    x[4, :] = LOWEST[dtype]
    x[4, [3, vocab - 1]] = -2.0
    x[5, ::2] = LOWEST[dtype]
    x[6, ::2] = -math.inf
    x[6, 1::2] = LOWEST[dtype]
    x[7, 17] = math.nan
    x[8, 17] = math.inf
    x[9] = math.nan
    x[10] = -math.inf
    x[10, 5] = LOWEST[dtype]
    x[11] = -LOWEST[dtype]                      # the type's highest value
    for tok in (torch.full((12,), vocab // 2), torch.full((12,), 17), torch.full((12,), 16), torch.full((12,), vocab - 1)):
        for top in (0, 3, 32):
            check(x, tok.to(torch.int32).to(dev), top)


@pytest.mark.gpu
def test_tokens_that_are_none(dev):
    rng = np.random.default_rng(2)
    x = rows_of(rng, 6, 3001, F32, dev)
    check(x, torch.tensor([-1, 3001, 0, 3000, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev), 4)
    check(x, torch.tensor([-1, 3001, 0, 3000, 2 ** 40, -2 ** 40], dtype=torch.int64, device=dev), 4)


@pytest.mark.gpu
def test_argmax_and_alternatives_agree(dev):
    from weightstream_b200 import ops
    rng = np.random.default_rng(12)
    x = rows_of(rng, 33, 12345, BF16, dev)
    r = ops.token_logprobs(x, torch.zeros(33, dtype=torch.int32, device=dev), top=32)
    again = ops.token_logprobs(x, r.top_ids[:, 7].contiguous(), top=32)
    assert (again.rank == 7).all() and torch.equal(again.logprobs, r.top_logprobs[:, 7]) and torch.equal(again.entropy, r.entropy)


@pytest.mark.gpu
def test_no_rows_another_stream_and_a_graph(dev):
    from weightstream_b200 import ops
    r = ops.token_logprobs(torch.zeros((0, 50), device=dev), torch.zeros(0, dtype=torch.int64, device=dev), top=2)
    assert r.logprobs.shape == (0,) and r.top_ids.shape == (0, 2)
    rng = np.random.default_rng(1)
    x, tok = rows_of(rng, 5, 40000, F32, dev), tokens(rng, 5, 40000, dev)
    a = ops.token_logprobs(x, tok, top=9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    b = ops.token_logprobs(x, tok, top=9, stream=s)
    s.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        c = ops.token_logprobs(x, tok, top=9)
    x.neg_()
    g.replay()
    compare(x, tok, 9, c)


BAD = [
    (ValueError, dict(logits=torch.zeros(50))),
    (ValueError, dict(logits=torch.zeros((3, 0)))),
    (ValueError, dict(logits=torch.zeros((3, 100))[:, ::2])),
    (ValueError, dict(logits=torch.zeros((1, 50)).expand(3, 50))),
    (TypeError, dict(logits=torch.zeros((3, 50), dtype=torch.float16))),
    (ValueError, dict(tokens=torch.zeros(2, dtype=torch.int32))),
    (ValueError, dict(tokens=torch.zeros(6, dtype=torch.int32)[::2])),
    (TypeError, dict(tokens=torch.zeros(3))),
    (ValueError, dict(top=-1)),
    (ValueError, dict(top=33)),
]


def plain():
    return dict(logits=torch.zeros((3, 50)), tokens=torch.zeros(3, dtype=torch.int32), top=2)


@pytest.mark.parametrize("error,change", BAD)
def test_refuses(error, change):
    from weightstream_b200 import ops
    ops._token_logprobs_args(**plain())
    with pytest.raises(error):
        ops._token_logprobs_args(**{**plain(), **change})


@pytest.mark.gpu
def test_calls_refuse(dev):
    from weightstream_b200 import ops

    def move(d):  # with the same strides
        put = lambda t: torch.zeros(max(t.untyped_storage().nbytes(), 16) // t.element_size(), dtype=t.dtype, device=dev).as_strided(t.size(), t.stride())
        return {k: put(v) if isinstance(v, torch.Tensor) else v for k, v in d.items()}

    ops.token_logprobs(**move(plain()))
    for error, change in BAD:
        with pytest.raises(error):
            ops.token_logprobs(**{**move(plain()), **move(change)})
    with pytest.raises(ValueError):
        ops.token_logprobs(**plain())
    with pytest.raises(ValueError):
        ops.token_logprobs(**{**move(plain()), "tokens": plain()["tokens"]})


@pytest.mark.parametrize("name", ["logits", "tokens", "logprob", "entropy", "rank", "top_id", "top_logprob"])
def test_c_entry_refuses_what_is_not_aligned(name):
    """Results as well as inputs, before anything is launched."""
    import ctypes as C
    from weightstream_b200 import _lib
    L, err = _lib.load(), C.create_string_buffer(256)
    a = _lib.TokenLogprobsArgs(m=1, vocab=64, ld=64, top=2, dtype=_lib.WS_ACT_F32, token_bytes=4)
    room = torch.zeros(7, 128)
    for i, n in enumerate(["logits", "tokens", "logprob", "entropy", "rank", "top_id", "top_logprob"]):
        setattr(a, n, room[i].data_ptr() + (2 if n == name else 0))
    assert L.ws_token_logprobs(C.byref(a), None, err, len(err)) == _lib.WS_ERR_INVALID and b"aligned" in err.value
