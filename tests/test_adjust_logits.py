"""Biases, penalties and masks on logits (ops.adjust_logits) against the definition in 64 bits.

Tolerance (u = 2^-24): one rounding each of the bias' sum, the quotient or product, the frequency's and the presence's: 4 u of
the sum of all magnitudes on the way; then the result's own rounding.
"""
import math

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


def batch(seed, m, vocab, dtype, dev, *, history=40, biases=5, masks=2, pad=0, offsets=torch.int32):
    """Arguments of a call; histories and lists of biases of every length, tokens outside the vocabulary among them."""
    rng = np.random.default_rng(seed)
    put = lambda a, t: torch.from_numpy(np.asarray(a)).to(t).to(dev)
    a = dict(logits=put(rng.standard_normal((m, vocab + pad)) * 3, dtype)[:, :vocab])
    if history:
        n = rng.integers(0, 2 * history, m) * (rng.random(m) < 0.8)
        tok = rng.integers(0, max(1, min(vocab, history // 2)), int(n.sum()))
        tok = np.where(rng.random(tok.size) < 0.3, rng.integers(0, vocab, tok.size), tok)
        tok = np.where(rng.random(tok.size) < 0.05, rng.choice([-1, vocab, 2 ** 31 - 1, -2 ** 31], tok.size), tok)
        a.update(tokens=put(tok, torch.int32), offsets=put(np.concatenate([[0], np.cumsum(n)]), offsets), prompt_lens=put(rng.integers(-1, 1 + 2 * history, m), torch.int32),
                 repetition=put(0.5 + rng.random(m) * 1.5, F32), frequency=put(rng.random(m) - 0.3, F32), presence=put(rng.random(m) - 0.3, F32))
    if biases:
        n = rng.integers(0, 2 * biases, m)
        ids = rng.integers(-1, vocab + 1, int(n.sum()))
        a.update(bias_ids=put(ids, torch.int32), bias=put(rng.standard_normal(ids.size) * 5, F32), bias_offsets=put(np.concatenate([[0], np.cumsum(n)]), offsets))
    if masks:
        words = (vocab + 31) // 32 + pad
        a.update(mask=put(rng.integers(-2 ** 31, 2 ** 31, (masks, words)), torch.int32), mask_rows=put(rng.integers(-1, masks, m), torch.int32))
    return a


def definition(a):
    """Values, and what they may be off by before the rounding to the logits' type."""
    z = a["logits"].double().cpu().numpy().copy()
    m, vocab = z.shape
    size = np.abs(np.where(np.isfinite(z), z, 0.0))
    n = {k: v.cpu().numpy() for k, v in a.items() if isinstance(v, torch.Tensor) and k != "logits"}
    clip = lambda v, top: min(max(int(v), 0), top)
    for t in range(m):
        if "bias_ids" in n:
            lo = clip(n["bias_offsets"][t], n["bias_ids"].size)
            hi = max(lo, clip(n["bias_offsets"][t + 1], n["bias_ids"].size))
            last = {int(v): float(b) for v, b in zip(n["bias_ids"][lo:hi], n["bias"][lo:hi]) if 0 <= v < vocab}
            for v, b in last.items():
                z[t, v] += b
                size[t, v] += abs(b)
        if "tokens" in n:
            lo = clip(n["offsets"][t], n["tokens"].size)
            hi = max(lo, clip(n["offsets"][t + 1], n["tokens"].size))
            one = n["tokens"][lo:hi]
            answer = one[max(0, int(n["prompt_lens"][t])) if "prompt_lens" in n else 0:]
            one, answer = one[(one >= 0) & (one < vocab)], answer[(answer >= 0) & (answer < vocab)]
            seen, count = np.bincount(one, minlength=vocab) > 0, np.bincount(answer, minlength=vocab)
            r, f, p = (float(n[k][t]) if k in n else d for k, d in (("repetition", 1.0), ("frequency", 0.0), ("presence", 0.0)))
            with np.errstate(invalid="ignore"):
                z[t] = np.where(seen, np.where(z[t] > 0, z[t] / r, z[t] * r), z[t])
            size[t] = size[t] * np.where(seen, max(r, 1 / r), 1.0) + np.where(count > 0, abs(f) * count + abs(p), 0.0)
            z[t] -= np.where(count > 0, f * count + p, 0.0)
        if "mask" in n:
            which = int(n["mask_rows"][t]) if "mask_rows" in n else t
            if 0 <= which < n["mask"].shape[0]:
                v = np.arange(vocab)
                z[t][(n["mask"][which].view(np.uint32)[v >> 5] >> (v & 31).astype(np.uint32)) & 1 == 0] = -math.inf
    return z, 4 * U * size


def check(a, out=None, stream=None):
    from weightstream_b200 import ops
    z, off = definition(a)
    dtype = a["logits"].dtype
    got = ops.adjust_logits(**a, out=out, stream=stream)
    if stream is not None:
        stream.synchronize()
    assert got.dtype == dtype and got.shape == a["logits"].shape
    g = got.double().cpu().numpy()
    fine = np.isfinite(z)
    assert np.array_equal(g[~fine], z[~fine], equal_nan=True)
    assert np.isfinite(g[fine]).all()
    tol = off + torch.finfo(dtype).eps / 2 * (np.abs(np.where(fine, z, 0)) + off)
    bad = np.abs(g - np.where(fine, z, g))[fine] > tol[fine]
    assert not bad.any()
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [1, 3, 31, 32, 33, 500, 4099, 16390, 50257, 129280])
@pytest.mark.parametrize("m", [1, 4])
def test_sizes(dev, dtype, vocab, m):
    check(batch(vocab + m, m, vocab, dtype, dev, offsets=torch.int64 if m == 1 else torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("vocab", [20011, 33000])
def test_many_rows(dev, dtype, vocab):
    check(batch(5, 77, vocab, dtype, dev, history=300))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("parts", [("tokens",), ("bias",), ("mask",), ("tokens", "mask"), ("bias", "mask"), ("tokens", "bias"), ()])
def test_parts(dev, dtype, parts):
    for vocab in (777, 30000):
        check(batch(6, 50, vocab, dtype, dev, history=60 if "tokens" in parts else 0, biases=9 if "bias" in parts else 0, masks=3 if "mask" in parts else 0))


@pytest.mark.gpu
@pytest.mark.parametrize("without", ["prompt_lens", "repetition", "frequency", "presence", "mask_rows"])
def test_defaults(dev, without):
    a = batch(7, 6, 1000, F32, dev, masks=6)
    del a[without]
    check(a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pad", [1, 3, 8, 16])
@pytest.mark.parametrize("vocab", [40, 9001])
def test_strides_offsets_and_results(dev, dtype, pad, vocab):
    a = batch(8, 5, vocab, dtype, dev, pad=pad)
    want = check(a)
    wide = torch.full((5, vocab + 40), 7.0, dtype=dtype, device=dev)
    check(a, out=wide[:, pad:pad + vocab])                              # a result that lies otherwise
    assert (wide[:, :pad] == 7.0).all() and (wide[:, pad + vocab:] == 7.0).all()
    b = {**a, "logits": torch.nn.functional.pad(a["logits"], (pad, 24))[:, pad:pad + vocab]}
    got = check(b, out=b["logits"])                                     # in place
    assert got is b["logits"] and torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_logits_that_are_not_finite(dev, dtype):
    a = batch(9, 8, 300, dtype, dev, history=400, biases=100, masks=0)
    a["logits"][:, ::3], a["logits"][:, 1::7], a["logits"][:, 2::11] = -math.inf, math.inf, float("nan")
    a["logits"][:, 5] = torch.finfo(dtype).min
    a["presence"].zero_()
    a["repetition"].fill_(1.0)
    check(a)


@pytest.mark.gpu
def test_every_token_masked(dev):
    a = batch(10, 3, 5000, F32, dev)
    a["mask"].zero_()
    a["mask_rows"] = torch.tensor([0, -1, 1], dtype=torch.int32, device=dev)
    got = check(a)
    assert (got[0] == -math.inf).all() and (got[2] == -math.inf).all() and torch.isfinite(got[1]).all()


@pytest.mark.gpu
def test_offsets_and_rows_out_of_range(dev):
    a = batch(11, 6, 2000, F32, dev)
    n, b = a["tokens"].shape[0], a["bias"].shape[0]
    a["offsets"] = torch.tensor([-5, 3, 2, n + 9, n, 4, 2 ** 31 - 1], dtype=torch.int32, device=dev)
    a["bias_offsets"] = torch.tensor([b + 3, 1, 0, -7, b, b + 1, 2], dtype=torch.int32, device=dev)
    a["mask_rows"] = torch.tensor([0, 1, 2, -1, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32, device=dev)
    a["prompt_lens"] = torch.tensor([-2 ** 31, 2 ** 31 - 1, 0, 1, 2, 3], dtype=torch.int32, device=dev)
    check(a)


@pytest.mark.gpu
def test_a_token_repeated_very_often(dev):
    a = batch(12, 2, 1000, F32, dev, masks=0)
    a["tokens"] = torch.full((200000,), 17, dtype=torch.int32, device=dev)
    a["offsets"] = torch.tensor([0, 70000, 200000], dtype=torch.int32, device=dev)
    a["prompt_lens"] = torch.tensor([1, 65536], dtype=torch.int32, device=dev)
    check(a)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_long_lists_of_biases(dev, dtype):
    check(batch(13, 3, 700, dtype, dev, biases=3000))
    check(batch(14, 70, 20003, dtype, dev, biases=400))


@pytest.mark.gpu
def test_more_touched_values_than_are_noted(dev):
    """A slice of a row where nearly every token has occurred, in batches of few and of many rows."""
    for m, vocab in ((1, 5000), (80, 17000)):
        a = batch(15, m, vocab, F32, dev, masks=3)
        a["tokens"] = torch.arange(vocab - 7, dtype=torch.int32, device=dev).repeat(m)
        a["offsets"] = torch.arange(m + 1, dtype=torch.int32, device=dev) * (vocab - 7)
        check(a)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [32767, 32768])
def test_histories_around_the_short_ones(dev, length):
    a = batch(16, 2, 300, BF16, dev)
    a["tokens"] = torch.cat([torch.full((length,), 5, dtype=torch.int32, device=dev), torch.randint(0, 300, (length,), dtype=torch.int32, device=dev)])
    a["offsets"] = torch.tensor([0, length, 2 * length], dtype=torch.int64, device=dev)
    a["bias_offsets"] = a["bias_offsets"].to(torch.int32)
    a["prompt_lens"] = torch.tensor([length, length // 2], dtype=torch.int32, device=dev)
    check(a)


@pytest.mark.gpu
def test_no_rows_and_no_masks(dev):
    from weightstream_b200 import ops
    assert ops.adjust_logits(torch.empty((0, 100), device=dev)).shape == (0, 100)
    a = batch(14, 4, 100, F32, dev)
    a["mask"] = a["mask"][:0]
    a["tokens"], a["bias_ids"], a["bias"] = a["tokens"][:0], a["bias_ids"][:0], a["bias"][:0]
    got = check(a)
    assert torch.equal(got, a["logits"])


@pytest.mark.gpu
def test_stream_and_graph(dev):
    from weightstream_b200 import ops
    a = batch(15, 9, 3001, F32, dev)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    check(a, stream=s)
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            got = ops.adjust_logits(**a)
    torch.cuda.current_stream().wait_stream(s)
    a["logits"].copy_(torch.randn_like(a["logits"]))
    a["tokens"].add_(3)
    graph.replay()
    assert torch.equal(got, check(a))


def arguments():
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32)
    return dict(logits=torch.zeros((2, 40)), tokens=i32(1, 2, 3), offsets=i32(0, 1, 3), prompt_lens=i32(0, 1), repetition=torch.ones(2), frequency=torch.ones(2),
                presence=torch.ones(2), bias_ids=i32(4), bias=torch.ones(1), bias_offsets=i32(0, 1, 1), mask=torch.zeros((3, 2), dtype=torch.int32), mask_rows=i32(0, 1))


@pytest.mark.parametrize("change,error", [
    (dict(logits=torch.zeros(40)), ValueError), (dict(logits=torch.zeros((2, 0))), ValueError), (dict(logits=torch.zeros((2, 40), dtype=torch.float16)), TypeError),
    (dict(logits=torch.zeros((2, 80))[:, ::2]), ValueError), (dict(tokens=None), ValueError), (dict(offsets=None), ValueError), (dict(offsets=torch.zeros(3)), TypeError),
    (dict(offsets=torch.zeros(2, dtype=torch.int32)), ValueError), (dict(tokens=torch.zeros(3)), TypeError), (dict(tokens=torch.zeros((1, 3), dtype=torch.int32)), ValueError),
    (dict(tokens=None, offsets=None), ValueError), (dict(prompt_lens=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(prompt_lens=torch.zeros(2)), TypeError),
    (dict(repetition=torch.ones(1)), ValueError), (dict(repetition=torch.ones(2, dtype=BF16)), TypeError), (dict(frequency=torch.ones(4)[::2]), ValueError),
    (dict(presence=torch.ones(2, dtype=torch.float64)), TypeError), (dict(bias=None), ValueError), (dict(bias=torch.ones(2)), ValueError), (dict(bias=torch.ones(1, dtype=BF16)), TypeError),
    (dict(bias_ids=None), ValueError), (dict(bias_offsets=None), ValueError), (dict(mask=torch.zeros((3, 1), dtype=torch.int32)), ValueError),
    (dict(mask=torch.zeros((3, 2), dtype=torch.int64)), TypeError), (dict(mask=torch.zeros((3, 4), dtype=torch.int32)[:, ::2]), ValueError), (dict(mask=None), ValueError),
    (dict(mask_rows=None), ValueError), (dict(mask_rows=torch.zeros(3, dtype=torch.int32)), ValueError), (dict(mask_rows=torch.zeros(2)), TypeError),
    (dict(out=torch.zeros((2, 41))), ValueError), (dict(out=torch.zeros((2, 40), dtype=BF16)), TypeError), (dict(out=torch.zeros((1, 40)).expand(2, 40)), ValueError),
    (dict(logits=None), TypeError), (dict(repetition=1.2), TypeError), (dict(mask=[[1]]), TypeError),
])
def test_refusals(change, error):
    from weightstream_b200 import ops
    with pytest.raises(error):
        ops.adjust_logits(**{**arguments(), **change})


def test_host_tensors_are_refused():
    from weightstream_b200 import ops
    with pytest.raises(ValueError, match="CUDA"):
        ops.adjust_logits(**arguments())


def lopsided(seed, m, vocab, length, dtype, dev, *, row=1, others=0, pad=0, **how):
    """A batch in which one row lists `length` biases and the others few or none."""
    rng = np.random.default_rng(seed)
    a = batch(seed, m, vocab, dtype, dev, biases=0, pad=pad, **how)
    n = np.full(m, others)
    n[row] = length
    ids = rng.integers(-1, vocab + 1, int(n.sum()))
    put = lambda v, t: torch.from_numpy(np.asarray(v)).to(t).to(dev)  # noqa: E731
    a.update(bias_ids=put(ids, torch.int32), bias=put(rng.standard_normal(ids.size) * 5, F32), bias_offsets=put(np.concatenate([[0], np.cumsum(n)]), torch.int32))
    return a


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,vocab,length,others", [(2, 700, 200, 0), (9, 2500, 1000, 3), (40, 20003, 4000, 7), (100, 20003, 9000, 2), (300, 4111, 30000, 0), (500, 8192, 20000, 20),
                                                   (7, 129, 700, 1)])
@pytest.mark.parametrize("pad", [0, 3])
def test_one_long_list_of_biases(dev, dtype, m, vocab, length, others, pad):
    a = lopsided(m + length, m, vocab, length, dtype, dev, others=others, pad=pad, row=m - 1)
    got = check(a)
    b = {**a, "logits": a["logits"].clone()}
    assert torch.equal(check(b, out=b["logits"]), got)
    check(lopsided(m, m, vocab, length, dtype, dev, others=others, row=0, history=0, masks=0))


@pytest.mark.gpu
def test_the_last_entry_counts_in_a_long_list(dev):
    for length in (129, 5000):
        a = lopsided(17, 64, 3000, length, F32, dev, history=0, masks=0)
        a["bias_ids"][:] = torch.arange(length, dtype=torch.int32, device=dev) % 3      # every entry but the last three is overtaken
        check(a)


@pytest.mark.gpu
def test_one_long_list_among_many_rows_takes_no_longer_than_it_is(dev):
    """One of 512 rows lists 50000 tokens, or all rows list 97 each.  A block that goes through the list a constant number of
    times takes some hundred rounds of its threads for it; one that looks for each of its listed values in the whole list takes as
    many times that as it has values for a thread."""
    from weightstream_b200 import ops
    a = lopsided(18, 512, 50000, 50000, BF16, dev, history=0, masks=0)
    a["bias_ids"] = torch.randperm(50000, device=dev).to(torch.int32)
    b = {**a, "bias_offsets": torch.arange(513, dtype=torch.int32, device=dev) * 97}

    def elapsed(how):
        times = []
        for _ in range(5):
            begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            ops.adjust_logits(**how)
            begin.record()
            for _ in range(5):
                ops.adjust_logits(**how)
            end.record()
            end.synchronize()
            times.append(begin.elapsed_time(end))
        return min(times)

    assert elapsed(a) < 8 * elapsed(b), (elapsed(a), elapsed(b))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("m,vocab,length,others", [(3, 129, 192, 0), (3, 129, 193, 0), (20, 700, 1000, 3), (4, 33000, 250, 0), (40, 20003, 2000, 7), (200, 20003, 9000, 2),
                                                   (600, 4111, 30000, 0), (25, 129280, 1500, 1)])
@pytest.mark.parametrize("pad", [0, 5])
def test_one_long_list_in_a_batch_of_short_ones(dev, dtype, m, vocab, length, others, pad):
    """No more than 64 biases a row on average, so a long list's places share the table of the counts."""
    for row, how in ((m - 1, {}), (0, dict(history=0)), (1, dict(masks=0))):
        a = lopsided(m + length, m, vocab, length, dtype, dev, others=others, pad=pad, row=row, **how)
        assert a["bias"].shape[0] // m <= 64
        got = check(a)
        b = {**a, "logits": a["logits"].clone()}
        assert torch.equal(check(b, out=b["logits"]), got)


@pytest.mark.gpu
def test_the_last_entry_counts_in_a_long_list_among_short_ones(dev):
    for m, length in ((40, 193), (128, 5000)):
        a = lopsided(17, m, 3000, length, F32, dev, history=0, masks=0)
        a["bias_ids"][:] = torch.arange(length, dtype=torch.int32, device=dev) % 3
        check(a)


@pytest.mark.gpu
def test_long_histories_beside_a_long_list(dev):
    """A history beyond 32767 tokens is counted in wider fields, in both halves."""
    a = lopsided(19, 30, 20003, 1500, BF16, dev, row=2, history=30)
    n = 40000
    a["tokens"] = torch.cat([a["tokens"][:0], torch.randint(0, 20003, (n,), dtype=torch.int32, device=dev), torch.full((n,), 11, dtype=torch.int32, device=dev)])
    a["offsets"] = torch.tensor([0, 0, 0] + [2 * n] * 28, dtype=torch.int32, device=dev)
    a["prompt_lens"][2] = n // 2
    check(a)
