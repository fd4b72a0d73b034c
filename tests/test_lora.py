"""Adapters of many requests (ops.lora_add, lora_shrink, lora_expand) against the formula in 64 bits.

Tolerance, from the arithmetic: the products of bf16 parts are exact, and an accumulating product step cuts or rounds its
sum at 2^-23 twice for every 16 terms.  A warp's chain is at most k / 128 steps of 16 long and 40 additions join the
warps, blocks and parts, so a shrunk value errs by at most (k / 64 + 80) 2^-23 of the sum of its terms' magnitudes; an
expanded one by (rank / 2 + 40) 2^-23 of its own, plus what the shrunk ones carry, plus the result's rounding.
"""
import numpy as np
import pytest

torch = pytest.importorskip("torch")

F32, BF16 = torch.float32, torch.bfloat16


@pytest.fixture()
def dev():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    return torch.device("cuda:0")


def make(rng, shape, dtype, dev, scale=1.0, pad=0):
    wide = shape[:-1] + (shape[-1] + pad,)
    v = torch.from_numpy(rng.standard_normal(wide).astype(np.float32) * scale).to(dtype).to(dev)
    return v[..., :shape[-1]] if pad else v


def batch(rng, m, adapters, dev, none=0.1):
    ids = rng.integers(0, adapters, m)
    ids[rng.random(m) < none] = -1
    return torch.from_numpy(ids.astype(np.int32)).to(dev)


def ref(y, x, a, b, ids, scale, shrunk=None):
    """(shrunk, its error bound, out, its error bound) in 64 bits."""
    d = lambda t: t.double().cpu()
    m, r = ids.shape[0], (a if a is not None else b.transpose(1, 2)).shape[1]
    s, se = torch.zeros((m, r), dtype=torch.float64), torch.zeros((m, r), dtype=torch.float64)
    if shrunk is not None:
        s = d(shrunk)
    out, err = (d(y), torch.zeros_like(d(y))) if y is not None else (None, None)
    count = (a if a is not None else b).shape[0]
    for i in torch.unique(ids).tolist():
        if not 0 <= i < count:
            continue
        rows = torch.nonzero(ids.cpu() == i).squeeze(1)
        if a is not None:
            xa, aa = d(x)[rows], d(a[i])
            s[rows] = xa @ aa.t()
            se[rows] = (a.shape[2] / 64 + 80) * 2.0 ** -23 * (xa.abs() @ aa.abs().t())
        if b is not None:
            f = float(scale[i]) if scale is not None else 1.0
            bb = d(b[i])
            out[rows] += f * (s[rows] @ bb.t())
            err[rows] = abs(f) * ((se[rows] + (r / 2 + 40) * 2.0 ** -23 * s[rows].abs()) @ bb.abs().t())
    return s, se, out, err


def close(got, want, err):
    tol = err * (1 + 2.0 ** -8) + (2.0 ** -8 if got.dtype == BF16 else 2.0 ** -24) * want.abs() + 1e-30
    bad = ~((got.double().cpu() - want).abs() <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, first at {torch.nonzero(bad)[0].tolist()}"


def check(dev, m, k, n, rank, adapters, xt=BF16, yt=F32, scaled=True, pad=0, ids=None, seed=0):
    from weightstream_b200 import ops
    rng = np.random.default_rng(seed + m * 31 + k + n + rank)
    x, y = make(rng, (m, k), xt, dev, pad=pad), make(rng, (m, n), yt, dev, pad=pad)
    a, b = make(rng, (adapters, rank, k), BF16, dev, k ** -0.5), make(rng, (adapters, n, rank), BF16, dev, 0.3)
    scale = make(rng, (adapters,), F32, dev) if scaled else None
    ids = batch(rng, m, adapters, dev) if ids is None else ids
    s, se, out, err = ref(y, x, a, b, ids, scale)
    got = ops.lora_add(y, x, a, b, ids, scale)
    assert got.dtype == yt and got.data_ptr() != y.data_ptr()
    close(got, out, err)
    t = ops.lora_shrink(x, a, ids)
    assert t.dtype == F32
    close(t, s, se)
    _, _, out2, err2 = ref(y, None, None, b, ids, scale, shrunk=t)
    close(ops.lora_expand(y, t, b, ids, scale), out2, err2)
    place = y.clone() if pad == 0 else torch.empty_like(y, memory_format=torch.contiguous_format).copy_(y)
    assert ops.lora_add(place, x, a, b, ids, scale, out=place) is place and torch.equal(place, got)


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [1, 4, 8, 16, 24, 32, 56, 64, 72, 128])
@pytest.mark.parametrize("m", [1, 9, 40, 256, 257, 512, 513, 700])
def test_ranks_and_batches(dev, rank, m):
    check(dev, m, 640, 520, rank, 7)


@pytest.mark.gpu
@pytest.mark.parametrize("k,n", [(1, 1), (8, 4), (7, 130), (33, 64), (2304, 5120), (8192, 7168), (1000, 8), (96, 2050)])
@pytest.mark.parametrize("m,adapters", [(1, 1), (17, 40), (300, 3)])
def test_sizes(dev, k, n, m, adapters):
    check(dev, m, k, n, 16, adapters)
    check(dev, m, k, n, 8, adapters, xt=F32, yt=BF16, scaled=False)


@pytest.mark.gpu
@pytest.mark.parametrize("k,n", [(1025, 516), (1030, 516), (1024, 517), (1025, 517), (129, 3), (1, 65)])
@pytest.mark.parametrize("rank", [8, 32, 64, 128])
@pytest.mark.parametrize("xt,yt", [(BF16, F32), (F32, BF16)])
def test_sorted_odd_sizes(dev, k, n, rank, xt, yt):
    check(dev, 600, k, n, rank, 3, xt=xt, yt=yt)


@pytest.mark.gpu
@pytest.mark.parametrize("xt", [F32, BF16])
@pytest.mark.parametrize("yt", [F32, BF16])
@pytest.mark.parametrize("rank", [16, 32, 64, 128])
@pytest.mark.parametrize("m", [5, 100, 600])
def test_types(dev, xt, yt, rank, m):
    check(dev, m, 1024, 768, rank, 5, xt=xt, yt=yt)


@pytest.mark.gpu
@pytest.mark.parametrize("pad", [1, 2, 8, 24])
def test_strides(dev, pad):
    for m in (6, 70, 290, 600):
        check(dev, m, 512, 256, 16, 4, pad=pad)
        check(dev, m, 512, 256, 64, 4, xt=F32, yt=BF16, pad=pad)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 8, 65, 256, 257, 512, 1100])
def test_ids(dev, m):
    full = lambda v: torch.full((m,), v, dtype=torch.int32, device=dev)
    check(dev, m, 256, 192, 16, 3, ids=full(-1))                      # nobody has one
    check(dev, m, 256, 192, 16, 3, ids=full(2))                       # all share one
    check(dev, m, 256, 192, 16, 3, ids=full(3))                       # beyond the table: none
    check(dev, m, 256, 192, 16, 3, ids=full(2 ** 31 - 1))
    check(dev, m, 256, 192, 16, 1200, ids=torch.arange(m, dtype=torch.int32, device=dev))      # each its own
    check(dev, m, 256, 192, 16, 2, ids=torch.arange(m, dtype=torch.int32, device=dev) % 3 - 1)


@pytest.mark.gpu
def test_many_adapters(dev):
    from weightstream_b200 import ops
    check(dev, 500, 64, 32, 8, 16384)
    m = 513  # a batch that is sorted
    x, y = torch.zeros((m, 8), dtype=BF16, device=dev), torch.zeros((m, 4), device=dev)
    a, b = torch.zeros((16385, 8, 8), dtype=BF16, device=dev), torch.zeros((16385, 4, 8), dtype=BF16, device=dev)
    ids = torch.zeros(m, dtype=torch.int32, device=dev)
    with pytest.raises(RuntimeError, match="CAPACITY"):
        ops.lora_add(y, x, a, b, ids)
    ops.lora_add(y[:512], x[:512], a, b, ids[:512])


@pytest.mark.gpu
def test_a_table_past_31_bits(dev):
    """The last adapter of a table of more than 2^31 values."""
    from weightstream_b200 import ops
    rng = np.random.default_rng(6)
    k, n, rank, count = 16384, 64, 128, 1040
    a, b = torch.zeros((count, rank, k), dtype=BF16, device=dev), torch.zeros((count, n, rank), dtype=BF16, device=dev)
    assert a.numel() > 2 ** 31
    a[-1], b[-1] = make(rng, (rank, k), BF16, dev, k ** -0.5), make(rng, (n, rank), BF16, dev, 0.3)
    x, y = make(rng, (3, k), BF16, dev), make(rng, (3, n), F32, dev)
    ids = torch.tensor([count - 1, 0, count - 1], dtype=torch.int32, device=dev)
    _, _, out, err = ref(y, x, a[-1:], b[-1:], torch.where(ids > 0, 0, -1), None)
    close(ops.lora_add(y, x, a, b, ids), out, err)


@pytest.mark.gpu
def test_results_do_not_depend_on_the_batch_around(dev):
    """The same token in another place of a sorted batch, and the same call twice: the same bits."""
    from weightstream_b200 import ops
    rng = np.random.default_rng(5)
    m = 900
    x, y = make(rng, (m, 512), BF16, dev), make(rng, (m, 256), F32, dev)
    a, b = make(rng, (6, 32, 512), BF16, dev, 0.05), make(rng, (6, 256, 32), BF16, dev, 0.3)
    ids = batch(rng, m, 6, dev)
    one = ops.lora_add(y, x, a, b, ids)
    for _ in range(3):
        assert torch.equal(ops.lora_add(y, x, a, b, ids), one)
    perm = torch.from_numpy(rng.permutation(m)).to(dev)
    assert torch.equal(ops.lora_add(y[perm], x[perm], a, b, ids[perm]), one[perm])


@pytest.mark.gpu
def test_values_that_are_not_finite(dev):
    """They stay with their token; large ones do not become infinite on the way."""
    from weightstream_b200 import ops
    rng = np.random.default_rng(7)
    for xt in (F32, BF16):
        x, y = make(rng, (12, 64), xt, dev), make(rng, (12, 64), F32, dev)
        a, b = make(rng, (2, 16, 64), BF16, dev, 0.1), make(rng, (2, 64, 16), BF16, dev, 0.1)
        ids = torch.zeros(12, dtype=torch.int32, device=dev)
        x[3, 5], x[7, 1] = float("inf"), float("nan")
        got = ops.lora_add(y, x, a, b, ids)
        bad = ~torch.isfinite(got).all(1)
        assert bad.nonzero().squeeze(1).tolist() == [3, 7]
    x = torch.zeros((1, 64), device=dev)
    x[0, 0] = torch.finfo(F32).max
    a = torch.zeros((1, 16, 64), dtype=BF16, device=dev)
    a[0, 0, 0] = 0.5
    b = torch.zeros((1, 64, 16), dtype=BF16, device=dev)
    b[0, :, 0] = 1.0
    assert (ops.lora_add(torch.zeros((1, 64), device=dev), x, a, b, ids[:1]) == x[0, 0] * 0.5).all()


@pytest.mark.gpu
@pytest.mark.parametrize("world", [2, 8])
@pytest.mark.parametrize("m", [3, 40])
def test_sharded_over_k(dev, world, m):
    """Every rank shrinks its slice, the ranks add the shrunk rows, every rank expands: as the whole."""
    from weightstream_b200 import ops, tp
    rng = np.random.default_rng(world)
    k, n, rank, adapters = 1024, 512, 16, 5
    x, y = make(rng, (m, k), BF16, dev), make(rng, (m, n), F32, dev)
    a, b = make(rng, (adapters, rank, k), BF16, dev, k ** -0.5), make(rng, (adapters, n, rank), BF16, dev, 0.3)
    ids, scale = batch(rng, m, adapters, dev), make(rng, (adapters,), F32, dev)
    grp = tp.LocalGroup(world, max_m=m, max_n=n)
    try:
        cuts = [tp.Sharding(world, r).slice_of(k) for r in range(world)]
        parts = [ops.lora_shrink(x[:, c:c + w], a[:, :, c:c + w].contiguous(), ids) for c, w in cuts]
        sums = grp.allreduce([p.reshape(-1) for p in parts])
        outs = [ops.lora_expand(y, s.reshape(m, rank), b, ids, scale) for s in sums]
        grp.check()
    finally:
        grp.close()
    _, _, want, err = ref(y, x, a, b, ids, scale)
    for o in outs:
        assert torch.equal(o, outs[0])
        close(o, want, err)


@pytest.mark.gpu
def test_no_rows_another_stream_and_a_graph(dev):
    from weightstream_b200 import ops
    rng = np.random.default_rng(3)
    a, b = make(rng, (4, 16, 256), BF16, dev, 0.1), make(rng, (4, 128, 16), BF16, dev, 0.1)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    assert ops.lora_add(torch.zeros((0, 128), device=dev), torch.zeros((0, 256), device=dev), a, b, none).shape == (0, 128)
    assert ops.lora_shrink(torch.zeros((0, 256), device=dev), a, none).shape == (0, 16)
    for m in (20, 500):
        x, y, ids = make(rng, (m, 256), BF16, dev), make(rng, (m, 128), F32, dev), batch(rng, m, 4, dev)
        want = ops.lora_add(y, x, a, b, ids)
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        outs = [ops.lora_add(y, x, a, b, ids, stream=s) for _ in range(3)]
        s.synchronize()
        assert all(torch.equal(o, want) for o in outs)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = ops.lora_add(y, x, a, b, ids)
        x.mul_(2.0)
        ids.copy_(ids.flip(0))
        g.replay()
        assert torch.equal(got, ops.lora_add(y, x, a, b, ids))


BAD = [
    (ValueError, dict(x=torch.zeros((3, 31), dtype=BF16))),
    (ValueError, dict(x=torch.zeros((2, 32), dtype=BF16))),
    (ValueError, dict(x=torch.zeros((3, 64), dtype=BF16)[:, ::2])),
    (TypeError, dict(x=torch.zeros((3, 32), dtype=torch.float16))),
    (ValueError, dict(y=torch.zeros((3, 15)))),
    (ValueError, dict(y=torch.zeros((1, 16)).expand(3, 16))),
    (TypeError, dict(a=torch.zeros((2, 8, 32)))),
    (ValueError, dict(a=torch.zeros((8, 32), dtype=BF16))),
    (ValueError, dict(a=torch.zeros((2, 32, 8), dtype=BF16).transpose(1, 2))),
    (ValueError, dict(a=torch.zeros((2, 4, 32), dtype=BF16))),
    (ValueError, dict(a=torch.zeros((3, 8, 32), dtype=BF16))),
    (ValueError, dict(a=torch.zeros((2, 129, 32), dtype=BF16), b=torch.zeros((2, 16, 129), dtype=BF16))),
    (ValueError, dict(a=torch.zeros((2, 0, 32), dtype=BF16), b=torch.zeros((2, 16, 0), dtype=BF16))),
    (ValueError, dict(a=torch.zeros((0, 8, 32), dtype=BF16), b=torch.zeros((0, 16, 8), dtype=BF16))),
    (TypeError, dict(ids=torch.zeros(3, dtype=torch.int64))),
    (ValueError, dict(ids=torch.zeros(2, dtype=torch.int32))),
    (ValueError, dict(ids=torch.zeros((3, 1), dtype=torch.int32))),
    (ValueError, dict(scale=torch.zeros(3))),
    (TypeError, dict(scale=torch.zeros(2, dtype=BF16))),
    (TypeError, dict(out=torch.zeros((3, 16), dtype=BF16))),
    (ValueError, dict(out=torch.zeros((3, 17)))),
]


def plain():
    return dict(y=torch.zeros((3, 16)), x=torch.zeros((3, 32), dtype=BF16), a=torch.zeros((2, 8, 32), dtype=BF16),
                b=torch.zeros((2, 16, 8), dtype=BF16), ids=torch.zeros(3, dtype=torch.int32), scale=torch.zeros(2))


@pytest.mark.parametrize("error,change", BAD)
def test_refuses(error, change):
    from weightstream_b200 import ops
    ops._lora_args(**plain())
    with pytest.raises(error):
        ops._lora_args(**{**plain(), **change})


@pytest.mark.parametrize("error,shrunk", [(ValueError, torch.zeros((3, 7))), (TypeError, torch.zeros((3, 8), dtype=BF16)),
                                          (ValueError, torch.zeros((3, 16))[:, ::2])])
def test_refuses_shrunk_rows(error, shrunk):
    from weightstream_b200 import ops
    half = {k: v for k, v in plain().items() if k not in ("x", "a")}
    ops._lora_args(**half, shrunk=torch.zeros((3, 8)))
    with pytest.raises(error):
        ops._lora_args(**half, shrunk=shrunk)


@pytest.mark.gpu
def test_calls_refuse(dev):
    from weightstream_b200 import ops

    def move(d):  # with the same strides
        put = lambda t: torch.zeros(max(t.untyped_storage().nbytes(), 16) // t.element_size(), dtype=t.dtype, device=dev).as_strided(t.size(), t.stride())
        return {k: put(v) if isinstance(v, torch.Tensor) else v for k, v in d.items()}

    ops.lora_add(**move(plain()))
    for error, change in BAD:
        with pytest.raises(error):
            ops.lora_add(**{**move(plain()), **move(change)})
    with pytest.raises(ValueError):
        ops.lora_add(**plain())
    with pytest.raises(ValueError):
        ops.lora_add(**{**move(plain()), "ids": plain()["ids"]})


@pytest.mark.gpu
def test_c_entry_refuses_a_short_workspace(dev):
    import ctypes as C
    from weightstream_b200 import _lib, ops
    L, err = _lib.load(), C.create_string_buffer(256)
    m = 513
    p = dict(y=torch.zeros((m, 16), device=dev), x=torch.zeros((m, 32), dtype=BF16, device=dev), a=torch.zeros((2, 8, 32), dtype=BF16, device=dev),
             b=torch.zeros((2, 16, 8), dtype=BF16, device=dev), ids=torch.zeros(m, dtype=torch.int32, device=dev))
    a = ops._lora_args(**p)
    a.out, a.ldo = p["y"].data_ptr(), 16
    need = L.ws_lora_workspace(m, 2, 8)
    work = torch.zeros(need + 16, dtype=torch.uint8, device=dev)
    for ptr, size in ((None, need), (work.data_ptr(), need - 1), (work.data_ptr() + 4, need)):
        a.workspace, a.workspace_bytes = ptr, size
        assert L.ws_lora_add(C.byref(a), None, err, len(err)) == _lib.WS_ERR_INVALID and b"workspace" in err.value


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 16, 32, 64, 128, 7])
@pytest.mark.parametrize("m", [20, 513, 600])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_shrunk_rows_at_any_float(dev, rank, m, offset):
    """Shrunk rows that begin anywhere in a buffer, as a view into what one all-reduce returned for several projections."""
    from weightstream_b200 import ops
    rng = np.random.default_rng(17 * rank + m + offset)
    y, b = make(rng, (m, 136), F32, dev), make(rng, (5, 136, rank), BF16, dev, 0.3)
    ids, scale = batch(rng, m, 5, dev), make(rng, (5,), F32, dev)
    many = make(rng, (offset + m * rank,), F32, dev)
    t = many[offset:].view(m, rank)
    assert t.is_contiguous() and t.data_ptr() % 16 == 4 * offset
    _, _, out, err = ref(y, None, None, b, ids, scale, shrunk=t)
    got = ops.lora_expand(y, t, b, ids, scale)
    close(got, out, err)
    assert torch.equal(got, ops.lora_expand(y, t.clone(), b, ids, scale))


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [1, 7, 8, 16, 24, 40, 72, 100])
@pytest.mark.parametrize("m", [1, 5, 200, 512, 600])
@pytest.mark.parametrize("xt", [F32, BF16])
def test_an_infinite_activation_is_infinite_at_any_rank(dev, rank, m, xt):
    """Positive weights and one infinite activation of a sign: the definition gives that infinity and no NaN, however many
    ranks a tile is filled up to."""
    from weightstream_b200 import ops
    rng = np.random.default_rng(rank + m)
    x, y = make(rng, (m, 72), xt, dev), make(rng, (m, 68), F32, dev)
    a, b = make(rng, (3, rank, 72), BF16, dev).abs() + 0.01, make(rng, (3, 68, rank), BF16, dev).abs() + 0.01
    ids = torch.arange(m, dtype=torch.int32, device=dev) % 3
    x[m // 2, 5], x[m - 1, 71] = float("inf"), -float("inf")
    for got in (ops.lora_add(y, x, a, b, ids), ops.lora_expand(y, ops.lora_shrink(x, a, ids), b, ids)):
        if m > 1:
            assert (got[m // 2] == float("inf")).all() and (got[m - 1] == -float("inf")).all()
        assert (~torch.isfinite(got).all(1)).nonzero().squeeze(1).tolist() == ([m // 2, m - 1] if m > 1 else [0])


@pytest.mark.gpu
@pytest.mark.parametrize("rank", [8, 32, 64, 128])
@pytest.mark.parametrize("xt", [F32, BF16])
def test_a_table_that_is_hardly_used(dev, rank, xt):
    """A sorted batch is worked on by the tiles that it has, not by those that its table has adapters for: the same bits
    with a few adapters and with many more that no token names."""
    from weightstream_b200 import ops
    rng = np.random.default_rng(rank)
    m, k, n = 600, 2304, 72
    x, y = make(rng, (m, k), xt, dev), make(rng, (m, n), F32, dev)
    a, b = make(rng, (16, rank, k), BF16, dev, k ** -0.5), make(rng, (16, n, rank), BF16, dev, 0.3)
    few = torch.from_numpy(rng.integers(0, 16, m).astype(np.int32)).to(dev)
    many_a, many_b = torch.zeros((900, rank, k), dtype=BF16, device=dev), torch.zeros((900, n, rank), dtype=BF16, device=dev)
    many_a[::60][:15], many_b[::60][:15] = a[:15], b[:15]
    many_a[899], many_b[899] = a[15], b[15]
    many = torch.where(few == 15, 899, few * 60).to(torch.int32)
    for ids, far in ((few, many), (torch.full_like(few, 15), torch.full_like(few, 899))):
        s, se, out, err = ref(y, x, a, b, ids, None)
        t = ops.lora_shrink(x, many_a, far)
        close(t, s, se)
        close(ops.lora_add(y, x, many_a, many_b, far), out, err)
        assert torch.equal(t, ops.lora_shrink(x, a, ids))
        assert torch.equal(ops.lora_add(y, x, many_a, many_b, far), ops.lora_add(y, x, a, b, ids))


@pytest.mark.gpu
@pytest.mark.parametrize("rank,k,xt", [(16, 2305, BF16), (32, 2304, F32), (64, 2304, BF16), (128, 1000, F32)])
@pytest.mark.parametrize("used", [1, 18, 19, 37, 38, 74, 75, 148, 149, 600])
def test_sorted_batches_of_any_number_of_tiles(dev, rank, k, xt, used):
    """Both sides of every number of tiles at which the work is split in another way: a tile an adapter here."""
    m = 601
    order = torch.from_numpy(np.random.default_rng(used).permutation(m).astype(np.int32)).to(dev)
    check(dev, m, k, 8, rank, 640, xt=xt, ids=order % used * (640 // used))
    check(dev, m, k, 8, rank, used, xt=xt, ids=torch.where(order < 40, -1, order % used).to(torch.int32))


@pytest.mark.gpu
@pytest.mark.parametrize("m,adapters", [(700, 4), (700, 400)])
def test_a_sorted_batch_on_another_stream_and_in_a_graph(dev, m, adapters):
    """More than 512 tokens: several launches that overlap, and a workspace that belongs to the call's stream."""
    from weightstream_b200 import ops
    rng = np.random.default_rng(30 + adapters)
    a, b = make(rng, (adapters, 16, 2048), BF16, dev, 0.1), make(rng, (adapters, 128, 16), BF16, dev, 0.1)
    x, y, ids = make(rng, (m, 2048), BF16, dev), make(rng, (m, 128), F32, dev), batch(rng, m, adapters, dev)
    want, rows = ops.lora_add(y, x, a, b, ids), ops.lora_shrink(x, a, ids)
    _, _, out, err = ref(y, x, a, b, ids, None)
    close(want, out, err)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    outs = []
    for _ in range(4):  # (each call's workspace is the one before's, freed on that stream)
        outs += [ops.lora_add(y, x, a, b, ids, stream=s)]
        t = ops.lora_shrink(x, a, ids, stream=s)
        outs += [ops.lora_expand(y, t, b, ids, stream=s)]
    s.synchronize()
    assert torch.equal(t, rows) and all(torch.equal(o, want) for o in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = ops.lora_add(y, x, a, b, ids)
        t = ops.lora_shrink(x, a, ids)
        halves = ops.lora_expand(y, t, b, ids)
    for _ in range(2):
        x.mul_(2.0)
        ids.copy_(ids.flip(0).clamp(max=adapters // 2))  # other tiles, and fewer
        g.replay()
        want = ops.lora_add(y, x, a, b, ids)
        torch.cuda.synchronize()
        assert torch.equal(got, want) and torch.equal(halves, want)


@pytest.mark.gpu
def test_a_sorted_batch_with_the_largest_table(dev):
    check(dev, 600, 64, 32, 8, 16384)
    check(dev, 600, 64, 32, 7, 16384, xt=F32)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4096, 4097, 4500, 9000])
@pytest.mark.parametrize("rank", [16, 12])
def test_more_tokens_than_the_plan_asks_for_at_once(dev, m, rank):
    check(dev, m, 72, 24, rank, 37)
    check(dev, m, 72, 24, rank, 3, xt=F32, yt=BF16)
    check(dev, m, 72, 24, rank, 2, ids=(torch.arange(m, dtype=torch.int32, device=dev) > 4094).to(torch.int32))
