"""What the operators around the reduction points ask of their callers, and what their C entries refuse by themselves."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")

from weightstream_b200 import _lib  # noqa: E402


def calls():
    from weightstream_b200 import ops
    x, b = torch.zeros((3, 64)), lambda *shape: torch.zeros(shape, dtype=torch.uint8)
    return {"head_norm_rope": (ops.head_norm_rope, dict(q=torch.zeros((3, 2, 8)))),
            "moe_route": (ops.moe_route, dict(logits=x, top_k=2)),
            "moe_layer": (ops.moe_layer, dict(x=x, route_ids=torch.zeros((3, 2), dtype=torch.int32), route_w=torch.zeros((3, 2)), w1=b(4, 32, 32), s1=b(4, 32, 2),
                                              w3=b(4, 32, 32), s3=b(4, 32, 2), w2=b(4, 64, 16), s2=b(4, 64, 1))),
            "adjust_logits": (ops.adjust_logits, dict(logits=x))}


NAMES = ["head_norm_rope", "moe_route", "moe_layer", "adjust_logits"]


class StreamOf:
    def __init__(self, device):
        self.device, self.used = torch.device(device), False

    @property
    def cuda_stream(self):
        self.used = True
        return 0


@pytest.mark.parametrize("name", NAMES)
def test_a_stream_of_another_device_is_refused(name):
    f, args = calls()[name]
    s = StreamOf("cuda:1")
    with pytest.raises(ValueError, match="stream of cuda:1"):
        f(**args, stream=s)
    assert not s.used


@pytest.mark.parametrize("name", NAMES)
def test_what_is_no_tensor_is_a_type_error(name):
    f, args = calls()[name]
    for missing in [k for k, v in args.items() if isinstance(v, torch.Tensor)]:
        for value in (None, [1.0, 2.0]):
            with pytest.raises(TypeError, match=missing):
                f(**{**args, missing: value})


def refused(name, args, status=_lib.WS_ERR_INVALID, text=""):
    err = C.create_string_buffer(256)
    st = getattr(_lib.load(), name)(C.byref(args), None, err, len(err))
    assert st == status and text in err.value.decode(), (st, err.value)


def fill(cls, **values):
    a = cls()
    for k, v in values.items():
        setattr(a, k, v)
    return a


P = 1 << 20         # an address that is only looked at


@pytest.mark.parametrize("change,status", [
    (dict(m=-1), -1), (dict(d=0), -1), (dict(start=1), -1), (dict(pairs=-1), -1), (dict(pairs=1025, d=4096), -5), (dict(dtype=2), -1), (dict(weight_dtype=-1), -1),
    (dict(position_bytes=2), -1), (dict(eps=-1.0), -1), (dict(q=None), -1), (dict(q_out=None), -1), (dict(k_out=None), -1), (dict(positions=None), -1),
    (dict(inv_freq=None), -1), (dict(q=P + 2), -1), (dict(positions=P + 4), -1), (dict(q_weight=P + 1, weight_dtype=0), -1), (dict(q_heads=1 << 25), -1),
])
def test_heads_entry_refuses(change, status):
    base = dict(q=P, k=P, q_out=P, k_out=P, positions=P, inv_freq=P, m=2, q_heads=2, k_heads=1, d=16, pairs=8, dtype=1, weight_dtype=1, position_bytes=8, norm=1)
    refused("ws_head_norm_rope", fill(_lib.HeadNormRopeArgs, **{**base, **change}), status)


@pytest.mark.parametrize("change,status", [
    (dict(m=-1), -1), (dict(experts=0), -1), (dict(top_k=0), -1), (dict(top_k=9), -1), (dict(experts=1025, ld=1025), -5), (dict(experts=64, ld=64, top_k=33), -5), (dict(score=3), -1),
    (dict(dtype=5), -1), (dict(logits=None), -1), (dict(ids=None), -1), (dict(weights=None), -1), (dict(ld=7), -1), (dict(logits=P + 1), -1), (dict(bias=P + 2), -1),
])
def test_route_entry_refuses(change, status):
    base = dict(logits=P, ids=P, weights=P, ld=8, m=1, experts=8, top_k=2, dtype=1)
    refused("ws_moe_route", fill(_lib.MoeRouteArgs, **{**base, **change}), status)


@pytest.mark.parametrize("change,status", [
    (dict(m=-1), -1), (dict(hidden=48), -1), (dict(inter=0), -1), (dict(top_k=0), -1), (dict(top_k=9), -5), (dict(m=257), -5), (dict(e_len=0), -1), (dict(e_len=513), -5),
    (dict(e_start=-1), -1), (dict(hidden=24608, ldx=24608, ldo=24608), -5), (dict(x_dtype=3), -1), (dict(out_dtype=-1), -1), (dict(x=None), -1), (dict(s3=None), -1), (dict(out=None), -1),
    (dict(ldx=63), -1), (dict(ldo=63), -1), (dict(w1=P + 8), -1), (dict(s2_stride=24), -1), (dict(w2_stride=16), -1), (dict(workspace=None), -1), (dict(workspace=P + 8), -1),
    (dict(workspace_bytes=100), -1), (dict(route_w=P + 1), -1), (dict(x=P + 2), -1),
])
def test_layer_entry_refuses(change, status):
    base = dict(x=P, ldx=64, route_ids=P, route_w=P, w1=P, s1=P, w3=P, s3=P, w2=P, s2=P, w1_stride=1024, s1_stride=64, w3_stride=1024, s3_stride=64, w2_stride=1024, s2_stride=64,
                out=P, ldo=64, workspace=P, workspace_bytes=1 << 20, m=3, hidden=64, inter=32, top_k=2, e_len=4, x_dtype=1, out_dtype=1)
    refused("ws_moe_layer", fill(_lib.MoeLayerArgs, **{**base, **change}), status)


@pytest.mark.parametrize("change", [
    dict(m=-1), dict(vocab=0), dict(vocab=2 ** 31 - 1), dict(dtype=2), dict(offset_bytes=2), dict(bias_offset_bytes=0), dict(n_tokens=-1), dict(n_bias=-1), dict(n_bias=2 ** 31),
    dict(mask_count=-1), dict(logits=None), dict(out=None), dict(offsets=None), dict(bias=None), dict(bias_offsets=None), dict(ld=39), dict(ldo=39), dict(ld_mask=1),
    dict(logits=P + 2), dict(out=P + 1), dict(tokens=P + 2), dict(offsets=P + 4), dict(mask=P + 1), dict(repetition=P + 2), dict(mask_rows=P + 3),
])
def test_adjust_entry_refuses(change):
    base = dict(logits=P, out=P, ld=40, ldo=40, tokens=P, offsets=P, bias_ids=P, bias=P, bias_offsets=P, mask=P, n_tokens=5, n_bias=5, ld_mask=2, m=2, vocab=40, mask_count=2,
                offset_bytes=8, bias_offset_bytes=8, dtype=1)
    refused("ws_adjust_logits", fill(_lib.AdjustLogitsArgs, **{**base, **change}))


def test_null_arguments_and_no_rows():
    L = _lib.load()
    for name, cls in (("ws_head_norm_rope", _lib.HeadNormRopeArgs), ("ws_moe_route", _lib.MoeRouteArgs), ("ws_moe_layer", _lib.MoeLayerArgs), ("ws_adjust_logits", _lib.AdjustLogitsArgs)):
        err = C.create_string_buffer(64)
        assert getattr(L, name)(None, None, err, len(err)) == _lib.WS_ERR_INVALID and err.value == b"null args"
        assert getattr(L, name)(None, None, None, 0) == _lib.WS_ERR_INVALID
    refused("ws_head_norm_rope", fill(_lib.HeadNormRopeArgs, d=8, dtype=1, weight_dtype=1, position_bytes=4), _lib.WS_OK)
    refused("ws_moe_route", fill(_lib.MoeRouteArgs, experts=8, top_k=1, dtype=1), _lib.WS_OK)
    refused("ws_moe_layer", fill(_lib.MoeLayerArgs, hidden=64, inter=32, top_k=1, e_len=1, x_dtype=1, out_dtype=1), _lib.WS_OK)
    refused("ws_adjust_logits", fill(_lib.AdjustLogitsArgs, vocab=8, dtype=1), _lib.WS_OK)
    assert L.ws_moe_layer_workspace(0, 6, 64, 64) == 0 and L.ws_moe_layer_workspace(2, 3, 64, 32) == 6 * 32 * 4 + 6 * 64 * 4


FAR = (1 << 31) + 64        # elements of two bytes: rows that many apart are more than 2^32 bytes apart


@pytest.fixture()
def dev():
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    return torch.device("cuda:0")


def far_apart(t, stride):
    """The same values, those of the first dimension `stride` elements apart."""
    room = torch.empty(1 + (t.shape[0] - 1) * stride + sum((n - 1) * k for n, k in zip(t.shape[1:], t.stride()[1:])), dtype=t.dtype, device=t.device)
    far = room.as_strided(t.shape, (stride, *t.stride()[1:]))
    far.copy_(t)
    return far


@pytest.mark.gpu
def test_rows_and_experts_past_32_bits(dev):
    """Offsets that do not fit in 32 bits, in elements and in bytes: the results are those of compact tensors."""
    from weightstream_b200 import ops
    g = torch.Generator(dev).manual_seed(5)
    normal = lambda *shape: torch.randn(shape, generator=g, device=dev).bfloat16()
    whole = lambda lo, hi, *shape: torch.randint(lo, hi, shape, generator=g, device=dev, dtype=torch.uint8)
    x = normal(2, 640)
    mask = torch.randint(-2 ** 31, 2 ** 31 - 1, (2, 20), generator=g, device=dev, dtype=torch.int32)
    tokens, offsets = torch.tensor([3, 3, 639, 5], dtype=torch.int32, device=dev), torch.tensor([0, 2, 4], dtype=torch.int32, device=dev)
    how = dict(tokens=tokens, offsets=offsets, frequency=torch.full((2,), 0.5, device=dev), mask=mask)
    assert torch.equal(ops.adjust_logits(far_apart(x, FAR), out=far_apart(x, FAR), **how), ops.adjust_logits(x, **how))
    for got, want in zip(ops.moe_route(far_apart(x, FAR), 8), ops.moe_route(x, 8)):
        assert torch.equal(got, want)
    q = normal(2, 3, 128)
    how = dict(positions=torch.tensor([7, 1000], dtype=torch.int32, device=dev), inv_freq=10000.0 ** (-torch.arange(64, device=dev) / 64))
    assert torch.equal(ops.head_norm_rope(far_apart(q, FAR), q_out=far_apart(q, FAR), **how)[0], ops.head_norm_rope(q, **how)[0])
    odd = q[:, :, :126]
    how["inv_freq"] = how["inv_freq"][:63].contiguous()
    assert torch.equal(ops.head_norm_rope(far_apart(odd, FAR), q_out=far_apart(odd, FAR), **how)[0], ops.head_norm_rope(odd, **how)[0])
    x = normal(2, 256)
    ids, w = torch.tensor([[0, 1], [1, 0]], dtype=torch.int32, device=dev), torch.rand((2, 2), generator=g, device=dev)
    weights = [f(*shape) for shape, f in zip([(2, 64, 128), (2, 64, 8), (2, 64, 128), (2, 64, 8), (2, 256, 32), (2, 256, 2)], [lambda *n: whole(0, 256, *n), lambda *n: whole(126, 129, *n)] * 3)]
    want = ops.moe_layer(x, ids, w, *weights)
    far = [far_apart(t, 2 * FAR) for t in weights]
    assert torch.equal(ops.moe_layer(far_apart(x, FAR), ids, w, *far, out=far_apart(torch.zeros_like(want), FAR)), want)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [2 ** 31, 2 ** 32 + 1, 2 ** 63, -2 ** 70])
def test_whole_numbers_beyond_a_word_are_value_errors(dev, value):
    """Of device tensors too, which the native front end takes first."""
    from weightstream_b200 import ops
    f, args = calls()["moe_layer"]
    args = {k: v.to(dev) for k, v in args.items()}
    with pytest.raises(ValueError, match="e_start"):
        f(**args, e_start=value)
    with pytest.raises(ValueError, match="top_k"):
        ops.moe_route(args["x"], value)
    with pytest.raises(ValueError, match="top"):
        ops.token_logprobs(args["x"], torch.zeros(3, dtype=torch.int32, device=dev), top=value)


def test_layer_entry_refuses_a_limit_that_is_no_number():
    base = dict(x=P, ldx=64, route_ids=P, route_w=P, w1=P, s1=P, w3=P, s3=P, w2=P, s2=P, w1_stride=1024, s1_stride=64, w3_stride=1024, s3_stride=64, w2_stride=1024, s2_stride=64,
                out=P, ldo=64, workspace=P, workspace_bytes=1 << 20, m=3, hidden=64, inter=32, top_k=2, e_len=4, x_dtype=1, out_dtype=1, limit=float("nan"))
    refused("ws_moe_layer", fill(_lib.MoeLayerArgs, **base), text="limit")
