"""What all operators of :mod:`weightstream_b200.ops` ask of their callers."""
import pytest

torch = pytest.importorskip("torch")

BF16 = torch.bfloat16


def calls():
    """Name, function and arguments of every operator, on the host."""
    from weightstream_b200 import ops
    y, x, ids = torch.zeros((3, 16)), torch.zeros((3, 32), dtype=BF16), torch.zeros(3, dtype=torch.int32)
    a, b = torch.zeros((2, 8, 32), dtype=BF16), torch.zeros((2, 16, 8), dtype=BF16)
    return [("block_norm", ops.block_norm, dict(y=y)),
            ("lora_add", ops.lora_add, dict(y=y, x=x, a=a, b=b, ids=ids)),
            ("lora_shrink", ops.lora_shrink, dict(x=x, a=a, ids=ids)),
            ("lora_expand", ops.lora_expand, dict(y=y, shrunk=torch.zeros((3, 8)), b=b, ids=ids)),
            ("token_logprobs", ops.token_logprobs, dict(logits=y, tokens=ids))]


NAMES = ["block_norm", "lora_add", "lora_shrink", "lora_expand", "token_logprobs"]


class StreamOf:
    """What a call looks at before it uses a stream."""

    def __init__(self, device):
        self.device, self.used = torch.device(device), False

    @property
    def cuda_stream(self):
        self.used = True
        return 0


@pytest.mark.parametrize("name", NAMES)
def test_a_stream_of_another_device_is_refused(name):
    """Before its handle goes anywhere, so that no device is handed another one's memory."""
    f, args = next((f, a) for n, f, a in calls() if n == name)
    s = StreamOf("cuda:1")
    with pytest.raises(ValueError, match="stream of cuda:1"):
        f(**args, stream=s)
    assert not s.used


@pytest.mark.parametrize("name", NAMES)
def test_what_is_no_tensor_is_a_type_error(name):
    f, args = next((f, a) for n, f, a in calls() if n == name)
    for missing in args:
        for value in (None, [1.0, 2.0]):
            with pytest.raises(TypeError, match=missing):
                f(**{**args, missing: value})
    for more in {"block_norm": ("residual", "post_weight", "next_weight", "gate", "out"), "lora_add": ("scale", "out"),
                 "lora_expand": ("scale", "out")}.get(name, ()):
        with pytest.raises(TypeError, match=more):
            f(**{**args, more: [1.0, 2.0]})
