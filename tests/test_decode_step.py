"""The operators of a decode step together with the tensor-parallel steps, as examples/decode_step.py runs them."""
import math
import os
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

from weightstream_b200 import formats  # noqa: E402

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import decode_step
    finally:
        sys.path.pop(0)
    return decode_step


class Recorder:
    """Arguments and results of the operators that a step calls."""

    def __init__(self, ops, names):
        self.ops, self.kept, self.calls = ops, {n: getattr(ops, n) for n in names}, []

    def __enter__(self):
        for name, real in self.kept.items():
            def call(*args, _name=name, _real=real, **kw):
                keep = lambda v: v.clone() if isinstance(v, torch.Tensor) else v
                seen = ([keep(a) for a in args], {k: keep(v) for k, v in kw.items()})
                out = _real(*args, **kw)
                self.calls.append((_name, *seen, [keep(t) for t in (out if isinstance(out, tuple) else (out,))]))
                return out
            setattr(self.ops, name, call)
        return self

    def __exit__(self, *_):
        for name, real in self.kept.items():
            setattr(self.ops, name, real)


def d(t):
    return t.double().cpu()


def rotated(x, w, positions, inv_freq):
    v = d(x)
    v = v / torch.sqrt((v * v).mean(2, keepdim=True) + 1e-6) * d(w)
    f = inv_freq.shape[0]
    angle = (d(positions)[:, None] * d(inv_freq))[:, None]
    a, b = v[..., :f], v[..., f:]
    return torch.cat([a * torch.cos(angle) - b * torch.sin(angle), a * torch.sin(angle) + b * torch.cos(angle)], 2)


def widen(w, s):
    codes = torch.stack([w & 15, w >> 4], -1).flatten(-2).cpu().numpy()
    scale = np.ldexp(1.0, s.cpu().numpy().astype(np.int64) - 127)
    return torch.from_numpy(formats.FP4_TABLE.astype(np.float64)[codes] * np.repeat(scale, 32, axis=2))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 6, 33])
def test_decode_step(m):
    """Every operator's result is what its formula in 64 bits makes of the step's tensors around it."""
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    from weightstream_b200 import ops
    layer = example().DecodeStep(m=m)
    dev, rng = layer.dev, np.random.default_rng(3)
    put = lambda a, t: torch.from_numpy(np.asarray(a)).to(dev).to(t)
    x, residual = (put(rng.standard_normal((m, layer.wqkv.shape[0])), torch.bfloat16) for _ in range(2))
    lengths = rng.integers(0, 60, m)
    history = dict(tokens=put(rng.integers(0, 300, lengths.sum()), torch.int32), offsets=put(np.concatenate([[0], np.cumsum(lengths)]), torch.int32),
                   repetition=put(1.0 + rng.random(m), torch.float32), mask=put(rng.integers(-2 ** 31, 2 ** 31, (2, layer.vocab // 32)), torch.int32),
                   mask_rows=put(np.arange(m) % 3 - 1, torch.int32),
                   bias=(put(np.arange(m), torch.int32), put(np.full(m, 5.0), torch.float32), put(np.arange(m + 1), torch.int32)))
    for turn in range(2):                                                   # the second step reads the keys of the first
        with Recorder(ops, ("head_norm_rope", "moe_route", "moe_layer", "adjust_logits", "token_logprobs")) as seen:
            greedy, scores = layer.step(x, residual, put(100000 + turn + np.arange(m), torch.int64), **history)
        layer.ep.check()
        assert [c[0] for c in seen.calls] == ["head_norm_rope", "moe_route", "moe_layer", "adjust_logits", "token_logprobs"]
        heads, route, experts, adjust, _ = seen.calls
        # queries and keys (a bf16 rounding is within 2^-8)
        for x_in, w, got in zip(heads[1], (layer.q_norm, layer.k_norm), heads[3]):
            want = rotated(x_in, w, heads[2]["positions"], layer.inv_freq)
            assert ((d(got) - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()
        # routes
        score = torch.sqrt(torch.log1p(torch.exp(d(route[1][0]))))
        order = torch.sort(score + d(layer.gate_bias), dim=1, descending=True, stable=True).indices[:, :layer.top_k]
        w = score.gather(1, order)
        assert torch.equal(route[3][0].long().cpu(), order)
        assert (d(route[3][1]) - 1.5 * w / w.sum(1, keepdim=True)).abs().max() < 1e-5
        # experts
        f = layer.expert
        w13, w2 = widen(layer.w13, layer.s13), widen(layer.w2, layer.s2)
        want = torch.zeros(experts[3][0].shape, dtype=torch.float64)
        for t in range(m):
            for e, weight in zip(order[t].tolist(), d(route[3][1])[t]):
                g, u = (w13[e] @ d(experts[1][0])[t]).split(f)
                want[t] += w2[e] @ (weight * torch.nn.functional.silu(g.clamp(max=10.0)) * u.clamp(-10.0, 10.0))
        assert (d(experts[3][0]) - want).abs().max() < 1e-4 * want.abs().max()
        # logits
        z, got = d(adjust[1][0]), d(adjust[3][0])
        for t in range(m):
            z[t, t] += 5.0
            one = history["tokens"][history["offsets"][t]:history["offsets"][t + 1]].long().cpu().unique()
            r = float(history["repetition"][t])
            z[t, one] = torch.where(z[t, one] > 0, z[t, one] / r, z[t, one] * r)
            if t % 3:
                bits = history["mask"][t % 3 - 1].cpu().numpy().view(np.uint32)
                v = np.arange(layer.vocab)
                z[t, torch.from_numpy((bits[v >> 5] >> (v & 31).astype(np.uint32) & 1) == 0)] = -math.inf
        fine = torch.isfinite(z)
        assert torch.equal(fine, torch.isfinite(got)) and (got - z)[fine].abs().max() < 1e-4
        assert torch.equal(greedy.cpu(), got.argmax(1)) and (scores.rank == 0).all()
    layer.close()


@pytest.mark.gpu
def test_example_runs():
    greedy, scores = example().main(3)
    assert greedy.shape == (3,) and torch.isfinite(scores.logprobs).all()
