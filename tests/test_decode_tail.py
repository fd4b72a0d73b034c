"""The operators and the tensor-parallel steps together, as examples/decode_tail.py runs them."""
import os
import sys

import numpy as np
import pytest

torch = pytest.importorskip("torch")

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
@pytest.mark.parametrize("m", [1, 6, 40])
def test_decode_tail(m):
    """Every operator's result is what its formula in 64 bits makes of the step's tensors around it."""
    if not torch.cuda.is_available():
        pytest.fail("a CUDA device is required for -m gpu tests")
    sys.path.insert(0, os.path.join(ROOT, "examples"))
    try:
        import decode_tail
    finally:
        sys.path.pop(0)
    from weightstream_b200 import ops, synth
    tail = decode_tail.DecodeTail()
    dev = tail.wo.device
    rng = np.random.default_rng(3)
    put = lambda *shape: torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dev).to(torch.bfloat16)
    attn, residual = put(m, tail.wo.shape[1]), put(m, tail.wo.shape[0])
    ids = torch.tensor([i % 5 - 1 for i in range(m)], dtype=torch.int32, device=dev)
    route_ids, route_w = (torch.from_numpy(a).to(dev) for a in synth.routes(rng, m, tail.experts, tail.top_k))
    calls = []

    def record(name):
        real = getattr(ops, name)

        def call(*args, **kw):
            seen = [a.clone() if isinstance(a, torch.Tensor) else a for a in args]
            out = real(*args, **kw)
            calls.append((name, seen, [t.clone() if isinstance(t, torch.Tensor) else t for t in (out if isinstance(out, tuple) else (out,))]))
            return out
        return call

    names = ("lora_add", "block_norm", "token_logprobs")
    kept = {n: getattr(ops, n) for n in names}
    try:
        for n in names:
            setattr(ops, n, record(n))
        greedy, scores = tail.step(attn, residual, ids, route_ids, route_w)
        tail.ep.check()
    finally:
        for n, f in kept.items():
            setattr(ops, n, f)
    assert [c[0] for c in calls] == ["lora_add", "block_norm", "block_norm", "token_logprobs"]
    d = lambda t: t.double().cpu()
    # adapters
    y, x, a, b, who, scale = calls[0][1]
    want = d(y)
    for t, i in enumerate(who.tolist()):
        if i >= 0:
            want[t] += float(scale[i]) * (d(b[i]) @ (d(a[i]) @ d(x[t])))
    assert (d(calls[0][2][0]) - want).abs().max() < 1e-4 * want.abs().max()
    # the gated block and the next one: the stream and what follows it (a bf16 rounding is within 2^-8)
    for call, post, nxt, gate in ((calls[1], 0, 1, tail.gate), (calls[2], 2, 3, None)):
        y, r = call[1]
        u = d(y) / torch.sqrt((d(y) ** 2).mean(1, keepdim=True) + 1e-6) * d(tail.norms[post])
        h = d(r) + (u if gate is None else u * torch.sigmoid(d(gate)))
        z = h / torch.sqrt((h ** 2).mean(1, keepdim=True) + 1e-6) * d(tail.norms[nxt])
        for got, ref in zip(call[2], (h, z)):
            assert ((d(got) - ref).abs() <= 2.0 ** -8 * ref.abs() + 1e-4).all()
    assert torch.equal(calls[2][2][0], residual)  # updated in place
    # scores
    logits, tok = calls[3][1]
    lp = torch.log_softmax(d(logits), 1)
    assert (d(scores.logprobs) - lp.gather(1, tok.long().cpu().unsqueeze(1)).squeeze(1)).abs().max() < 1e-4
    assert (scores.rank == 0).all() and torch.equal(scores.top_ids[:, 0], greedy)
    tail.close()
