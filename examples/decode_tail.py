"""The tail of a decode step: everything from the attention's heads to the sampled token's score.

One layer's reduction points and the vocabulary head run on an :class:`~weightstream_b200.tp.Endpoint`; between them stand
the operators of :mod:`weightstream_b200.ops`:

    heads -> output projection + all-reduce -> adapters of the requests -> norm, gate, residual, norm
          -> routed experts + combine + all-reduce -> norm, residual, norm -> vocabulary head -> scores

Run ``python examples/decode_tail.py`` on a machine with a B200; weights and activations are random, of small sizes.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from weightstream_b200 import ops, synth, tp  # noqa: E402


class DecodeTail:
    """Weights of one layer's tail and of the head on one rank, random."""

    def __init__(self, *, hidden=1024, heads=2048, expert=512, experts=8, top_k=2, vocab=8192, rank=16, adapters=4, max_m=64, seed=0):
        dev = torch.device("cuda", torch.cuda.current_device())
        rng = np.random.default_rng(seed)
        put = lambda a: torch.from_numpy(a).to(dev)
        normal = lambda *shape, scale=1.0: put(rng.standard_normal(shape).astype(np.float32) * scale).to(torch.bfloat16)
        self.vocab, self.experts, self.top_k = vocab, experts, top_k
        self.ep = tp.Endpoint(max_m=max_m, max_n=hidden, max_vocab=vocab)
        self.wo, self.wo_scales = (put(a) for a in synth.fp8_weight(rng, hidden, heads))
        self.w2, self.s2 = (put(a) for a in synth.fp4_experts(rng, experts, hidden, expert))
        self.head, self.head_scales = (put(a) for a in synth.fp8_weight(rng, vocab, hidden))
        self.lora_a, self.lora_b = normal(adapters, rank, heads, scale=heads ** -0.5), normal(adapters, hidden, rank, scale=0.1)
        self.lora_scale = torch.full((adapters,), 2.0, device=dev)
        self.norms = [normal(hidden, scale=0.1) + 1.0 for _ in range(4)]
        self.gate = normal(hidden)
        self.up = normal(hidden, expert, scale=hidden ** -0.5)      # stands in for the experts' first product

    def step(self, attn, residual, ids, route_ids, route_w, tokens=None, top=5):
        """``attn`` [m, heads] bf16, ``residual`` [m, hidden] bf16 (updated in place), ``ids`` [m] adapters, routes [m, top_k].

        Returns the greedy tokens and the scores of ``tokens`` (of the greedy ones if None)."""
        y = self.ep.fp8_rowpar_gemm_allreduce(attn, self.wo, self.wo_scales)
        y = ops.lora_add(y, attn, self.lora_a, self.lora_b, ids, self.lora_scale, out=y)
        _, x = ops.block_norm(y, residual, post_weight=self.norms[0], next_weight=self.norms[1], gate=self.gate, gate_act="sigmoid",
                              out=residual)
        h = torch.nn.functional.silu(x @ self.up).repeat_interleave(self.top_k, 0)
        y = self.ep.moe_down_combine_allreduce(h, route_ids, route_w, self.w2, self.s2, 0)
        _, x = ops.block_norm(y, residual, post_weight=self.norms[2], next_weight=self.norms[3], out=residual)
        logits, greedy = self.ep.lm_head_allgather_argmax(x, self.head, self.head_scales, vocab_row0=0, vocab=self.vocab)
        return greedy, ops.token_logprobs(logits, greedy if tokens is None else tokens, top=top)

    def close(self):
        self.ep.check()
        self.ep.close()


def main(m=6):
    tail = DecodeTail()
    dev = tail.wo.device
    rng = np.random.default_rng(1)
    attn = torch.from_numpy(rng.standard_normal((m, tail.wo.shape[1])).astype(np.float32)).to(dev).to(torch.bfloat16)
    residual = torch.from_numpy(rng.standard_normal((m, tail.wo.shape[0])).astype(np.float32)).to(dev).to(torch.bfloat16)
    ids = torch.tensor([i % 5 - 1 for i in range(m)], dtype=torch.int32, device=dev)        # -1: no adapter
    route_ids, route_w = (torch.from_numpy(a).to(dev) for a in synth.routes(rng, m, tail.experts, tail.top_k))
    greedy, scores = tail.step(attn, residual, ids, route_ids, route_w)
    for t in range(m):
        best = ", ".join(f"{i}: {p:.2f}" for i, p in zip(scores.top_ids[t].tolist(), scores.top_logprobs[t].tolist()))
        print(f"token {int(greedy[t])}  log probability {float(scores.logprobs[t]):.3f}  entropy {float(scores.entropy[t]):.3f}  best {best}")
    tail.close()
    return greedy, scores


if __name__ == "__main__":
    main()
