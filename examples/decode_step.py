"""A decode step of one layer and the head, from the attention's queries and keys to the next token.

The reduction points run on an :class:`~weightstream_b200.tp.Endpoint`; between them stand the operators of
:mod:`weightstream_b200.ops`:

    queries, keys -> norms and rotation -> attention -> output projection + all-reduce -> norm, residual, norm
                  -> gate -> routes -> expert layer + all-reduce -> norm, residual, norm -> vocabulary head
                  -> biases, penalties, grammar -> greedy token -> its score

The attention itself is a few elementary operations over a small cache.  Run ``python examples/decode_step.py`` on a machine
with a B200; weights and activations are random, of small sizes.
"""
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from weightstream_b200 import ops, synth, tp  # noqa: E402


class DecodeStep:
    """Weights of one layer and of the head on one rank, random, and the requests' keys and values so far."""

    def __init__(self, *, m=6, hidden=1024, heads=16, kv_heads=4, head=64, expert=512, experts=8, top_k=2, vocab=8192, past=40, seed=0):
        self.dev = torch.device("cuda", torch.cuda.current_device())
        rng = np.random.default_rng(seed)
        put = lambda a: torch.from_numpy(a).to(self.dev)
        normal = lambda *shape, scale=1.0: put(rng.standard_normal(shape).astype(np.float32) * scale).to(torch.bfloat16)
        self.m, self.heads, self.kv_heads, self.head, self.top_k, self.vocab = m, heads, kv_heads, head, top_k, vocab
        self.ep = tp.Endpoint(max_m=max(m, 1), max_n=hidden, max_vocab=vocab)
        self.wqkv = normal(hidden, (heads + 2 * kv_heads) * head, scale=hidden ** -0.5)
        self.q_norm, self.k_norm = normal(head, scale=0.1) + 1.0, normal(head, scale=0.1) + 1.0
        self.inv_freq = (1e4 ** (-torch.arange(head // 2, device=self.dev, dtype=torch.float64) / (head // 2))).float()
        self.wo, self.wo_scales = (put(a) for a in synth.fp8_weight(rng, hidden, heads * head))
        self.norms = [normal(hidden, scale=0.1) + 1.0 for _ in range(4)]
        self.gate = normal(hidden, experts, scale=hidden ** -0.5)
        self.gate_bias = put(rng.standard_normal(experts).astype(np.float32) * 0.1)
        # gate and up products of an expert as halves of one tensor
        (w13, s13), (w2, s2) = synth.fp4_experts(rng, experts, 2 * expert, hidden), synth.fp4_experts(rng, experts, hidden, expert)
        self.w13, self.s13, self.w2, self.s2 = put(w13), put(s13), put(w2), put(s2)
        self.expert = expert
        self.head_w, self.head_scales = (put(a) for a in synth.fp8_weight(rng, vocab, hidden))
        self.keys, self.values = normal(m, kv_heads, past, head), normal(m, kv_heads, past, head)

    def step(self, x, residual, positions, *, tokens, offsets, repetition, mask=None, mask_rows=None, bias=None):
        """``x`` [m, hidden] bf16 is the layer's normalised input, ``residual`` its stream (updated in place); ``tokens`` and
        ``offsets`` the requests' histories.  Returns the greedy tokens and their scores under what was asked of the logits."""
        qkv = (x @ self.wqkv).unflatten(1, (-1, self.head))
        q, k = ops.head_norm_rope(qkv[:, :self.heads], qkv[:, self.heads:self.heads + self.kv_heads], positions=positions, inv_freq=self.inv_freq,
                                  q_weight=self.q_norm, k_weight=self.k_norm)
        self.keys, self.values = (torch.cat([old, new.unsqueeze(2)], 2) for old, new in ((self.keys, k), (self.values, qkv[:, self.heads + self.kv_heads:])))
        q = q.unflatten(1, (self.kv_heads, -1)).float()
        p = torch.softmax(q @ self.keys.float().transpose(2, 3) * self.head ** -0.5, 3)
        attn = (p @ self.values.float()).to(torch.bfloat16).flatten(1)
        y = self.ep.fp8_rowpar_gemm_allreduce(attn, self.wo, self.wo_scales)
        _, x = ops.block_norm(y, residual, post_weight=self.norms[0], next_weight=self.norms[1], out=residual)
        ids, w = ops.moe_route((x @ self.gate).float(), self.top_k, score="sqrtsoftplus", bias=self.gate_bias, scale=1.5)
        f = self.expert
        y = ops.moe_layer(x, ids, w, self.w13[:, :f], self.s13[:, :f], self.w13[:, f:], self.s13[:, f:], self.w2, self.s2, limit=10.0)
        y = self.ep.allreduce_(y)
        _, x = ops.block_norm(y, residual, post_weight=self.norms[2], next_weight=self.norms[3], out=residual)
        logits, _ = self.ep.lm_head_allgather_argmax(x, self.head_w, self.head_scales, vocab_row0=0, vocab=self.vocab)
        more = {} if bias is None else dict(zip(("bias_ids", "bias", "bias_offsets"), bias))
        logits = ops.adjust_logits(logits, tokens=tokens, offsets=offsets, repetition=repetition, mask=mask, mask_rows=mask_rows, out=logits, **more)
        greedy = logits.argmax(1)
        return greedy, ops.token_logprobs(logits, greedy, top=3)

    def close(self):
        self.ep.check()
        self.ep.close()


def main(m=6):
    layer = DecodeStep(m=m)
    dev = layer.dev
    rng = np.random.default_rng(1)
    put = lambda a, t: torch.from_numpy(np.asarray(a)).to(dev).to(t)
    x, residual = (put(rng.standard_normal((m, layer.wqkv.shape[0])), torch.bfloat16) for _ in range(2))
    lengths = rng.integers(5, 40, m)
    mask = put(rng.integers(-2 ** 31, 2 ** 31, (2, layer.vocab // 32)), torch.int32)
    greedy, scores = layer.step(x, residual, put(1000 + np.arange(m), torch.int64), tokens=put(rng.integers(0, layer.vocab, lengths.sum()), torch.int32),
                                offsets=put(np.concatenate([[0], np.cumsum(lengths)]), torch.int32), repetition=put(np.full(m, 1.2), torch.float32), mask=mask,
                                mask_rows=put(np.arange(m) % 3 - 1, torch.int32))
    for t in range(m):
        print(f"token {int(greedy[t])}  log probability {float(scores.logprobs[t]):.3f}  entropy {float(scores.entropy[t]):.3f}")
    layer.close()
    return greedy, scores


if __name__ == "__main__":
    main()
