"""Workloads of the operators between the tensor-parallel steps, for timing and for comparing them with plain forms.

Three operators stand around the reduction points of ``weightstream_b200.tp``: the norms, gate and residual between
two blocks (``ops.block_norm``), low-rank adapters of many requests beside a shared projection (``ops.lora_add``, and
``ops.lora_shrink`` / ``ops.lora_expand`` where the projection is sharded over K), and the scores of given tokens on
the vocabulary head's logits (``ops.token_logprobs``).

``own`` chooses between the framework's operators and the same formulas in elementary torch operations in 32 bits.
"""
import math

import torch

own = False

HIDDEN, K_PROJ = 7168, 8192             # attention output projection
HIDDEN_NATIVE, K_NATIVE = 5120, 2304    # the reference model's own widths
VOCAB = 129280
EPS = 1e-6
NORM_BYTES_MAX = 8192 * HIDDEN * 12     # the largest listed case of each operator bounds the drawn ones
LORA_WORK_MAX = 4000 * 64 * (K_PROJ + HIDDEN)
SCORES_MAX = 2000 * VOCAB


def _norm(name, m, n, y="f32", res="bf16", gate="none", post=True, out="bf16"):
    return {"name": name, "op": "norm", "m": m, "n": n, "y": y, "res": res, "gate": gate, "post": post, "out": out}


def _lora(name, m, k, n, rank, adapters, used, batch, act="bf16", out="f32", op="lora"):
    return {"name": name, "op": op, "m": m, "k": k, "n": n, "rank": rank, "adapters": adapters, "used": used, "batch": batch,
            "act": act, "out": out}


def _scores(name, m, vocab, top, dtype="f32", masked=False):
    return {"name": name, "op": "scores", "m": m, "vocab": vocab, "top": top, "dtype": dtype, "masked": masked}


def listed():
    return [
        # One decoded token between attention and experts: fp32 sums of the projection in, bf16 activations out.
        _norm("norm_row", 1, HIDDEN),
        # A ragged serving batch at the reference model's own width, with a gate a channel and a fp32 residual stream.
        _norm("norm_batch", 61, HIDDEN_NATIVE, res="f32", gate="channel"),
        # A prompt: a gate for every value.
        _norm("norm_prefill", 8192, HIDDEN, gate="full"),
        # A width that no vector divides, bf16 block output, one gate a token, no norm of the block's output.
        _norm("norm_odd", 1503, 2307, y="bf16", gate="token", post=False, out="f32"),
        # One decoded token with an adapter on the attention output projection.
        _lora("lora_row", 1, K_PROJ, HIDDEN, 16, 8, 1, "decode"),
        # A serving batch: every request has its adapter, several share one, some have none.
        _lora("lora_batch", 64, K_PROJ, HIDDEN, 16, 48, 24, "decode"),
        # Prompts of a few requests one after the other.
        _lora("lora_prefill", 4000, K_PROJ, HIDDEN, 64, 8, 5, "prompts"),
        # The reference's own expert shape, fp32 activations and a narrow rank; the projection's result is bf16.
        _lora("lora_native", 333, K_NATIVE, HIDDEN_NATIVE, 8, 32, 20, "decode", act="f32", out="bf16"),
        # One rank of eight: its K slice is shrunk, the sums would be exchanged, every rank expands them.
        _lora("lora_shard", 40, K_PROJ // 8, HIDDEN, 32, 24, 12, "decode", op="lora_shard"),
        # One decoded token's score with the alternatives that an answer lists.
        _scores("scores_row", 1, VOCAB, 20),
        # A serving batch.
        _scores("scores_batch", 64, VOCAB, 5),
        # Every token of a prompt, without alternatives.
        _scores("scores_prompt", 2000, VOCAB, 0),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _size(rng, lo, hi, step):
    """A size of the range: mostly a multiple of the step, sometimes any."""
    v = _log_int(rng, lo, hi)
    if rng.random() < 0.75:
        v = max(lo, v // step * step)
    return v + step if v == 3072 else v


def draw(rng):
    op = rng.choice(["norm", "norm", "lora", "lora", "lora_shard", "scores", "scores"])
    if op == "norm":
        n = _size(rng, 512, 16384, 64)
        m = min(_log_int(rng, 1, 8192), NORM_BYTES_MAX // (n * 16))
        c = _norm("", m, n, rng.choice(["f32", "f32", "bf16"]), rng.choice(["bf16", "bf16", "f32"]),
                  rng.choice(["none", "channel", "token", "full"]), rng.random() < 0.6, rng.choice(["bf16", "bf16", "f32"]))
    elif op == "scores":
        vocab = _size(rng, 32000, 160000, 128)
        m = max(1, min(_log_int(rng, 1, 2000), SCORES_MAX // vocab))
        c = _scores("", m, vocab, rng.choice([0, 1, 5, 8, 20, 32]), rng.choice(["f32", "f32", "bf16"]), rng.random() < 0.3)
    else:
        rank = rng.choice([8, 16, 16, 32, 64])
        k = _size(rng, 512, K_PROJ, 64) if op == "lora" else _size(rng, 256, K_PROJ // 2, 64)
        n = _size(rng, 1024, HIDDEN, 64)
        batch = rng.choice(["decode", "prompts"])
        m = _log_int(rng, 1, 512) if batch == "decode" else _log_int(rng, 64, 4000)
        m = max(1, min(m, LORA_WORK_MAX // (rank * (k + n))))
        adapters = _log_int(rng, 1, 64)
        used = max(1, min(adapters, m, _log_int(rng, 1, 64 if batch == "decode" else 8)))
        c = _lora("", m, k, n, rank, adapters, used, batch, rng.choice(["bf16", "bf16", "f32"]), rng.choice(["f32", "f32", "bf16"]), op)
    c.pop("name")
    return c


# ------------------------------------------------------------------------------------------ inputs
def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _ids(case, g, dev):
    """Adapter of every token; exactly ``used`` of the table's adapters occur, and some tokens have none."""
    m, used = case["m"], case["used"]
    which = torch.randperm(case["adapters"], generator=g, device=dev)[:used].to(torch.int32)
    if case["batch"] == "prompts":      # one request after the other, of uneven lengths
        cuts = torch.sort(torch.randperm(m - 1, generator=g, device=dev)[:used - 1] + 1).values if used > 1 else torch.empty(0, dtype=torch.int64, device=dev)
        return which[torch.bucketize(torch.arange(m, device=dev), cuts, right=True)]
    slot = torch.randint(0, used, (m,), generator=g, device=dev)
    ids = torch.where(torch.rand((m,), generator=g, device=dev) < 0.1, torch.full_like(slot, -1).to(torch.int32), which[slot])
    place = torch.randperm(m, generator=g, device=dev)[:used]
    ids[place] = which
    return ids


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(shape, dtype, scale=1.0):
        return torch.empty(shape, dtype=torch.float32, device=dev).normal_(0.0, scale, generator=g).to(_type(dtype))

    op, m = case["op"], case["m"]
    s = {"op": op}
    if op == "norm":
        n = case["n"]
        s["y"] = normal((m, n), case["y"])
        s["residual"] = normal((m, n), case["res"], 3.0)
        s["post"] = normal((n,), "bf16", 0.1) + 1.0 if case["post"] else None
        s["next"] = normal((n,), "bf16", 0.1) + 1.0
        shape = {"none": None, "channel": (n,), "token": (m, 1), "full": (m, n)}[case["gate"]]
        s["gate"] = None if shape is None else normal(shape, "bf16")
        s["act"] = "none" if case["gate"] == "channel" else "sigmoid"
        s["residual_scale"], s["block_scale"] = 0.9, 1.25
        s["out"] = _type(case["out"])
    elif op == "scores":
        vocab = case["vocab"]
        x = torch.empty((m, vocab), dtype=torch.float32, device=dev).normal_(0.0, 2.5, generator=g)
        if case["masked"]:              # what a grammar forbids
            x.masked_fill_(torch.rand((vocab,), generator=g, device=dev) < 0.4, -math.inf)
        s["logits"] = x.to(_type(case["dtype"]))
        # the tokens that were sampled: one of the row's better entries, now and then any
        some = torch.randint(0, vocab, (m, 64), generator=g, device=dev)
        best = some.gather(1, x.gather(1, some).argmax(1, keepdim=True)).squeeze(1)
        s["tokens"] = torch.where(torch.rand((m,), generator=g, device=dev) < 0.1, some[:, 0], best).to(torch.int32)
        s["top"] = case["top"]
    else:
        k, n, r = case["k"], case["n"], case["rank"]
        s["x"] = normal((m, k), case["act"])
        s["y"] = normal((m, n), case["out"])
        s["a"] = normal((case["adapters"], r, k), "bf16", k ** -0.5)
        s["b"] = normal((case["adapters"], n, r), "bf16", 0.1)
        s["scale"] = 0.5 + torch.rand((case["adapters"],), generator=g, device=dev)
        s["ids"] = _ids(case, g, dev)
    return s


# ------------------------------------------------------------------------------------------ one pass
def _plain_norm(s):
    u = s["y"].float()
    if s["post"] is not None:
        u = u * torch.rsqrt((u * u).mean(1, keepdim=True) + EPS) * s["post"].float()
    u = u * s["block_scale"]
    if s["gate"] is not None:
        gate = s["gate"].float()
        u = u * (torch.sigmoid(gate) if s["act"] == "sigmoid" else gate)
    h = s["residual"].float() * s["residual_scale"] + u
    z = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * s["next"].float()
    return [h.to(s["residual"].dtype), z.to(s["out"])]


def _plain_shrink(s):
    """[m, adapters, rank]: the products with every adapter, zero but for a token's own."""
    adapters, r, k = s["a"].shape
    t = (s["x"].float() @ s["a"].float().reshape(adapters * r, k).t()).reshape(-1, adapters, r)
    mine = s["ids"].unsqueeze(1) == torch.arange(adapters, device=t.device, dtype=torch.int32)
    return torch.where(mine.unsqueeze(2), t, torch.zeros((), device=t.device))


def _plain_expand(s, t):
    adapters, n, r = s["b"].shape
    b = s["b"].float().permute(0, 2, 1).reshape(adapters * r, n)
    d = (t * s["scale"].reshape(1, adapters, 1)).reshape(-1, adapters * r) @ b
    return (s["y"].float() + d).to(s["y"].dtype)


def _plain_scores(s):
    x = s["logits"].float()
    tok = s["tokens"].long().unsqueeze(1)
    top = x.max(1, keepdim=True).values
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    mine = x.gather(1, tok)
    seen = torch.where(e > 0, x - top, torch.zeros((), device=x.device))
    entropy = torch.log(total) - (e * seen).sum(1, keepdim=True) / total
    before = (x > mine) | ((x == mine) & (torch.arange(x.shape[1], device=x.device) < tok))
    ids, vals = [], []
    left = x.clone() if s["top"] else x
    for _ in range(s["top"]):
        best = left.max(1, keepdim=True)
        vals.append(best.values - lse)
        ids.append(best.indices)
        left.scatter_(1, best.indices, -math.inf)
    out = [(mine - lse).squeeze(1), entropy.squeeze(1), before.sum(1).to(torch.int32)]
    return out + ([torch.cat(ids, 1).to(torch.int32), torch.cat(vals, 1)] if ids else [])


def run(state):
    s, op = state, state["op"]
    if not own:
        if op == "norm":
            return _plain_norm(s)
        if op == "scores":
            return _plain_scores(s)
        t = _plain_shrink(s)
        return [_plain_expand(s, t)] if op == "lora" else [t.sum(1), _plain_expand(s, t)]
    from weightstream_b200 import ops
    if op == "norm":
        hidden, normed = ops.block_norm(s["y"], s["residual"], post_weight=s["post"], next_weight=s["next"], gate=s["gate"],
                                        gate_act=s["act"], eps=EPS, residual_scale=s["residual_scale"], block_scale=s["block_scale"],
                                        normed_dtype=s["out"])
        return [hidden, normed]
    if op == "scores":
        r = ops.token_logprobs(s["logits"], s["tokens"], top=s["top"])
        out = [r.logprobs, r.entropy, r.rank]
        return out + ([r.top_ids, r.top_logprobs] if s["top"] else [])
    if op == "lora":
        return [ops.lora_add(s["y"], s["x"], s["a"], s["b"], s["ids"], s["scale"])]
    t = ops.lora_shrink(s["x"], s["a"], s["ids"])
    return [t, ops.lora_expand(s["y"], t, s["b"], s["ids"], s["scale"])]


# ------------------------------------------------------------------------------------------ yardsticks
def _bytes(name):
    return 4 if name == "f32" else 2


def work(case):
    op, m = case["op"], case["m"]
    if op == "norm":
        n = case["n"]
        gates = {"none": 0, "channel": n, "token": m, "full": m * n}[case["gate"]]
        row = _bytes(case["y"]) + 2 * _bytes(case["res"]) + _bytes(case["out"])
        return {"bytes": m * n * row + 2 * gates + 2 * n * (2 if case["post"] else 1), "flops": 12.0 * m * n}
    if op == "scores":
        return {"bytes": m * case["vocab"] * _bytes(case["dtype"]) + m * (16 + 8 * case["top"]), "flops": 6.0 * m * case["vocab"]}
    k, n, r = case["k"], case["n"], case["rank"]
    both = 2.0 * _bytes(case["out"]) * m * n + _bytes(case["act"]) * m * k + 2.0 * case["used"] * r * (k + n) + 4.0 * m
    if op == "lora_shard":
        both += 8.0 * m * r             # the shrunk rows go out and come back
    return {"bytes": both, "flops": 2.0 * m * r * (k + n)}


def exact(case, seed):
    """The operators' definitions in 64 bits, row by row or adapter by adapter."""
    s = prepare(case, seed)
    op = case["op"]
    if op == "norm":
        n = case["n"]
        hs, zs = [], []
        for i in range(0, case["m"], 512):
            y = s["y"][i:i + 512].double()
            if case["post"]:
                y = y / torch.sqrt(torch.linalg.vector_norm(y, dim=1, keepdim=True) ** 2 / n + EPS) * s["post"].double()
            if case["gate"] != "none":
                gate = (s["gate"] if case["gate"] == "channel" else s["gate"][i:i + 512]).double()
                y = y * gate if s["act"] == "none" else y / (1.0 + torch.exp(-gate))
            h = s["residual_scale"] * s["residual"][i:i + 512].double() + s["block_scale"] * y
            hs.append(h)
            zs.append(h / torch.sqrt(torch.linalg.vector_norm(h, dim=1, keepdim=True) ** 2 / n + EPS) * s["next"].double())
        return [torch.cat(hs), torch.cat(zs)]
    if op == "scores":
        parts = []
        for i in range(0, case["m"], 64):
            x = s["logits"][i:i + 64].double()
            tok = s["tokens"][i:i + 64].long()
            lp = torch.log_softmax(x, 1)
            p = torch.exp(lp)
            order = torch.sort(x, dim=1, descending=True, stable=True).indices
            rank = (order == tok.unsqueeze(1)).int().argmax(1).to(torch.int32)
            row = [lp.gather(1, tok.unsqueeze(1)).squeeze(1), -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1), rank]
            if case["top"]:
                ids = order[:, :case["top"]]
                row += [ids.to(torch.int32), lp.gather(1, ids)]
            parts.append(row)
        return [torch.cat(c) for c in zip(*parts)]
    t = torch.zeros((case["m"], case["rank"]), dtype=torch.float64, device=s["x"].device)
    out = s["y"].double()
    for i in torch.unique(s["ids"]).tolist():
        if i < 0:
            continue
        rows = torch.nonzero(s["ids"] == i).squeeze(1)
        t[rows] = s["x"][rows].double() @ s["a"][i].double().t()
        out[rows] += s["scale"][i].double() * (t[rows] @ s["b"][i].double().t())
    return [out] if op == "lora" else [t, out]
