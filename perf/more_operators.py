"""Workloads of the operators of a decode step around the reduction points, for timing and for comparing with plain forms.

Four operators: norms of queries and keys for each head with the position rotation (``ops.head_norm_rope``), the choice of
experts from the gate's logits (``ops.moe_route``), a whole mixture-of-experts layer of a few tokens over MXFP4 experts
(``ops.moe_layer``), and bias, penalties and grammar masks on the vocabulary head's logits (``ops.adjust_logits``).

``own`` chooses between the framework's operators and the same formulas in elementary torch operations in 32 bits.
"""
import math

import numpy as np
import torch

own = False

HIDDEN, EXPERT = 7168, 2048             # model width, width of a routed expert
HIDDEN_NATIVE, EXPERT_NATIVE = 5120, 2304   # the reference model's own widths
VOCAB, EXPERTS = 129280, 384
EPS = 1e-6
HEADS_MAX = 8192 * 72 * 128             # values of the largest listed case; bounds the drawn ones
LOGITS_MAX = 512 * VOCAB
EXPERTS_MAX = 42 * HIDDEN * EXPERT      # experts x width x width


def _heads(name, m, hq, hk, d, rot, start=0, inter=False, act="bf16", weight=True, far=4096):
    return {"name": name, "op": "heads", "m": m, "hq": hq, "hk": hk, "d": d, "rot": rot, "start": start, "inter": inter,
            "act": act, "weight": weight, "far": far}


def _route(name, m, experts, top_k, score="softmax", bias=False, act="f32"):
    return {"name": name, "op": "route", "m": m, "experts": experts, "top_k": top_k, "score": score, "bias": bias, "act": act}


def _layer(name, m, hidden, expert, local, used, routes, top_k=6, act="bf16", out="f32", quant=False, limit=0.0):
    return {"name": name, "op": "layer", "m": m, "hidden": hidden, "expert": expert, "local": local, "used": used, "routes": routes,
            "top_k": top_k, "act": act, "out": out, "quant": quant, "limit": limit}


def _adjust(name, m, vocab, history, penalties=True, biases=0, masks=0, dtype="f32"):
    return {"name": name, "op": "adjust", "m": m, "vocab": vocab, "history": history, "penalties": penalties, "biases": biases,
            "masks": masks, "dtype": dtype}


def listed():
    return [
        # One decoded token between the attention's input projections and the attention: grouped heads, all of a head rotated.
        _heads("heads_row", 1, 64, 8, 128, 128),
        # A ragged serving batch far into a long context; latent attention: one wide key head, its last 64 values rotated.
        _heads("heads_latent", 61, 64, 1, 512, 64, start=448, inter=True, far=1 << 20),
        # A prompt.
        _heads("heads_prompt", 8192, 64, 8, 128, 128, far=8192),
        # A serving batch's routes, weights by softmax over the chosen.
        _route("route_batch", 64, EXPERTS, 6),
        # A prompt's routes, chosen by score plus a bias that balances the experts.
        _route("route_prompt", 4096, EXPERTS, 8, score="sqrtsoftplus", bias=True),
        # One decoded token through its six experts, all on this rank.
        _layer("layer_row", 1, HIDDEN, EXPERT, 48, 6, 6),
        # A serving batch on one rank of eight: 48 of the 384 experts, most of the routes are other ranks'.
        _layer("layer_shard", 64, HIDDEN, EXPERT, 48, 30, 48),
        # The same experts with all routes on this rank.
        _layer("layer_batch", 16, HIDDEN, EXPERT, 48, 42, 96),
        # The reference's own widths and its rounding of activations, fp32 activations in, a clamped SwiGLU.
        _layer("layer_native", 5, HIDDEN_NATIVE, EXPERT_NATIVE, 32, 20, 28, act="f32", out="bf16", quant=True, limit=10.0),
        # One sampled token: penalties over a long answer, a few biased tokens.
        _adjust("adjust_row", 1, VOCAB, 6000, biases=20),
        # A serving batch, some of its requests under a grammar.
        _adjust("adjust_batch", 64, VOCAB, 4000, biases=8, masks=6),
        # The largest batch, bf16 logits, penalties and masks.
        _adjust("adjust_large", 512, VOCAB, 2000, masks=32, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def _size(rng, lo, hi, step, odd):
    """A size of the range: mostly a multiple of the step, else of `odd`."""
    v, step = _log_int(rng, lo, hi), step if rng.random() < 0.75 else odd
    return max(lo, v // step * step)


def draw(rng):
    op = rng.choice(["heads", "heads", "route", "layer", "layer", "layer", "adjust", "adjust"])
    if op == "heads":
        d = rng.choice([64, 80, 96, 128, 128, 192, 256, 512, 576])
        rot = rng.choice([d, d, d // 2, 64 if d >= 64 else d])
        start = rng.choice([0, d - rot])
        hq = _log_int(rng, 1, 128)
        hk = rng.choice([1, hq, max(1, hq // 8), max(1, hq // 4)])
        m = max(1, min(_log_int(rng, 1, 8192), HEADS_MAX // (2 * d * (hq + hk))))
        c = _heads("", m, hq, hk, d, rot, start, rng.random() < 0.5, rng.choice(["bf16", "bf16", "f32"]), rng.random() < 0.8,
                   _log_int(rng, 512, 1 << 20))
    elif op == "route":
        experts = _size(rng, 8, 512, 8, 1)
        c = _route("", _log_int(rng, 1, 4096), experts, rng.randint(1, min(8, experts)), rng.choice(["softmax", "sigmoid", "sqrtsoftplus"]),
                   rng.random() < 0.5, rng.choice(["f32", "f32", "bf16"]))
    elif op == "layer":
        hidden, expert = _size(rng, 512, HIDDEN, 256, 32), _size(rng, 128, EXPERT_NATIVE, 128, 32)
        m, local, top_k = _log_int(rng, 1, 64), _log_int(rng, 4, 64), rng.randint(1, 8)
        local = min(local, 48 * HIDDEN * EXPERT // (hidden * expert))
        used = max(1, min(local, m * top_k, _log_int(rng, 1, 48), EXPERTS_MAX // (hidden * expert)))
        routes = rng.randint(used, max(used, m * min(top_k, used)))
        quant = rng.random() < 0.3
        c = _layer("", m, hidden, expert, local, used, routes, top_k, rng.choice(["bf16", "bf16", "f32"]),
                   "bf16" if quant else rng.choice(["f32", "f32", "bf16"]), quant, rng.choice([0.0, 0.0, 10.0]))
    else:
        vocab = _size(rng, 32000, 160000, 128, 1)
        m = max(1, min(_log_int(rng, 1, 512), LOGITS_MAX // (2 * vocab)))
        history = _log_int(rng, 16, 30000)
        c = _adjust("", m, vocab, max(1, min(history, (1 << 21) // m)), rng.random() < 0.85, rng.choice([0, 0, 5, 64, 300]),
                    rng.choice([0, 0, 1, 8]), rng.choice(["f32", "f32", "bf16"]))
    c.pop("name")
    return c


# ------------------------------------------------------------------------------------------ inputs
def _type(name):
    return torch.float32 if name == "f32" else torch.bfloat16


def _routes(case, rng):
    """Ids [m, top_k]: exactly ``used`` of the rank's experts occur in exactly ``routes`` places; the other places are other
    ranks' experts or empty."""
    m, k, local, used = case["m"], case["top_k"], case["local"], case["used"]
    experts = rng.permutation(local)[:used]
    mine = [[] for _ in range(m)]
    for i, e in enumerate(experts):             # every one of them once, over the tokens in turn
        mine[i % m].append(int(e))
    left = case["routes"] - used
    popular = experts[:max(1, used // 3)]
    while left > 0:
        room = [t for t in range(m) if len(mine[t]) < min(k, used)]
        if not room:
            break
        for t in rng.permutation(room)[:left]:
            wanted = popular if rng.random() < 0.5 and len(mine[t]) < len(popular) else experts
            fresh = [int(e) for e in wanted if int(e) not in mine[t]] or [int(e) for e in experts if int(e) not in mine[t]]
            mine[t].append(fresh[rng.integers(len(fresh))])
            left -= 1
    start = 2 * local if case["m"] % 2 else 0
    ids = np.full((m, k), -1, dtype=np.int32)
    for t in range(m):
        places = rng.permutation(k)
        for e, j in zip(mine[t], places):
            ids[t, j] = start + e
        for j in places[len(mine[t]):]:
            ids[t, j] = start + local + int(rng.integers(local)) if rng.random() < 0.9 else -1
    return ids, start


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)

    def normal(shape, dtype, scale=1.0):
        return torch.empty(shape, dtype=torch.float32, device=dev).normal_(0.0, scale, generator=g).to(_type(dtype))

    def whole(lo, hi, shape, dtype):
        return torch.randint(lo, hi, shape, generator=g, device=dev, dtype=dtype)

    op, m = case["op"], case["m"]
    s = {"op": op}
    if op == "heads":
        hq, hk, d = case["hq"], case["hk"], case["d"]
        # queries and keys as the projection leaves them: side by side in a token's row
        both = normal((m, hq + hk, d), case["act"])
        s["q"], s["k"] = both[:, :hq], both[:, hq:]
        s["wq"] = normal((d,), "bf16", 0.1) + 1.0 if case["weight"] else None
        s["wk"] = normal((d,), "bf16", 0.1) + 1.0 if case["weight"] else None
        f = case["rot"] // 2
        s["inv_freq"] = (1e4 ** (-torch.arange(f, device=dev, dtype=torch.float64) / f)).float()
        s["positions"] = whole(0, case["far"], (m,), torch.int64)
        s["start"], s["inter"] = case["start"], case["inter"]
    elif op == "route":
        s["logits"] = normal((m, case["experts"]), case["act"], 1.5)
        s["bias"] = normal((case["experts"],), "f32", 0.1) if case["bias"] else None
        s["top_k"], s["score"] = case["top_k"], case["score"]
    elif op == "layer":
        h, f, n = case["hidden"], case["expert"], case["local"]
        ids, s["start"] = _routes(case, np.random.default_rng(seed))
        s["ids"] = torch.from_numpy(ids).to(dev)
        w = torch.rand((m, case["top_k"]), generator=g, device=dev) + 0.1
        s["w"] = w / w.sum(1, keepdim=True) * 1.5
        s["x"] = normal((m, h), case["act"])
        # codes of every value, and exponents that keep a product near its activations
        for name, rows, k in (("1", f, h), ("3", f, h), ("2", h, f)):
            s["w" + name] = whole(0, 256, (n, rows, k // 2), torch.uint8)
            mid = 126 - int(round(math.log2(2.93 * math.sqrt(k))))
            s["s" + name] = whole(mid, mid + 3, (n, rows, k // 32), torch.uint8)
        s["out"], s["quant"], s["limit"] = _type(case["out"]), case["quant"], case["limit"] or None
    else:
        vocab, mean = case["vocab"], case["history"]
        s["logits"] = normal((m, vocab), case["dtype"], 3.0)
        length = np.random.default_rng(seed).integers(mean // 2, mean + mean // 2 + 1, size=m)
        ends = np.concatenate([[0], np.cumsum(length)])
        s["offsets"] = torch.from_numpy(ends.astype(np.int32)).to(dev)
        # words of an answer: few tokens make up most of it
        u = torch.rand((int(ends[-1]),), generator=g, device=dev, dtype=torch.float64)
        s["tokens"] = (vocab * u ** 4).to(torch.int32).clamp_(max=vocab - 1) if case["penalties"] else None
        s["prompt"] = (torch.from_numpy(length).to(dev) * torch.rand((m,), generator=g, device=dev)).to(torch.int32)
        s["rep"], s["freq"], s["pres"] = (lo + span * torch.rand((m,), generator=g, device=dev) for lo, span in ((1.0, 0.3), (0.0, 0.5), (0.0, 0.5)))
        s["bias_ids"] = None
        if case["biases"]:
            n = case["biases"]
            first = whole(0, vocab, (m, 1), torch.int64)
            s["bias_ids"] = ((first + 101 * torch.arange(n, device=dev)) % vocab).to(torch.int32).reshape(-1)
            s["bias"] = normal((m * n,), "f32", 4.0)
            s["bias_offsets"] = torch.arange(0, m * n + 1, n, device=dev, dtype=torch.int32)
        s["mask"] = None
        if case["masks"]:       # one bit a token, as a grammar's compiler packs them; some requests have none
            words = (vocab + 31) // 32
            s["mask"] = whole(-2 ** 31, 2 ** 31, (case["masks"], words), torch.int32) & whole(-2 ** 31, 2 ** 31, (case["masks"], words), torch.int32)
            s["mask_rows"] = whole(-1, case["masks"], (m,), torch.int32)
    return s


# ------------------------------------------------------------------------------------------ one pass
def _turn(u, cos, sin, start, inter):
    f = cos.shape[-1]
    part = u[..., start:start + 2 * f]
    a, b = (part[..., 0::2], part[..., 1::2]) if inter else (part[..., :f], part[..., f:])
    x, y = a * cos - b * sin, a * sin + b * cos
    turned = torch.stack([x, y], -1).flatten(-2) if inter else torch.cat([x, y], -1)
    return torch.cat([u[..., :start], turned, u[..., start + 2 * f:]], -1)


def _plain_heads(s):
    angle = s["positions"].double().unsqueeze(1) * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)

    def one(t, w):
        u = t.float()
        u = u * torch.rsqrt((u * u).mean(-1, keepdim=True) + EPS)
        return _turn(u if w is None else u * w.float(), cos, sin, s["start"], s["inter"]).to(t.dtype)
    return [one(s["q"], s["wq"]), one(s["k"], s["wk"])]


def _plain_route(s):
    x = s["logits"].double()                    # the choice is one of neighbours
    if s["score"] == "softmax":
        score = torch.exp(x - x.max(1, keepdim=True).values)
        score = score / score.sum(1, keepdim=True)
    elif s["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-x))
    else:
        score = torch.sqrt(torch.log1p(torch.exp(x)))
    key = score if s["bias"] is None else score + s["bias"].double()
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :s["top_k"]]
    w = score.gather(1, ids)
    return [ids.to(torch.int32), (w / w.sum(1, keepdim=True) * 2.5).float()]


def _plain_weight(w, s):
    codes = torch.stack([w & 15, w >> 4], -1).flatten(-2)
    size = (codes & 7).float()
    value = torch.where(size < 4, size * 0.5, torch.where(size < 6, size - 2.0, 2.0 * size - 8.0))
    value = torch.where(codes > 7, -value, value)
    e, rows, k = value.shape
    return (value.reshape(e, rows, k // 32, 32) * torch.exp2(s.float() - 127.0).unsqueeze(-1)).reshape(e, rows, k)


def _plain_round(v):
    """To E4M3 with a power of two for 32 values."""
    b = v.reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    part, exponent = torch.frexp(b.abs().amax(-1, keepdim=True).clamp(min=1e-4) / 448.0)
    scale = torch.exp2(torch.where(part == 0.5, exponent - 1, exponent).to(v.dtype))
    return ((b / scale).clamp(-448.0, 448.0).to(torch.float8_e4m3fn).to(v.dtype) * scale).reshape(v.shape)


def _plain_layer(s):
    x = _plain_round(s["x"].float()) if s["quant"] else s["x"].float()
    n = s["w1"].shape[0]
    gate = torch.matmul(x, _plain_weight(s["w1"], s["s1"]).transpose(1, 2))     # [experts, m, width]
    up = torch.matmul(x, _plain_weight(s["w3"], s["s3"]).transpose(1, 2))
    if s["limit"] is not None:
        gate, up = gate.clamp(max=s["limit"]), up.clamp(-s["limit"], s["limit"])
    here = s["ids"].unsqueeze(0) - s["start"] == torch.arange(n, device=x.device, dtype=torch.int32).reshape(n, 1, 1)
    weight = torch.where(here, s["w"], torch.zeros((), device=x.device)).sum(2)
    h = weight.unsqueeze(2) * (gate / (1.0 + torch.exp(-gate)) * up)
    h = _plain_round(h) if s["quant"] else h
    return [torch.matmul(h, _plain_weight(s["w2"], s["s2"]).transpose(1, 2)).sum(0).to(s["out"])]


def _plain_adjust(s):
    x = s["logits"].float()
    m, vocab = x.shape
    if s["bias_ids"] is not None:
        row = torch.bucketize(torch.arange(s["bias_ids"].shape[0], device=x.device), s["bias_offsets"][1:], right=True)
        x = x.index_put((row, s["bias_ids"].long()), s["bias"], accumulate=True)
    if s["tokens"] is not None:
        at = torch.arange(s["tokens"].shape[0], device=x.device)
        row = torch.bucketize(at, s["offsets"][1:], right=True)
        answer = at - s["offsets"][row] >= s["prompt"][row]
        place = row * vocab + s["tokens"]
        seen = torch.zeros(m * vocab, dtype=torch.int32, device=x.device).index_fill_(0, place, 1).reshape(m, vocab)
        count = torch.zeros(m * vocab, dtype=torch.int32, device=x.device).scatter_add_(0, place, answer.to(torch.int32)).reshape(m, vocab)
        rep, freq, pres = s["rep"].unsqueeze(1), s["freq"].unsqueeze(1), s["pres"].unsqueeze(1)
        x = torch.where(seen > 0, torch.where(x > 0, x / rep, x * rep), x)
        x = x - freq * count - pres * (count > 0)
    if s["mask"] is not None:
        bits = (s["mask"].unsqueeze(-1) >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        open_ = bits.reshape(bits.shape[0], -1)[:, :vocab][s["mask_rows"].clamp(min=0).long()] > 0
        x = torch.where(open_ | (s["mask_rows"] < 0).unsqueeze(1), x, torch.full((), -math.inf, device=x.device))
    return [x.to(s["logits"].dtype)]


def run(state):
    s, op = state, state["op"]
    if not own:
        return {"heads": _plain_heads, "route": _plain_route, "layer": _plain_layer, "adjust": _plain_adjust}[op](s)
    from weightstream_b200 import ops
    if op == "heads":
        return list(ops.head_norm_rope(s["q"], s["k"], q_weight=s["wq"], k_weight=s["wk"], eps=EPS, positions=s["positions"],
                                       inv_freq=s["inv_freq"], rotary_start=s["start"], interleaved=s["inter"]))
    if op == "route":
        return list(ops.moe_route(s["logits"], s["top_k"], score=s["score"], bias=s["bias"], scale=2.5))
    if op == "layer":
        return [ops.moe_layer(s["x"], s["ids"], s["w"], s["w1"], s["s1"], s["w3"], s["s3"], s["w2"], s["s2"], s["start"],
                              limit=s["limit"], act_quant=s["quant"], out_dtype=s["out"])]
    more = {}
    if s["tokens"] is not None:
        more.update(tokens=s["tokens"], offsets=s["offsets"], prompt_lens=s["prompt"], repetition=s["rep"], frequency=s["freq"], presence=s["pres"])
    if s["bias_ids"] is not None:
        more.update(bias_ids=s["bias_ids"], bias=s["bias"], bias_offsets=s["bias_offsets"])
    if s["mask"] is not None:
        more.update(mask=s["mask"], mask_rows=s["mask_rows"])
    return [ops.adjust_logits(s["logits"], **more)]


# ------------------------------------------------------------------------------------------ yardsticks
def _bytes(name):
    return 4 if name == "f32" else 2


def work(case):
    op, m = case["op"], case["m"]
    if op == "heads":
        values = m * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * values * _bytes(case["act"]) + 8 * m + 2 * case["rot"] + (4 * case["d"] if case["weight"] else 0), "flops": 8.0 * values}
    if op == "route":
        return {"bytes": m * case["experts"] * _bytes(case["act"]) + 8 * m * case["top_k"], "flops": 4.0 * m * case["experts"]}
    if op == "layer":
        one = 3 * case["hidden"] * case["expert"]
        return {"bytes": case["used"] * one * (1 / 2 + 1 / 32) + m * case["hidden"] * (_bytes(case["act"]) + _bytes(case["out"])) + 8 * m * case["top_k"],
                "flops": 2.0 * case["routes"] * one}
    size = 2 * m * case["vocab"] * _bytes(case["dtype"]) + 8 * m * case["biases"] + case["masks"] * case["vocab"] / 8
    return {"bytes": size + (4 * m * case["history"] if case["penalties"] else 0), "flops": 4.0 * m * case["vocab"]}


_E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0]


def _exact_heads(s):
    out = []
    for t, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        parts = []
        for i in range(0, t.shape[0], 512):
            v = t[i:i + 512].double()
            v = v / torch.sqrt(torch.linalg.vector_norm(v, dim=2, keepdim=True) ** 2 / v.shape[2] + EPS)
            if w is not None:
                v = v * w.double()
            turn = torch.polar(torch.ones((), dtype=torch.float64, device=v.device),
                               torch.outer(s["positions"][i:i + 512].double(), s["inv_freq"].double())).unsqueeze(1)
            f, a = turn.shape[2], s["start"]
            first, second = (slice(a, a + 2 * f, 2), slice(a + 1, a + 2 * f, 2)) if s["inter"] else (slice(a, a + f), slice(a + f, a + 2 * f))
            z = torch.complex(v[..., first], v[..., second]) * turn
            v[..., first], v[..., second] = z.real, z.imag
            parts.append(v)
        out.append(torch.cat(parts))
    return out


def _exact_route(s):
    x = s["logits"].double()
    score = {"softmax": lambda: torch.softmax(x, 1), "sigmoid": lambda: torch.sigmoid(x),
             "sqrtsoftplus": lambda: torch.nn.functional.softplus(x, threshold=1e9) ** 0.5}[s["score"]]()
    key = score.clone() if s["bias"] is None else score + s["bias"].double()
    ids = []
    for _ in range(s["top_k"]):
        best = (key == key.max(1, keepdim=True).values).int().argmax(1, keepdim=True)       # the lowest index of equal ones
        ids.append(best)
        key.scatter_(1, best, -math.inf)
    ids = torch.cat(ids, 1)
    w = score.gather(1, ids)
    return [ids.to(torch.int32), 2.5 * w / w.sum(1, keepdim=True)]


def _exact_weight(w, s):
    table = torch.tensor(_E2M1, dtype=torch.float64, device=w.device)
    v = torch.empty((w.shape[0], 2 * w.shape[1]), dtype=torch.float64, device=w.device)
    v[:, 0::2], v[:, 1::2] = table[(w & 15).int()], table[(w >> 4).int()]
    return v * torch.pow(2.0, s.double() - 127.0).repeat_interleave(32, 1)


def _exact_round(v):
    b = v.reshape(v.shape[0], -1, 32)
    scale = torch.pow(2.0, torch.ceil(torch.log2(b.abs().amax(2, keepdim=True).clamp(min=1e-4) / 448.0)))
    q = torch.clamp(b / scale, -448.0, 448.0)
    step = torch.pow(2.0, torch.clamp(torch.floor(torch.log2(q.abs().clamp(min=1e-30))), min=-6.0) - 3.0)
    return (torch.round(q / step) * step * scale).reshape(v.shape)


def _exact_layer(s):
    x = s["x"].double()
    x = _exact_round(x) if s["quant"] else x
    out = torch.zeros_like(x)
    for e in range(s["w1"].shape[0]):
        at = torch.nonzero(s["ids"] == s["start"] + e)
        if not at.shape[0]:
            continue
        g = x[at[:, 0]] @ _exact_weight(s["w1"][e], s["s1"][e]).t()
        u = x[at[:, 0]] @ _exact_weight(s["w3"][e], s["s3"][e]).t()
        if s["limit"] is not None:
            g, u = torch.clamp(g, max=s["limit"]), torch.clamp(u, -s["limit"], s["limit"])
        h = torch.nn.functional.silu(g) * u * s["w"].double()[at[:, 0], at[:, 1]].unsqueeze(1)
        out.index_add_(0, at[:, 0], (_exact_round(h) if s["quant"] else h) @ _exact_weight(s["w2"][e], s["s2"][e]).t())
    return [out]


def _exact_adjust(s):
    out = []
    for t in range(s["logits"].shape[0]):
        z = s["logits"][t].double()
        vocab = z.shape[0]
        if s["bias_ids"] is not None:
            n = s["bias_ids"].shape[0] // s["logits"].shape[0]
            z[s["bias_ids"][t * n:t * n + n].long()] += s["bias"][t * n:t * n + n].double()
        if s["tokens"] is not None:
            one = s["tokens"][s["offsets"][t]:s["offsets"][t + 1]]
            count = torch.bincount(one[s["prompt"][t]:], minlength=vocab)
            seen = torch.bincount(one, minlength=vocab) > 0
            rep = s["rep"][t].double()
            z = torch.where(seen & (z > 0), z / rep, torch.where(seen, z * rep, z))
            z = z - s["freq"][t].double() * count - torch.where(count > 0, s["pres"][t].double(), 0.0)
        if s["mask"] is not None and int(s["mask_rows"][t]) >= 0:
            bytes_ = s["mask"][s["mask_rows"][t]].view(torch.uint8)
            bits = (bytes_.unsqueeze(1) & (2 ** torch.arange(8, device=z.device)).to(torch.uint8)) != 0
            z[~bits.reshape(-1)[:vocab]] = -math.inf
        out.append(z)
    return [torch.stack(out)]


def exact(case, seed):
    """The operators' definitions in 64 bits, token by token or expert by expert."""
    return {"heads": _exact_heads, "route": _exact_route, "layer": _exact_layer, "adjust": _exact_adjust}[case["op"]](prepare(case, seed))
