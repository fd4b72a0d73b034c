"""Operators between the tensor-parallel steps, on the tensors that the steps take and return.

A decode engine does more between two reduction points than the steps of :mod:`weightstream_b200.tp`: it normalises a
block's output, gates it, adds it to the residual stream and normalises that for the next block (:func:`block_norm`),
it adds the requests' low-rank adapters to a projection's result (:func:`lora_add`), and it scores given tokens on the
vocabulary head's logits (:func:`token_logprobs`).

Every function runs on the GPU that holds its tensors, on ``stream`` or the current stream, and does not synchronise.
Results are allocated on that stream.  A tensor that a call reads has to live until the stream has passed the call, as
with torch's own operators.  Wrong arguments raise ``TypeError`` or ``ValueError``, sizes beyond what a kernel counts
``WsError``, before anything is launched.  The operators are for serving: a result has no gradient, whatever its inputs ask.
"""
from __future__ import annotations

import contextlib
import ctypes as C
from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import BlockNormArgs, LoraArgs, TokenLogprobsArgs, WsError, WS_ACT_BF16, WS_ACT_F32, WS_GATE_LINEAR, WS_GATE_SIGMOID, \
    WS_LORA_MAX_RANK, WS_MAX_TOP, WS_OK

_TYPES = {torch.bfloat16: WS_ACT_BF16, torch.float32: WS_ACT_F32}
_GATES = {"none": WS_GATE_LINEAR, "sigmoid": WS_GATE_SIGMOID}


def _code(t: torch.Tensor, name: str) -> int:
    try:
        return _TYPES[t.dtype]
    except KeyError:
        raise TypeError(f"{name} must be bf16 or fp32, got {t.dtype}") from None


def _rows(t: torch.Tensor, name: str, m: int, n: int) -> int:
    """Row stride of a [m, n] tensor whose rows are stored one value after the other."""
    if t.dim() != 2 or t.shape[0] != m or t.shape[1] != n:
        raise ValueError(f"{name} must be [{m}, {n}], got {list(t.shape)}")
    if n > 1 and t.stride(1) != 1 and m:
        raise ValueError(f"{name} needs unit inner stride")
    if m > 1 and t.stride(0) < n:
        raise ValueError(f"{name}: rows of {n} values lie {t.stride(0)} apart")
    return t.stride(0) if m > 1 else n


def _vector(t: torch.Tensor, name: str, n: int, dtype=None) -> None:
    if t.dim() != 1 or t.shape[0] != n or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of {n} values, got {list(t.shape)}")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def _tensors(optional: bool = False, **given) -> None:
    for name, t in given.items():
        if not isinstance(t, torch.Tensor) and not (optional and t is None):
            raise TypeError(f"{name} must be a tensor, got {type(t).__name__}")


def _same_device(first: torch.Tensor, *others) -> None:
    for t in others:
        if t is not None and t.device != first.device:
            raise ValueError(f"tensors on {first.device} and {t.device}")


def _on(device: torch.device, stream):
    """Current device and stream of a call: what it allocates belongs to the stream that writes it."""
    if device.type != "cuda":
        raise ValueError(f"tensors must be on a CUDA device, got {device}")
    both = contextlib.ExitStack()
    both.enter_context(torch.cuda.device(device))
    if stream is not None:
        both.enter_context(torch.cuda.stream(stream))
    return both


def _handle(stream, t) -> Optional[int]:
    """A stream's handle, None for the current one.  Entering a stream of another device would make that device the
    current one, which then reads this one's memory.  (A stream that is only a handle cannot be told from its own.)"""
    if stream is None:
        return None
    device = getattr(stream, "device", None)
    if device is not None and isinstance(t, torch.Tensor) and device != t.device:
        raise ValueError(f"a stream of {device} for tensors on {t.device}")
    return stream.cuda_stream


def _call(name: str, args) -> None:
    L, err = _lib.load(), C.create_string_buffer(256)
    st = getattr(L, name)(C.byref(args), int(torch.cuda.current_stream().cuda_stream), err, len(err))
    if st != WS_OK:
        raise WsError(st, err.value.decode())


_native = None  # the front end for torch tensors, once it is loaded


def _load():
    global _native
    _native = _lib.torch_front()
    return _native


def _dim(*sizes: int) -> None:
    for v in sizes:
        if v >= 2 ** 31:
            raise ValueError(f"a dimension of {v} is beyond 31 bits")


# ----------------------------------------------------------------------------- norms around a block
def _block_norm_args(y, residual, post_weight, next_weight, gate, gate_act, eps, weight_offset, residual_scale, block_scale,
                     out, out_dtype, normed_dtype) -> Tuple[BlockNormArgs, torch.dtype, torch.dtype]:
    if y.dim() != 2 or y.shape[1] < 1:
        raise ValueError(f"y must be [m, n] with n >= 1, got {list(y.shape)}")
    m, n = y.shape
    _dim(m, n)
    a = BlockNormArgs()
    a.m, a.n = m, n
    a.y, a.ldy, a.y_dtype = y.data_ptr(), _rows(y, "y", m, n), _code(y, "y")
    if residual is not None:
        a.residual, a.ldr, a.residual_dtype = residual.data_ptr(), _rows(residual, "residual", m, n), _code(residual, "residual")
    if gate_act not in _GATES:
        raise ValueError(f"gate_act must be one of {sorted(_GATES)}, got {gate_act!r}")
    if gate is not None:
        if gate.dim() not in (1, 2):
            raise ValueError("gate must be [n], [m, 1] or [m, n]")
        g = gate if gate.dim() == 2 else gate.unsqueeze(0)
        if g.shape[0] not in (1, m) or g.shape[1] not in (1, n):
            raise ValueError(f"gate must be [{n}], [{m}, 1] or [{m}, {n}], got {list(gate.shape)}")
        if g.shape[1] > 1 and g.stride(1) not in (0, 1):
            raise ValueError("gate needs unit inner stride")
        a.gate, a.gate_dtype, a.gate_act = g.data_ptr(), _code(gate, "gate"), _GATES[gate_act]
        a.ldg = g.stride(0) if g.shape[0] > 1 else 0
        a.gate_inc = g.stride(1) if g.shape[1] > 1 else 0
    weights = [(w, name) for w, name in ((post_weight, "post_weight"), (next_weight, "next_weight")) if w is not None]
    for w, name in weights:
        _vector(w, name, n)
        a.weight_dtype = _code(w, name)
    if len(weights) == 2 and post_weight.dtype != next_weight.dtype:
        raise TypeError("post_weight and next_weight must have one type")
    a.post_weight = post_weight.data_ptr() if post_weight is not None else None
    a.next_weight = next_weight.data_ptr() if next_weight is not None else None
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    a.eps, a.weight_offset, a.residual_scale, a.block_scale = eps, weight_offset, residual_scale, block_scale
    hidden = out.dtype if out is not None else out_dtype or (residual.dtype if residual is not None else torch.bfloat16)
    if out is not None:
        a.hidden, a.ldh = out.data_ptr(), _rows(out, "out", m, n)
    for dtype in (hidden, normed_dtype):
        if dtype not in _TYPES:
            raise TypeError(f"results are bf16 or fp32, not {dtype}")
    a.hidden_dtype, a.normed_dtype = _TYPES[hidden], _TYPES[normed_dtype]
    _same_device(y, residual, gate, post_weight, next_weight, out)
    return a, hidden, normed_dtype


def block_norm(y: torch.Tensor, residual: Optional[torch.Tensor] = None, *, post_weight: Optional[torch.Tensor] = None,
               next_weight: Optional[torch.Tensor] = None, gate: Optional[torch.Tensor] = None, gate_act: str = "none",
               eps: float = 1e-6, weight_offset: float = 0.0, residual_scale: float = 1.0, block_scale: float = 1.0,
               out: Optional[torch.Tensor] = None, out_dtype: Optional[torch.dtype] = None,
               normed_dtype: torch.dtype = torch.bfloat16, stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Norms before and after a block, its gate, its residual scale and the residual stream, in one launch.

    ``y`` [m, n] is what the block returned (the fp32 sums of a reduction point, or bf16)::

        u      = y                                  with post_weight: y * rsqrt(mean(y^2) + eps) * (weight_offset + post_weight)
        hidden = residual_scale * residual + block_scale * act(gate) * u
        normed = hidden * rsqrt(mean(hidden^2) + eps) * (weight_offset + next_weight)

    ``gate`` is one value per channel ([n]), per token ([m, 1]) or per element ([m, n]); ``gate_act`` is ``"none"`` or
    ``"sigmoid"``.  ``weight_offset`` is 1 for models that keep their norm weights as a difference from one.  Everything
    between the loads and the results is held in 32 bits; ``normed`` is taken from ``hidden`` before it is rounded.

    Returns ``(hidden, normed)``; ``hidden`` is always written, ``normed`` is None without ``next_weight``.  ``hidden`` has the residual's type, or
    ``out_dtype``; ``out`` takes it and may be ``residual`` itself.
    """
    r = (_native or _load()).block_norm(y, residual, post_weight, next_weight, gate, _GATES.get(gate_act, -1), eps, weight_offset,
                                      residual_scale, block_scale, out, out_dtype, normed_dtype, _handle(stream, y))
    if r is not None:
        return r
    _tensors(y=y)
    _tensors(True, residual=residual, post_weight=post_weight, next_weight=next_weight, gate=gate, out=out)
    a, hidden_dtype, normed_dtype = _block_norm_args(y, residual, post_weight, next_weight, gate, gate_act, eps, weight_offset,
                                                     residual_scale, block_scale, out, out_dtype, normed_dtype)
    with _on(y.device, stream):
        hidden = out if out is not None else torch.empty((a.m, a.n), dtype=hidden_dtype, device=y.device)
        a.hidden, a.ldh = hidden.data_ptr(), a.ldh or a.n
        normed = None
        if next_weight is not None:
            normed = torch.empty((a.m, a.n), dtype=normed_dtype, device=y.device)
            a.normed, a.ldn = normed.data_ptr(), a.n
        _call("ws_block_norm", a)
    return hidden, normed


# ----------------------------------------------------------------------------- adapters of many requests
def _lora_args(ids, *, x=None, a=None, y=None, b=None, scale=None, shrunk=None, out=None) -> LoraArgs:
    """Arguments of the whole (x, a, y, b), of the shrinking half (x, a) or of the expanding one (shrunk, y, b)."""
    if ids.dtype != torch.int32:
        raise TypeError(f"ids must be int32, got {ids.dtype}")
    m = ids.shape[0] if ids.dim() == 1 else -1
    _vector(ids, "ids", m)
    r = LoraArgs()
    r.m, r.ids = m, ids.data_ptr()
    for t, name in ((a, "a"), (b, "b")):
        if t is None:
            continue
        if t.dtype != torch.bfloat16:
            raise TypeError(f"{name} must be bf16, got {t.dtype}")
        if t.dim() != 3 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous and 3-D, got {list(t.shape)}")
    if a is not None:
        r.adapters, r.rank, r.k = a.shape
        r.a, r.x, r.ldx, r.x_dtype = a.data_ptr(), x.data_ptr(), _rows(x, "x", m, a.shape[2]), _code(x, "x")
    if b is not None:
        if a is not None and (b.shape[0], b.shape[2]) != (a.shape[0], a.shape[1]):
            raise ValueError(f"a {list(a.shape)} and b {list(b.shape)} must be [adapters, rank, k] and [adapters, n, rank]")
        r.adapters, r.n, r.rank = b.shape
        r.b, r.y, r.ldy, r.y_dtype = b.data_ptr(), y.data_ptr(), _rows(y, "y", m, b.shape[1]), _code(y, "y")
        if out is not None:
            if out.dtype != y.dtype:
                raise TypeError(f"out must be {y.dtype} as y, got {out.dtype}")
            r.out, r.ldo = out.data_ptr(), _rows(out, "out", m, b.shape[1])
        if scale is not None:
            _vector(scale, "scale", r.adapters, torch.float32)
            r.scale = scale.data_ptr()
    _dim(m, *(a.shape if a is not None else ()), *(b.shape if b is not None else ()))
    if r.adapters < 1 or not 1 <= r.rank <= WS_LORA_MAX_RANK:
        raise ValueError(f"{r.adapters} adapters of rank {r.rank}: at least one, of rank 1..{WS_LORA_MAX_RANK}")
    if (a is not None and r.k < 1) or (b is not None and r.n < 1):
        raise ValueError("k and n must be at least 1")
    if shrunk is not None:
        if shrunk.dtype != torch.float32:
            raise TypeError(f"shrunk must be fp32, got {shrunk.dtype}")
        if list(shrunk.shape) != [m, r.rank] or not shrunk.is_contiguous():
            raise ValueError(f"shrunk must be contiguous [{m}, {r.rank}], got {list(shrunk.shape)}")
        r.shrunk = shrunk.data_ptr()
    _same_device(ids, x, a, y, b, scale, shrunk, out)
    return r


def _lora_call(name: str, args: LoraArgs, device) -> None:
    """On the current stream, whose memory the workspace is."""
    size = _lib.load().ws_lora_workspace(args.m, args.adapters, args.rank)
    work = torch.empty(size, dtype=torch.uint8, device=device)
    args.workspace, args.workspace_bytes = work.data_ptr(), size
    _call(name, args)


def lora_add(y: torch.Tensor, x: torch.Tensor, a: torch.Tensor, b: torch.Tensor, ids: torch.Tensor, scale: Optional[torch.Tensor] = None, *,
             out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """Low-rank adapters of many requests beside a shared projection: ``out[t] = y[t] + scale[i] * b[i] @ (a[i] @ x[t])``
    with ``i = ids[t]``.

    ``x`` [m, k] is what the projection read, ``y`` [m, n] what it returned (bf16 or fp32 each); ``a`` [adapters, rank, k]
    and ``b`` [adapters, n, rank] are bf16, ``scale`` [adapters] fp32, ``ids`` [m] int32 in any order.  A token whose id is
    outside [0, adapters), such as -1, has no adapter.  Ranks of 1 to 128; sums are fp32 and no activation is rounded on
    the way.  With more than 512 tokens a table has at most 16384 adapters; more raise ``WsError`` (the halves alike).
    Returns ``out``, of ``y``'s type, which may be ``y`` itself.
    """
    r = (_native or _load()).lora(0, y, x, a, b, ids, scale, None, out, _handle(stream, ids))
    if r is not None:
        return r
    _tensors(y=y, x=x, a=a, b=b, ids=ids)
    _tensors(True, scale=scale, out=out)
    args = _lora_args(ids, x=x, a=a, y=y, b=b, scale=scale, out=out)
    with _on(y.device, stream):
        out = out if out is not None else torch.empty((args.m, args.n), dtype=y.dtype, device=y.device)
        args.out, args.ldo = out.data_ptr(), args.ldo or args.n
        _lora_call("ws_lora_add", args, y.device)
    return out


def lora_shrink(x: torch.Tensor, a: torch.Tensor, ids: torch.Tensor, *, stream=None) -> torch.Tensor:
    """The first half of :func:`lora_add`, ``a[ids[t]] @ x[t]`` as fp32 [m, rank], for a projection whose K is sharded: each
    rank shrinks its slice of ``x`` with its slice of ``a``, ``Endpoint.allreduce_`` adds the ranks' rows up, and
    :func:`lora_expand` follows.  Rows of tokens without an adapter are zeros."""
    r = (_native or _load()).lora(1, None, x, a, None, ids, None, None, None, _handle(stream, ids))
    if r is not None:
        return r
    _tensors(x=x, a=a, ids=ids)
    args = _lora_args(ids, x=x, a=a)
    with _on(x.device, stream):
        shrunk = torch.empty((args.m, args.rank), dtype=torch.float32, device=x.device)
        args.shrunk = shrunk.data_ptr()
        _lora_call("ws_lora_shrink", args, x.device)
    return shrunk


def lora_expand(y: torch.Tensor, shrunk: torch.Tensor, b: torch.Tensor, ids: torch.Tensor, scale: Optional[torch.Tensor] = None, *,
                out: Optional[torch.Tensor] = None, stream=None) -> torch.Tensor:
    """The second half of :func:`lora_add`: ``out[t] = y[t] + scale[i] * b[i] @ shrunk[t]`` with ``i = ids[t]``."""
    r = (_native or _load()).lora(2, y, None, None, b, ids, scale, shrunk, out, _handle(stream, ids))
    if r is not None:
        return r
    _tensors(y=y, shrunk=shrunk, b=b, ids=ids)
    _tensors(True, scale=scale, out=out)
    args = _lora_args(ids, y=y, b=b, scale=scale, shrunk=shrunk, out=out)
    with _on(y.device, stream):
        out = out if out is not None else torch.empty((args.m, args.n), dtype=y.dtype, device=y.device)
        args.out, args.ldo = out.data_ptr(), args.ldo or args.n
        _lora_call("ws_lora_expand", args, y.device)
    return out


# ----------------------------------------------------------------------------- scores of given tokens
class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor                    # [m] fp32
    entropy: torch.Tensor                     # [m] fp32, in nats
    rank: torch.Tensor                        # [m] int32
    top_ids: Optional[torch.Tensor]           # [m, top] int32, None with top = 0
    top_logprobs: Optional[torch.Tensor]      # [m, top] fp32, None with top = 0


def _token_logprobs_args(logits, tokens, top) -> TokenLogprobsArgs:
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [m, vocab] with vocab >= 1, got {list(logits.shape)}")
    m, vocab = logits.shape
    _dim(m, vocab)
    a = TokenLogprobsArgs()
    a.m, a.vocab = m, vocab
    a.logits, a.ld, a.dtype = logits.data_ptr(), _rows(logits, "logits", m, vocab), _code(logits, "logits")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"tokens must be int32 or int64, got {tokens.dtype}")
    _vector(tokens, "tokens", m)
    a.tokens, a.token_bytes = tokens.data_ptr(), tokens.element_size()
    if not 0 <= top <= WS_MAX_TOP:
        raise ValueError(f"top must be in 0..{WS_MAX_TOP}, got {top}")
    a.top = top
    _same_device(logits, tokens)
    return a


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, *, top: int = 0, stream=None) -> TokenLogprobs:
    """Log probability of one given token a row, with the distribution's entropy, the token's rank and the ``top`` best
    alternatives, from one pass over the logits [m, vocab] (fp32 as ``lm_head_allgather_argmax`` returns them, or bf16).

    ``rank`` is the number of entries that come before the token, larger logits first and equal ones by index (0: the
    token is the argmax); ``top_ids`` holds the first ``top`` (at most 32) entries in that order.  Masked (-inf) and NaN
    logits are never alternatives; places that stay empty hold id -1 and log probability -inf.  A token outside
    [0, vocab), such as -1 for padding, is none: log probability 0, rank -1.  A row that is masked whole has log
    probability -inf and entropy 0; NaN or +inf in a row make its log probabilities and entropy NaN.
    """
    r = (_native or _load()).token_logprobs(logits, tokens, top, _handle(stream, logits))
    if r is not None:
        return tuple.__new__(TokenLogprobs, r)
    _tensors(logits=logits, tokens=tokens)
    a = _token_logprobs_args(logits, tokens, top)
    with _on(logits.device, stream):
        new = lambda *shape, dtype: torch.empty(shape, dtype=dtype, device=logits.device)
        r = TokenLogprobs(new(a.m, dtype=torch.float32), new(a.m, dtype=torch.float32), new(a.m, dtype=torch.int32),
                          new(a.m, top, dtype=torch.int32) if top else None, new(a.m, top, dtype=torch.float32) if top else None)
        a.logprob, a.entropy, a.rank = r.logprobs.data_ptr(), r.entropy.data_ptr(), r.rank.data_ptr()
        if top:
            a.top_id, a.top_logprob = r.top_ids.data_ptr(), r.top_logprobs.data_ptr()
        _call("ws_token_logprobs", a)
    return r
