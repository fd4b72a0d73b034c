"""Operators between the tensor-parallel steps, on the tensors that the steps take and return.

A decode engine does more between two reduction points than the steps of :mod:`weightstream_b200.tp`: it normalises a
block's output, gates it, adds it to the residual stream and normalises that for the next block (:func:`block_norm`),
normalises queries and keys head by head and rotates them by their positions (:func:`head_norm_rope`), adds the requests'
low-rank adapters to a projection's result (:func:`lora_add`), chooses experts (:func:`moe_route`) and runs them where the
tokens are few (:func:`moe_layer`), and on the vocabulary head's logits it applies biases, penalties and grammars
(:func:`adjust_logits`) and scores given tokens (:func:`token_logprobs`).

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
from ._lib import AdjustLogitsArgs, BlockNormArgs, HeadNormRopeArgs, LoraArgs, MoeLayerArgs, MoeRouteArgs, TokenLogprobsArgs, WsError, \
    WS_ACT_BF16, WS_ACT_F32, WS_GATE_LINEAR, WS_GATE_SIGMOID, WS_LORA_MAX_RANK, WS_MAX_PAIRS, WS_MAX_TOP, WS_OK, WS_SCORE_SIGMOID, \
    WS_SCORE_SOFTMAX, WS_SCORE_SQRTSOFTPLUS

_TYPES = {torch.bfloat16: WS_ACT_BF16, torch.float32: WS_ACT_F32}
_GATES = {"none": WS_GATE_LINEAR, "sigmoid": WS_GATE_SIGMOID}
_SCORES = {"softmax": WS_SCORE_SOFTMAX, "sigmoid": WS_SCORE_SIGMOID, "sqrtsoftplus": WS_SCORE_SQRTSOFTPLUS}


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


# ----------------------------------------------------------------------------- logits under biases, penalties and masks
def _adjust_args(logits, tokens, offsets, prompt_lens, repetition, frequency, presence, bias_ids, bias, bias_offsets, mask, mask_rows,
                 out) -> AdjustLogitsArgs:
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [m, vocab] with vocab >= 1, got {list(logits.shape)}")
    m, vocab = logits.shape
    _dim(m, vocab)
    a = AdjustLogitsArgs()
    a.m, a.vocab = m, vocab
    a.logits, a.ld, a.dtype = logits.data_ptr(), _rows(logits, "logits", m, vocab), _code(logits, "logits")
    if out is not None:
        if out.dtype != logits.dtype:
            raise TypeError(f"out must be {logits.dtype} as logits, got {out.dtype}")
        a.out, a.ldo = out.data_ptr(), _rows(out, "out", m, vocab)

    def entries(t, name, at, at_name):
        """Entries of all rows, one row after the other, and where each row's begin."""
        if t is None:
            if at is not None:
                raise ValueError(f"{at_name} needs {name}")
            return 0
        if at is None:
            raise ValueError(f"{name} needs {at_name}")
        if at.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{at_name} must be int32 or int64, got {at.dtype}")
        _vector(at, at_name, m + 1)
        _vector(t, name, t.shape[0] if t.dim() == 1 else -1, torch.int32)
        return at.element_size()

    a.offset_bytes = entries(tokens, "tokens", offsets, "offsets")
    per_row = (("prompt_lens", prompt_lens, torch.int32), ("repetition", repetition, torch.float32), ("frequency", frequency, torch.float32),
               ("presence", presence, torch.float32))
    for name, t, dtype in per_row:
        if t is not None:
            if tokens is None:
                raise ValueError(f"{name} needs tokens and offsets")
            _vector(t, name, m, dtype)
            setattr(a, name, t.data_ptr())
    if tokens is not None:
        a.tokens, a.offsets, a.n_tokens = tokens.data_ptr(), offsets.data_ptr(), tokens.shape[0]
    a.bias_offset_bytes = entries(bias_ids, "bias_ids", bias_offsets, "bias_offsets")
    if (bias is None) != (bias_ids is None):
        raise ValueError("bias and bias_ids come together")
    if bias is not None:
        _dim(bias_ids.shape[0])
        _vector(bias, "bias", bias_ids.shape[0], torch.float32)
        a.bias_ids, a.bias, a.bias_offsets, a.n_bias = bias_ids.data_ptr(), bias.data_ptr(), bias_offsets.data_ptr(), bias.shape[0]
    if mask is not None:
        if mask.dtype != torch.int32:
            raise TypeError(f"mask must be int32, got {mask.dtype}")
        words = (vocab + 31) // 32
        if mask.dim() != 2 or mask.shape[1] < words:
            raise ValueError(f"mask must be [masks, {words}] words, got {list(mask.shape)}")
        a.ld_mask, a.mask_count = _rows(mask, "mask", *mask.shape), mask.shape[0]
        if mask_rows is None and mask.shape[0] != m:
            raise ValueError(f"{mask.shape[0]} masks for {m} rows: mask_rows is needed")
        _dim(mask.shape[0])
        a.mask = mask.data_ptr() if mask.shape[0] else None
    if mask_rows is not None:
        if mask is None:
            raise ValueError("mask_rows needs mask")
        _vector(mask_rows, "mask_rows", m, torch.int32)
        a.mask_rows = mask_rows.data_ptr()
    _same_device(logits, tokens, offsets, prompt_lens, repetition, frequency, presence, bias_ids, bias, bias_offsets, mask, mask_rows, out)
    return a


def adjust_logits(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None, offsets: Optional[torch.Tensor] = None,
                  prompt_lens: Optional[torch.Tensor] = None, repetition: Optional[torch.Tensor] = None,
                  frequency: Optional[torch.Tensor] = None, presence: Optional[torch.Tensor] = None,
                  bias_ids: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None, bias_offsets: Optional[torch.Tensor] = None,
                  mask: Optional[torch.Tensor] = None, mask_rows: Optional[torch.Tensor] = None, out: Optional[torch.Tensor] = None,
                  stream=None) -> torch.Tensor:
    """Biases, penalties for repeated tokens and grammar masks on the logits [m, vocab] (fp32 as ``lm_head_allgather_argmax``
    returns them, or bf16), in this order, one pass::

        z = logits + bias                                of the tokens that the row lists
        z = z / repetition if z > 0 else z * repetition  of the tokens in the row's history
        z = z - frequency * count - presence             of those that occur ``count`` > 0 times behind its prompt
        z = -inf                                         of the tokens that the row's mask does not allow

    Row ``t``'s history is ``tokens[offsets[t]:offsets[t + 1]]`` (int32 tokens, int32 or int64 offsets [m + 1]), of which the
    first ``prompt_lens[t]`` (int32 [m]; none without it) are the prompt; ``repetition``, ``frequency`` and ``presence`` are fp32
    [m] (1, 0 and 0 without them).  Its biases are ``bias[j]`` (fp32) of ``bias_ids[j]`` (int32) for ``j`` from
    ``bias_offsets[t]`` to ``bias_offsets[t + 1]``; of a token that is listed twice the last entry counts.  Tokens outside
    [0, vocab), such as -1 for padding, are ignored.  ``mask`` is int32 [masks, words >= ceil(vocab / 32)], bit ``v % 32`` of word
    ``v // 32`` allows token ``v``; row ``t`` uses mask row ``mask_rows[t]`` (int32 [m]), or ``t`` without it.  A row whose mask row is
    outside [0, masks), such as -1, has no mask: all its tokens are allowed, so an index of a mask that is gone turns a grammar off.

    Returns ``out``, of the logits' type, which may be ``logits`` itself.  A row that no token is left of is -inf throughout;
    NaN stays NaN.
    """
    r = (_native or _load()).adjust_logits(logits, tokens, offsets, prompt_lens, repetition, frequency, presence, bias_ids, bias, bias_offsets,
                                         mask, mask_rows, out, _handle(stream, logits))
    if r is not None:
        return r
    _tensors(logits=logits)
    _tensors(True, tokens=tokens, offsets=offsets, prompt_lens=prompt_lens, repetition=repetition, frequency=frequency, presence=presence,
             bias_ids=bias_ids, bias=bias, bias_offsets=bias_offsets, mask=mask, mask_rows=mask_rows, out=out)
    a = _adjust_args(logits, tokens, offsets, prompt_lens, repetition, frequency, presence, bias_ids, bias, bias_offsets, mask, mask_rows, out)
    with _on(logits.device, stream):
        out = out if out is not None else torch.empty((a.m, a.vocab), dtype=logits.dtype, device=logits.device)
        a.out, a.ldo = out.data_ptr(), a.ldo or a.vocab
        _call("ws_adjust_logits", a)
    return out


# ----------------------------------------------------------------------------- norms and rotation of heads
def _heads(t: torch.Tensor, name: str, m: int, d: int) -> Tuple[int, int]:
    """Strides from token to token and from head to head of a [m, heads, d] tensor."""
    if t.dim() != 3 or t.shape[0] != m or t.shape[2] != d:
        raise ValueError(f"{name} must be [{m}, heads, {d}], got {list(t.shape)}")
    if d > 1 and t.stride(2) != 1 and t.numel():
        raise ValueError(f"{name} needs unit inner stride")
    heads = t.shape[1]
    return t.stride(0) if m > 1 else heads * d, t.stride(1) if heads > 1 else d


def _apart(t: torch.Tensor, name: str, like: torch.Tensor) -> Tuple[int, int]:
    """Strides of a result: no value is written twice."""
    if t.shape != like.shape:
        raise ValueError(f"{name} must be {list(like.shape)}, got {list(t.shape)}")
    if t.dtype != like.dtype:
        raise TypeError(f"{name} must be {like.dtype}, got {t.dtype}")
    m, heads, d = t.shape
    token, head = _heads(t, name, m, d)
    if not (head >= d and token >= (heads - 1) * head + d) and not (token >= d and head >= (m - 1) * token + d):
        raise ValueError(f"{name}: heads of different tokens overlap")
    return token, head


def _head_norm_rope_args(q, k, positions, inv_freq, q_weight, k_weight, norm, eps, weight_offset, rotary_start, interleaved, rope_scale,
                         q_out, k_out) -> HeadNormRopeArgs:
    if q.dim() != 3 or q.shape[2] < 1:
        raise ValueError(f"q must be [m, heads, d] with d >= 1, got {list(q.shape)}")
    m, q_heads, d = q.shape
    _dim(m, q_heads, d)
    a = HeadNormRopeArgs()
    a.m, a.q_heads, a.d, a.dtype = m, q_heads, d, _code(q, "q")
    a.q, (a.ldqt, a.ldqh) = q.data_ptr(), _heads(q, "q", m, d)
    if k is not None:
        if k.dtype != q.dtype:
            raise TypeError(f"k must be {q.dtype} as q, got {k.dtype}")
        a.ldkt, a.ldkh = _heads(k, "k", m, d)
        _dim(k.shape[1])
        a.k, a.k_heads = (k.data_ptr(), k.shape[1]) if k.numel() else (None, 0)
    elif k_weight is not None or k_out is not None:
        raise ValueError("k_weight and k_out need k")
    weights = [(w, name) for w, name in ((q_weight, "q_weight"), (k_weight, "k_weight")) if w is not None]
    for w, name in weights:
        _vector(w, name, d)
        a.weight_dtype = _code(w, name)
        setattr(a, name, w.data_ptr())
    if len(weights) == 2 and q_weight.dtype != k_weight.dtype:
        raise TypeError("q_weight and k_weight must have one type")
    if (positions is None) != (inv_freq is None):
        raise ValueError("positions and inv_freq come together")
    a.position_bytes = 8
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"positions must be int32 or int64, got {positions.dtype}")
        _vector(positions, "positions", m)
        _vector(inv_freq, "inv_freq", inv_freq.shape[0] if inv_freq.dim() == 1 else -1, torch.float32)
        if not 1 <= inv_freq.shape[0] <= WS_MAX_PAIRS:
            raise ValueError(f"inv_freq must hold 1..{WS_MAX_PAIRS} values, got {inv_freq.shape[0]}")
        a.positions, a.position_bytes, a.inv_freq, a.pairs = positions.data_ptr(), positions.element_size(), inv_freq.data_ptr(), inv_freq.shape[0]
        if rotary_start < 0 or rotary_start + 2 * a.pairs > d:
            raise ValueError(f"{a.pairs} pairs from {rotary_start} on are not within {d} values")
        a.start = rotary_start
    if not eps >= 0.0:
        raise ValueError("eps must not be negative")
    a.norm, a.interleaved, a.eps, a.weight_offset, a.scale = bool(norm), bool(interleaved), eps, weight_offset, rope_scale
    if q_out is not None:
        a.q_out, (a.ldqt_out, a.ldqh_out) = q_out.data_ptr(), _apart(q_out, "q_out", q)
    if k_out is not None:
        a.k_out, (a.ldkt_out, a.ldkh_out) = k_out.data_ptr(), _apart(k_out, "k_out", k)
    _same_device(q, k, positions, inv_freq, q_weight, k_weight, q_out, k_out)
    return a


def head_norm_rope(q: torch.Tensor, k: Optional[torch.Tensor] = None, *, positions: Optional[torch.Tensor] = None,
                   inv_freq: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                   norm: bool = True, eps: float = 1e-6, weight_offset: float = 0.0, rotary_start: int = 0, interleaved: bool = False,
                   rope_scale: float = 1.0, q_out: Optional[torch.Tensor] = None, k_out: Optional[torch.Tensor] = None,
                   stream=None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Norms of queries and keys head by head and the rotation of their positions, in one pass.

    ``q`` [m, heads, d] and ``k`` [m, other heads, d] (bf16 or fp32, any strides between tokens and heads, so slices of a fused
    projection's rows will do)::

        u        = x * rsqrt(mean(x^2) + eps) * (weight_offset + weight)      over the d values of a head
        (a', b') = rope_scale * (a cos - b sin, a sin + b cos)                angle = positions[t] * inv_freq[i]

    for the ``len(inv_freq)`` pairs of the part that begins at ``rotary_start``: value i and the one ``len(inv_freq)`` behind it,
    or with ``interleaved`` neighbours.  Values outside the part keep ``u``.  Without weights they count as one and
    ``weight_offset`` is not added; ``norm=False`` leaves the norm out, no ``positions`` the rotation.  The angle is exact for
    positions (int32 or int64) up to 2^53; everything else between the loads and the one rounding is held in 32 bits.

    Returns ``(q', k')`` of the inputs' type, contiguous or in ``q_out`` and ``k_out``, which may be ``q`` and ``k`` themselves.
    """
    r = (_native or _load()).head_norm_rope(q, k, positions, inv_freq, q_weight, k_weight, norm, eps, weight_offset, rotary_start, interleaved,
                                          rope_scale, q_out, k_out, _handle(stream, q))
    if r is not None:
        return r
    _tensors(q=q)
    _tensors(True, k=k, positions=positions, inv_freq=inv_freq, q_weight=q_weight, k_weight=k_weight, q_out=q_out, k_out=k_out)
    a = _head_norm_rope_args(q, k, positions, inv_freq, q_weight, k_weight, norm, eps, weight_offset, rotary_start, interleaved, rope_scale,
                             q_out, k_out)
    with _on(q.device, stream):
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
            a.q_out, (a.ldqt_out, a.ldqh_out) = q_out.data_ptr(), _apart(q_out, "q_out", q)
        if k is not None and k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=k.device)
            a.k_out, (a.ldkt_out, a.ldkh_out) = k_out.data_ptr(), _apart(k_out, "k_out", k)
        _call("ws_head_norm_rope", a)
    return q_out, k_out


# ----------------------------------------------------------------------------- experts
def _moe_route_args(logits, top_k, score, bias, renormalize, scale) -> MoeRouteArgs:
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [m, experts] with experts >= 1, got {list(logits.shape)}")
    m, experts = logits.shape
    _dim(m, experts)
    if not 1 <= top_k <= experts:
        raise ValueError(f"top_k must be in 1..{experts}, got {top_k}")
    if score not in _SCORES:
        raise ValueError(f"score must be one of {sorted(_SCORES)}, got {score!r}")
    a = MoeRouteArgs()
    a.m, a.experts, a.top_k, a.score, a.renormalize, a.scale = m, experts, top_k, _SCORES[score], bool(renormalize), scale
    a.logits, a.ld, a.dtype = logits.data_ptr(), _rows(logits, "logits", m, experts), _code(logits, "logits")
    if bias is not None:
        _vector(bias, "bias", experts, torch.float32)
        a.bias = bias.data_ptr()
    _same_device(logits, bias)
    return a


def moe_route(logits: torch.Tensor, top_k: int, *, score: str = "softmax", bias: Optional[torch.Tensor] = None, renormalize: bool = True,
              scale: float = 1.0, stream=None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Experts of every token and their weights from the gate's logits [m, experts] (fp32 or bf16), as
    ``Endpoint.moe_down_combine_allreduce`` and :func:`moe_layer` take them: ids int32 and weights fp32, [m, top_k].

    A token's experts are the ``top_k`` (at most 32, of at most 1024 experts; more raise ``WsError``) of the largest
    ``score + bias``, larger first and equal ones by index; ``bias`` (fp32 [experts]) counts for the choice alone.  ``score`` is
    ``"softmax"``, ``"sigmoid"`` or ``"sqrtsoftplus"`` of the logits.  A weight is ``scale * score``, with ``renormalize`` over the
    sum of the chosen scores.  The choice is that of exact scores: near ones are compared in 64 bits.

    Experts whose logit is -inf or NaN, or whose key is NaN (all of a row's with softmax and a logit of +inf), are never chosen;
    places that stay empty hold id -1 and weight 0.
    """
    r = (_native or _load()).moe_route(logits, top_k, _SCORES.get(score, -1), bias, renormalize, scale, _handle(stream, logits))
    if r is not None:
        return r
    _tensors(logits=logits)
    _tensors(True, bias=bias)
    a = _moe_route_args(logits, top_k, score, bias, renormalize, scale)
    with _on(logits.device, stream):
        ids = torch.empty((a.m, top_k), dtype=torch.int32, device=logits.device)
        weights = torch.empty((a.m, top_k), dtype=torch.float32, device=logits.device)
        a.ids, a.weights = ids.data_ptr(), weights.data_ptr()
        _call("ws_moe_route", a)
    return ids, weights


def _experts(w: torch.Tensor, s: torch.Tensor, name: str, rows: int, k: int, experts: int) -> Tuple[int, int]:
    """Bytes from expert to expert of packed weights [experts, rows, k / 2] and their scales [experts, rows, k / 32]."""
    strides = []
    for t, what, width in ((w, "w" + name, k // 2), (s, "s" + name, k // 32)):
        if t.element_size() != 1:
            raise TypeError(f"{what} must be bytes, got {t.dtype}")
        if list(t.shape) != [experts, rows, width]:
            raise ValueError(f"{what} must be [{experts}, {rows}, {width}], got {list(t.shape)}")
        if (width > 1 and t.stride(2) != 1) or t.stride(1) != width:
            raise ValueError(f"{what}: an expert's rows must lie one after the other")
        strides.append(t.stride(0) if experts > 1 else rows * width)
        if t.data_ptr() % 16 or strides[-1] % 16 or strides[-1] < rows * width:
            raise ValueError(f"{what}: experts must be 16-byte aligned and apart")
    return strides


def _moe_layer_args(x, route_ids, route_w, w1, s1, w3, s3, w2, s2, e_start, limit, act_quant, out, out_dtype) -> MoeLayerArgs:
    if x.dim() != 2 or x.shape[1] < 32 or x.shape[1] % 32:
        raise ValueError(f"x must be [m, hidden] with hidden a multiple of 32, got {list(x.shape)}")
    m, hidden = x.shape
    if w1.dim() != 3 or w1.shape[0] < 1 or w1.shape[1] < 32 or w1.shape[1] % 32:
        raise ValueError(f"w1 must be [experts, inter, hidden / 2] with inter a multiple of 32, got {list(w1.shape)}")
    experts, inter = w1.shape[:2]
    _dim(m, hidden, inter, experts)
    a = MoeLayerArgs()
    a.m, a.hidden, a.inter, a.e_start, a.e_len = m, hidden, inter, e_start, experts
    a.x, a.ldx, a.x_dtype = x.data_ptr(), _rows(x, "x", m, hidden), _code(x, "x")
    if route_ids.dtype != torch.int32 or route_w.dtype != torch.float32:
        raise TypeError(f"route_ids must be int32 and route_w fp32, got {route_ids.dtype} and {route_w.dtype}")
    if route_ids.dim() != 2 or route_ids.shape[0] != m or route_ids.shape[1] < 1 or route_w.shape != route_ids.shape:
        raise ValueError(f"route_ids and route_w must be [{m}, top_k], got {list(route_ids.shape)} and {list(route_w.shape)}")
    if not route_ids.is_contiguous() or not route_w.is_contiguous():
        raise ValueError("route_ids and route_w must be contiguous")
    a.top_k, a.route_ids, a.route_w = route_ids.shape[1], route_ids.data_ptr(), route_w.data_ptr()
    if not 0 <= e_start < 2 ** 31:
        raise ValueError(f"e_start must not be negative, got {e_start}")
    for name, w, s, rows, k in (("1", w1, s1, inter, hidden), ("3", w3, s3, inter, hidden), ("2", w2, s2, hidden, inter)):
        strides = _experts(w, s, name, rows, k, experts)
        for what, t, stride in (("w", w, strides[0]), ("s", s, strides[1])):
            setattr(a, what + name, t.data_ptr())
            setattr(a, what + name + "_stride", stride)
    if limit is not None and not C.c_float(limit).value > 0.0:
        raise ValueError(f"limit must be positive in 32 bits, got {limit}")
    a.limit, a.act_quant = limit or 0.0, bool(act_quant)
    dtype = out.dtype if out is not None else out_dtype
    if dtype not in _TYPES:
        raise TypeError(f"results are bf16 or fp32, not {dtype}")
    a.out_dtype = _TYPES[dtype]
    if out is not None:
        a.out, a.ldo = out.data_ptr(), _rows(out, "out", m, hidden)
    _same_device(x, route_ids, route_w, w1, s1, w3, s3, w2, s2, out)
    return a


def moe_layer(x: torch.Tensor, route_ids: torch.Tensor, route_w: torch.Tensor, w1: torch.Tensor, s1: torch.Tensor, w3: torch.Tensor,
              s3: torch.Tensor, w2: torch.Tensor, s2: torch.Tensor, e_start: int = 0, *, limit: Optional[float] = None,
              act_quant: bool = False, out: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.float32,
              stream=None) -> torch.Tensor:
    """A whole mixture-of-experts layer of a few tokens, in two kernels and a sum::

        g, u   = w1[e] @ x[t], w3[e] @ x[t]              with limit: min(g, limit), u between -limit and limit
        out[t] = sum over t's routes of w2[e] @ (route_w * silu(g) * u)

    ``x`` [m, hidden] is bf16 or fp32.  The experts are MXFP4 as ``moe_down_combine_allreduce`` takes them: packed E2M1 codes
    ``w1``, ``w3`` [experts, inter, hidden / 2] and ``w2`` [experts, hidden, inter / 2], a UE8M0 byte per 32 values of K in ``s1``, ``s3``
    and ``s2``.  An expert's rows lie one after the other, experts anywhere, so ``w1`` and ``w3`` may be halves of one tensor.
    ``route_ids`` int32 and ``route_w`` fp32 [m, top_k] are those of :func:`moe_route`; this rank holds the experts from ``e_start``
    on, and routes to others, such as -1, count nothing: the result is then this rank's part, for ``Endpoint.allreduce_``.

    bf16 activations are held as they are, fp32 ones and the weighted hidden in 22 bits or more, down to 2^-17 of their row's
    largest value (bf16: 2^-29) and below that to 2^-40 of it; ``act_quant`` rounds x and the weighted hidden to E4M3 with a power of
    two for 32 values, as the fused steps and the reference do.  Sums are fp32, in units of a row's largest activation, so scale bytes
    above 222 (2^95) may give infinities; a token's routes are added in the order of its slots.  At most 512 routes (m * top_k) of
    top_k 8, 512 experts and widths of 24576; more raise ``WsError``.  Routes and weights may be written by what stands in front of the
    call on its stream.  Returns ``out`` [m, hidden], fp32 or ``out_dtype``.
    """
    r = (_native or _load()).moe_layer(x, route_ids, route_w, w1, s1, w3, s3, w2, s2, e_start, 0.0 if limit is None else limit or -1.0, act_quant,
                                     out, out_dtype, _handle(stream, x))
    if r is not None:
        return r
    _tensors(x=x, route_ids=route_ids, route_w=route_w, w1=w1, s1=s1, w3=w3, s3=s3, w2=w2, s2=s2)
    _tensors(True, out=out)
    a = _moe_layer_args(x, route_ids, route_w, w1, s1, w3, s3, w2, s2, e_start, limit, act_quant, out, out_dtype)
    with _on(x.device, stream):
        out = out if out is not None else torch.empty((a.m, a.hidden), dtype=out_dtype, device=x.device)
        a.out, a.ldo = out.data_ptr(), a.ldo or a.hidden
        size = _lib.load().ws_moe_layer_workspace(a.m, a.top_k, a.hidden, a.inter)
        work = torch.empty(size, dtype=torch.uint8, device=x.device)
        a.workspace, a.workspace_bytes = work.data_ptr(), size
        _call("ws_moe_layer", a)
    return out
