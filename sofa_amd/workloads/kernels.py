"""Operators of the decoder training step as HIP kernels for MI355X.

    attention(q, k, v)            self-attention over grouped heads
    token_logprobs(logits, ids)   log p(token), entropy, alternatives
    residual_norm(x, branch, w)   residual sum and the RMS norm of it

All three are differentiable (first derivatives), run on the current stream of
their tensors' device, allocate what they return and nothing that outlives the
call, give the same bits for the same inputs, and can be captured into a graph.
They need tensors on a GPU: there is no other path, and a missing library is an
error.  Wrong arguments raise TypeError (types) or ValueError (shapes, values).

`Llama(kernels="hip")` and `python -m sofa_amd.workloads.llama --kernels hip`
run the decoder on them.  The kernels are in native/hip/model.
"""

from __future__ import annotations

import ctypes
import math
import os
from typing import NamedTuple, Optional, Tuple

import torch

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}

MAX_HEAD_DIM = 128
MAX_TOKENS = 1 << 24
MAX_TOP = 32
MAX_NORM_DIM = 16384
MAX_VOCAB = 1 << 30

_P, _I, _L, _F = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_float


def _struct(name, *fields):
    """A ctypes structure out of (type, "names ...") pairs, in order."""
    return type(name, (ctypes.Structure,), {
        "_fields_": [(n, t) for t, names in fields for n in names.split()]
    })


# the argument structures of the C entries, field by field
_AttentionArgs = _struct(
    "_AttentionArgs",
    (_P, "q k v o lse lengths dout delta dq dk dv stream"),
    (_L * 3, "q_stride k_stride v_stride o_stride dout_stride dq_stride dk_stride dv_stride"),
    (_F, "scale"),
    (_I, "batch heads kv_heads tokens dim causal device"),
)
_LogprobArgs = _struct(
    "_LogprobArgs",
    (_P, "logits tokens logprob entropy lse top_ids top_logprobs part_sums part_top "
         "dlogprob dentropy dlogits stream"),
    (_L, "rows inner outer_stride inner_stride grad_outer_stride grad_inner_stride "
         "grad2_outer_stride grad2_inner_stride token_outer_stride token_inner_stride ignore_index"),
    (_I, "vocab top parts part_size type device"),
)
_NormArgs = _struct(
    "_NormArgs",
    (_P, "x branch weight post gate r y dr dy dx dbranch partial dweight dpost dgate stream"),
    (_L, "rows group_rows"),
    (_F, "eps scale"),
    (_I, "dim x_type branch_type y_type weight_type post_type gate_type teams_per_group device"),
)

_lib_handle = None


def _lib():
    global _lib_handle
    if _lib_handle is None:
        path = os.path.join(
            os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
            "native", "lib", "libsofamodel.so",
        )
        if not os.path.exists(path):
            raise RuntimeError(f"{path} is not built: run python -m sofa_amd.native.build")
        lib = ctypes.CDLL(path)  # after torch, whose HIP runtime it shares
        for name in ("attention_forward", "attention_backward", "logprob_forward",
                     "logprob_backward", "norm_forward", "norm_backward"):
            entry = getattr(lib, "sofa_" + name)
            entry.argtypes, entry.restype = [_P], _I
        lib.sofa_norm_backward_teams.argtypes = [_L, _L, _I]
        lib.sofa_norm_backward_teams.restype = _I
        _lib_handle = lib
    return _lib_handle


def _call(name: str, args) -> None:
    status = getattr(_lib(), name)(ctypes.addressof(args))
    if status:
        what = "bad argument" if status < 0 else f"HIP error {status}"
        raise RuntimeError(f"{name} failed: {what}")


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _on_gpu(what: str, first: torch.Tensor, **others: Optional[torch.Tensor]) -> None:
    if first.device.type != "cuda":
        raise ValueError(f"{what}: tensors on a GPU are needed, got one on {first.device}")
    for name, t in others.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{what}: {name} is on {t.device}, not on {first.device}")


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def _recorded(*tensors: Optional[torch.Tensor]) -> bool:
    """Whether autograd will ask for a backward pass."""
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------ attention
def _rows16(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy, with dense rows that start at multiples of 16 bytes."""
    if (t.stride(3) == 1 and t.data_ptr() % 16 == 0
            and all(s % 8 == 0 or n == 1 for s, n in zip(t.stride()[:3], t.shape[:3]))):
        return t
    return t.contiguous()


def _token_major(batch: int, heads: int, tokens: int, dim: int, like: torch.Tensor) -> torch.Tensor:
    """(batch, heads, tokens, dim) laid out as (batch, tokens, heads, dim): what
    the projection behind it reads as one matrix without a copy."""
    return torch.empty((batch, tokens, heads, dim), dtype=like.dtype, device=like.device).transpose(1, 2)


def _attention_args(q, k, v, o, lse, lengths, scale, causal):
    a = _AttentionArgs()
    a.q, a.k, a.v, a.o = q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr()
    a.lse, a.lengths = _ptr(lse), _ptr(lengths)
    a.q_stride[:], a.k_stride[:] = q.stride()[:3], k.stride()[:3]
    a.v_stride[:], a.o_stride[:] = v.stride()[:3], o.stride()[:3]
    a.scale, a.causal = scale, causal
    a.batch, a.heads, a.tokens, a.dim = q.shape
    a.kv_heads = k.shape[1]
    a.device = q.device.index
    a.stream = _stream(q.device)
    return a


def _attention_forward(q, k, v, lengths, scale, causal, with_lse):
    q, k, v = _rows16(q), _rows16(k), _rows16(v)
    o = _token_major(*q.shape, q)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if with_lse else None
    _call("sofa_attention_forward", _attention_args(q, k, v, o, lse, lengths, scale, causal))
    return q, k, v, o, lse


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, lengths, scale, causal):
        q, k, v, o, lse = _attention_forward(q, k, v, lengths, scale, causal, True)
        ctx.save_for_backward(q, k, v, o, lse, lengths)
        ctx.scale, ctx.causal = scale, causal
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dout):
        q, k, v, o, lse, lengths = ctx.saved_tensors
        dout = _rows16(dout)
        delta = torch.empty_like(lse)
        dq = _token_major(*q.shape, q)
        dk, dv = _token_major(*k.shape, k), _token_major(*v.shape, v)
        a = _attention_args(q, k, v, o, lse, lengths, ctx.scale, ctx.causal)
        a.dout, a.delta = dout.data_ptr(), delta.data_ptr()
        a.dq, a.dk, a.dv = dq.data_ptr(), dk.data_ptr(), dv.data_ptr()
        a.dout_stride[:], a.dq_stride[:] = dout.stride()[:3], dq.stride()[:3]
        a.dk_stride[:], a.dv_stride[:] = dk.stride()[:3], dv.stride()[:3]
        _call("sofa_attention_backward", a)
        return dq, dk, dv, None, None, None


def attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    *,
    lengths: Optional[torch.Tensor] = None,
    causal: bool = True,
    scale: Optional[float] = None,
) -> torch.Tensor:
    """softmax(scale q k^T + mask) v for queries and keys of the same tokens.

    q is (batch, heads, tokens, dim); k and v are (batch, kv_heads, tokens, dim),
    where kv_heads divides heads and query head i reads key head
    i // (heads // kv_heads).  All are bfloat16; dim is a multiple of 8 up to
    128; any strides (rows that are not dense or not at multiples of 16 bytes
    are copied first).  scale is above 0, 1 / sqrt(dim) if not given.

    causal: token i sees tokens 0..i, otherwise all.  lengths: int32 (batch,),
    the valid tokens at the front of each sequence, taken as within 0..tokens;
    what stands behind them is never used, whatever it is, and its results and
    gradients are zeros.  Valid tokens have to be finite, the later ones that a
    causal mask hides included.

    float16 is refused: the gradient of a score, which the products of the
    backward pass take in the inputs' type, is below float16's smallest normal
    value in long sequences.

    Returns (batch, heads, tokens, dim), laid out as (batch, tokens, heads, dim).
    """
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 4:
            raise ValueError(f"attention: {name} has to be (batch, heads, tokens, dim), got {tuple(t.shape)}")
        if t.dtype != torch.bfloat16:
            raise TypeError(f"attention: {name} has to be bfloat16, got {t.dtype}")
    batch, heads, tokens, dim = q.shape
    if k.shape != v.shape or k.shape[0] != batch or k.shape[2:] != q.shape[2:]:
        raise ValueError(
            f"attention: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if min(k.shape[1], heads) < 1 or heads % k.shape[1]:
        raise ValueError(f"attention: {heads} heads cannot share {k.shape[1]} key heads")
    if dim < 8 or dim % 8 or dim > MAX_HEAD_DIM:
        raise ValueError(f"attention: dim has to be a multiple of 8 up to {MAX_HEAD_DIM}, got {dim}")
    if tokens > MAX_TOKENS or batch * heads * -(-tokens // 128) > 2**31 - 1:
        raise ValueError(f"attention: {tuple(q.shape)} is too large")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    elif not (math.isfinite(scale) and scale > 0):
        raise ValueError(f"attention: scale has to be above 0 and finite, got {scale}")
    if lengths is not None:
        if lengths.dtype != torch.int32:
            raise TypeError(f"attention: lengths has to be int32, got {lengths.dtype}")
        if lengths.shape != (batch,):
            raise ValueError(f"attention: lengths has to be ({batch},), got {tuple(lengths.shape)}")
    _on_gpu("attention", q, k=k, v=v, lengths=lengths)
    if q.numel() == 0:
        return q + 0 * (k.sum() + v.sum())  # no tokens: empty, and still part of the graph
    if lengths is not None:
        lengths = lengths.contiguous()
    if not _recorded(q, k, v):
        return _attention_forward(q, k, v, lengths, float(scale), bool(causal), False)[3]
    return _Attention.apply(q, k, v, lengths, float(scale), bool(causal))


# ------------------------------------------------------------------ token log probabilities
class TokenLogprobs(NamedTuple):
    """logprob and entropy (differentiable) have the tokens' shape; top_ids and
    top_logprobs have one more axis of `top`, most likely first, or are None."""

    logprob: torch.Tensor
    entropy: torch.Tensor
    top_ids: Optional[torch.Tensor]
    top_logprobs: Optional[torch.Tensor]


def _two_level(t: torch.Tensor, axes: int) -> Optional[Tuple[int, int, int]]:
    """(inner, outer_stride, inner_stride) such that element i of t's first `axes`
    axes is at i // inner * outer_stride + i % inner * inner_stride; None if two
    levels are not enough."""
    levels = []  # innermost first: [size, stride]
    for n, s in zip(reversed(t.shape[:axes]), reversed(t.stride()[:axes])):
        if n == 1:
            continue
        if levels and s == levels[-1][0] * levels[-1][1]:
            levels[-1][0] *= n
        else:
            levels.append([n, s])
    if len(levels) > 2:
        return None
    inner, inner_stride = levels[0] if levels else (1, 0)
    return inner, levels[1][1] if len(levels) > 1 else 0, inner_stride


def _same_split(inner: int, rows: int, t: torch.Tensor, axes: int):
    """t's strides over rows that are split at `inner`, copying t if it needs it."""
    split = _two_level(t, axes)
    if split is not None:
        n, outer, step = split
        if n == inner:
            return t, outer, step
        if n >= rows:  # one level: it can be split anywhere
            return t, inner * step, step
    t = t.contiguous()
    return t, inner, 1


def _logprob_split(rows: int, vocab: int) -> Tuple[int, int]:
    """(parts, part_size): a row goes to one workgroup while there are rows for
    every compute unit twice over; below that it is cut into parts."""
    step = 2048  # what a workgroup of 256 threads reads at a time
    parts = max(1, min(64, -(-512 // rows), -(-vocab // step)))
    size = -(-vocab // (parts * step)) * step
    return -(-vocab // size), size


def _logprob_args(logits, tokens, ignore_index, logprob, entropy, lse):
    a = _LogprobArgs()
    axes = logits.dim() - 1
    a.rows, a.vocab = logprob.numel(), logits.shape[-1]
    a.inner, a.outer_stride, a.inner_stride = _two_level(logits, axes)
    tokens, a.token_outer_stride, a.token_inner_stride = _same_split(a.inner, a.rows, tokens, axes)
    a.logits, a.tokens = logits.data_ptr(), tokens.data_ptr()
    a.logprob, a.entropy, a.lse = logprob.data_ptr(), entropy.data_ptr(), lse.data_ptr()
    a.ignore_index = ignore_index
    a.parts, a.part_size = _logprob_split(a.rows, a.vocab)
    a.type, a.device = _TYPES[logits.dtype], logits.device.index
    a.stream = _stream(logits.device)
    return a, tokens


def _logprob_forward(logits, tokens, top, ignore_index):
    if logits.stride(-1) != 1 or _two_level(logits, logits.dim() - 1) is None:
        logits = logits.contiguous()
    device = logits.device
    logprob, entropy, lse = (torch.empty(tokens.shape, dtype=torch.float32, device=device) for _ in range(3))
    a, tokens = _logprob_args(logits, tokens, ignore_index, logprob, entropy, lse)
    ids = values = None
    if top:
        ids = torch.empty((*tokens.shape, top), dtype=torch.int64, device=device)
        values = torch.empty((*tokens.shape, top), dtype=torch.float32, device=device)
        a.top, a.top_ids, a.top_logprobs = top, ids.data_ptr(), values.data_ptr()
    if a.parts > 1:
        part_sums = torch.empty((a.rows, a.parts, 3), dtype=torch.float32, device=device)
        a.part_sums = part_sums.data_ptr()
        if top:
            part_top = torch.empty((a.rows, a.parts, top), dtype=torch.int64, device=device)
            a.part_top = part_top.data_ptr()
    _call("sofa_logprob_forward", a)
    return logits, tokens, logprob, entropy, lse, ids, values


class _TokenLogprobs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, top, ignore_index):
        logits, tokens, logprob, entropy, lse, ids, values = _logprob_forward(logits, tokens, top, ignore_index)
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(logits, tokens, entropy, lse)
        ctx.ignore_index = ignore_index
        if top:
            ctx.mark_non_differentiable(ids, values)
        return logprob, entropy, ids, values

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dlogprob, dentropy, _ids, _values):
        if dlogprob is None and dentropy is None:
            return None, None, None, None
        logits, tokens, entropy, lse = ctx.saved_tensors
        dlogits = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
        a, tokens = _logprob_args(logits, tokens, ctx.ignore_index, entropy, entropy, lse)
        axes = tokens.dim()
        if dlogprob is not None:
            dlogprob, a.grad_outer_stride, a.grad_inner_stride = _same_split(a.inner, a.rows, dlogprob, axes)
            a.dlogprob = dlogprob.data_ptr()
        if dentropy is not None:
            dentropy, a.grad2_outer_stride, a.grad2_inner_stride = _same_split(a.inner, a.rows, dentropy, axes)
            a.dentropy = dentropy.data_ptr()
        a.dlogits = dlogits.data_ptr()
        _call("sofa_logprob_backward", a)
        return dlogits, None, None, None


def token_logprobs(
    logits: torch.Tensor,
    tokens: torch.Tensor,
    *,
    top: int = 0,
    ignore_index: int = -100,
) -> TokenLogprobs:
    """log p of given tokens, the entropy of their distributions, and the `top`
    (up to 32) most likely tokens, from one reading of the logits.

    logits is (..., vocab) in float32, bfloat16 or float16; tokens is int64 (...).
    The cross entropy of a batch is -logprob.sum() / counted, and needs no copy
    of the logits in 32 bits.  Results are float32, gradients have the logits'
    type.

    A token equal to ignore_index has log probability 0 and passes no gradient
    on; its entropy and alternatives are there all the same.  Any other token
    outside 0..vocab-1 has log probability NaN.  Logits of -inf are tokens that
    are not allowed.  A row without an allowed token has log probability -inf,
    entropy 0 and gradient 0; one with a NaN or +inf has NaN throughout.
    Alternatives of equal logits come in the order of their tokens.
    """
    if logits.dim() < 1 or logits.shape[:-1] != tokens.shape:
        raise ValueError(
            f"token_logprobs: logits {tuple(logits.shape)} and tokens {tuple(tokens.shape)} do not belong together")
    if logits.dtype not in _TYPES:
        raise TypeError(f"token_logprobs: logits have to be float32, bfloat16 or float16, got {logits.dtype}")
    if tokens.dtype != torch.int64:
        raise TypeError(f"token_logprobs: tokens have to be int64, got {tokens.dtype}")
    vocab = logits.shape[-1]
    if not 1 <= vocab <= MAX_VOCAB:
        raise ValueError(f"token_logprobs: a vocabulary of 1 to {MAX_VOCAB} is needed, got {vocab}")
    if not 0 <= top <= min(MAX_TOP, vocab):
        raise ValueError(f"token_logprobs: top has to be within 0..{min(MAX_TOP, vocab)}, got {top}")
    if tokens.numel() > 2**31 - 1:
        raise ValueError(f"token_logprobs: {tokens.numel()} rows are too many")
    _on_gpu("token_logprobs", logits, tokens=tokens)
    if tokens.numel() == 0:
        none = logits.sum(-1, dtype=torch.float32)  # empty, and still part of the graph
        ids = torch.empty((*tokens.shape, top), dtype=torch.int64, device=logits.device) if top else None
        return TokenLogprobs(none, none * 1, ids, None if ids is None else ids.float())
    if not _recorded(logits):
        _, _, logprob, entropy, _, ids, values = _logprob_forward(logits, tokens, int(top), int(ignore_index))
        return TokenLogprobs(logprob, entropy, ids, values)
    return TokenLogprobs(*_TokenLogprobs.apply(logits, tokens, int(top), int(ignore_index)))


# ------------------------------------------------------------------ residual norm
def _dense(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    return None if t is None else t.contiguous()


def _norm_args(x, branch, weight, post, gate, scale, eps, y_type):
    a = _NormArgs()
    a.x, a.branch, a.weight, a.post, a.gate = x.data_ptr(), _ptr(branch), weight.data_ptr(), _ptr(post), _ptr(gate)
    a.dim = x.shape[-1]
    a.rows = x.numel() // a.dim
    a.group_rows = a.rows if gate is None else a.rows // (gate.numel() // a.dim)
    a.eps, a.scale = eps, scale
    a.x_type, a.y_type, a.weight_type = _TYPES[x.dtype], _TYPES[y_type], _TYPES[weight.dtype]
    # without a branch the type only chooses a kernel, and one is built for it
    a.branch_type = _TYPES[y_type if branch is None else branch.dtype]
    a.post_type = 0 if post is None else _TYPES[post.dtype]
    a.gate_type = 0 if gate is None else _TYPES[gate.dtype]
    a.device = x.device.index
    a.stream = _stream(x.device)
    return a


def _norm_forward(x, branch, weight, post, gate, scale, eps, out_dtype):
    y = torch.empty(x.shape, dtype=out_dtype, device=x.device)
    r = None if branch is None else torch.empty_like(x)
    a = _norm_args(x, branch, weight, post, gate, scale, eps, out_dtype)
    a.r, a.y = _ptr(r), y.data_ptr()
    _call("sofa_norm_forward", a)
    return r, y


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, weight, post, gate, scale, eps, out_dtype):
        r, y = _norm_forward(x, branch, weight, post, gate, scale, eps, out_dtype)
        ctx.set_materialize_grads(False)
        uses_branch = post is not None or gate is not None
        ctx.save_for_backward(x if r is None else r, branch if uses_branch else None, weight, post, gate)
        ctx.scale, ctx.eps, ctx.out_dtype = scale, eps, out_dtype
        ctx.branch_dtype = None if branch is None else branch.dtype
        return r, y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dr, dy):
        if dr is None and dy is None:
            return (None,) * 8
        r, branch, weight, post, gate = ctx.saved_tensors
        dr, dy = _dense(dr), _dense(dy)
        a = _norm_args(r, branch, weight, post, gate, ctx.scale, ctx.eps, ctx.out_dtype)
        if ctx.branch_dtype is not None:
            a.branch_type = _TYPES[ctx.branch_dtype]
        _, need_branch, need_weight, need_post, need_gate = ctx.needs_input_grad[:5]
        dx = torch.empty_like(r)
        dbranch = torch.empty(r.shape, dtype=ctx.branch_dtype, device=r.device) if need_branch else None
        dweight = torch.empty_like(weight) if need_weight else None
        dpost = torch.empty_like(post) if need_post else None
        dgate = torch.empty_like(gate) if need_gate else None
        a.dr, a.dy, a.dx, a.dbranch = _ptr(dr), _ptr(dy), dx.data_ptr(), _ptr(dbranch)
        a.dweight, a.dpost, a.dgate = _ptr(dweight), _ptr(dpost), _ptr(dgate)
        sums = sum(t is not None for t in (dweight, dpost, dgate))
        a.teams_per_group = _lib().sofa_norm_backward_teams(a.rows, a.group_rows, a.dim)
        if sums:
            partial = torch.empty(
                (sums, a.rows // a.group_rows * a.teams_per_group, a.dim), dtype=torch.float32, device=r.device)
            a.partial = partial.data_ptr()
        _call("sofa_norm_backward", a)
        return dx, dbranch, dweight, dpost, dgate, None, None, None


def residual_norm(
    x: torch.Tensor,
    branch: Optional[torch.Tensor],
    weight: torch.Tensor,
    *,
    eps: float = 1e-5,
    post_weight: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    scale: float = 1.0,
    out_dtype: Optional[torch.dtype] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """A block's output onto the residual stream, and the next block's norm of it:

        h = branch, or with post_weight its RMS norm times post_weight
        r = x + scale * gate * h
        y = RMS norm of r, times weight

    in one pass; returns (r, y).  Without a branch r is x itself.  x and branch
    are (..., dim) with dim up to 16384; weight and post_weight are (dim,); gate
    is (dim,), or one row for each sequence, (batch, 1, ..., 1, dim).  r has x's
    type.  y has out_dtype, x's or the branch's type (default: x's).  x is float32
    with a branch of any of the three types, or both are the same 16-bit type;
    weights and gates are of any of them.  The norm is taken of the 32-bit sum,
    before r is rounded.  Tensors that are not contiguous are copied first.
    """
    if x.dim() < 1 or not 1 <= x.shape[-1] <= MAX_NORM_DIM:
        raise ValueError(f"residual_norm: x has to be (..., dim) with dim within 1..{MAX_NORM_DIM}, got {tuple(x.shape)}")
    dim = x.shape[-1]
    for name, t in (("x", x), ("branch", branch), ("weight", weight), ("post_weight", post_weight), ("gate", gate)):
        if t is not None and t.dtype not in _TYPES:
            raise TypeError(f"residual_norm: {name} has to be float32, bfloat16 or float16, got {t.dtype}")
    if branch is None:
        if post_weight is not None or gate is not None or scale != 1.0:
            raise ValueError("residual_norm: post_weight, gate and scale need a branch")
    elif branch.shape != x.shape:
        raise ValueError(f"residual_norm: x {tuple(x.shape)} and branch {tuple(branch.shape)} differ")
    for name, t in (("weight", weight), ("post_weight", post_weight)):
        if t is not None and t.shape != (dim,):
            raise ValueError(f"residual_norm: {name} has to be ({dim},), got {tuple(t.shape)}")
    if gate is not None and gate.shape != (dim,) and (
            x.dim() < 2 or gate.shape != (x.shape[0], *(1,) * (x.dim() - 2), dim)):
        raise ValueError(f"residual_norm: gate has to be ({dim},) or one row a sequence, got {tuple(gate.shape)}")
    if out_dtype is None:
        out_dtype = x.dtype
    branch_dtype = out_dtype if branch is None else branch.dtype
    if x.dtype != torch.float32 and branch_dtype != x.dtype:
        raise TypeError(f"residual_norm: a branch of {branch_dtype} onto {x.dtype} is not built")
    if out_dtype not in (x.dtype, branch_dtype):
        raise TypeError(f"residual_norm: out_dtype has to be {x.dtype} or {branch_dtype}, got {out_dtype}")
    if not (math.isfinite(eps) and eps >= 0):
        raise ValueError(f"residual_norm: eps has to be 0 or more, got {eps}")
    if not math.isfinite(scale):
        raise ValueError(f"residual_norm: scale has to be finite, got {scale}")
    if x.numel() // dim > 2**31 - 1:
        raise ValueError(f"residual_norm: {x.numel() // dim} rows are too many")
    _on_gpu("residual_norm", x, branch=branch, weight=weight, post_weight=post_weight, gate=gate)
    if x.numel() == 0:  # empty, and still part of the graph
        r = x
        for t in (branch, post_weight, gate):
            r = r if t is None else r * t.to(x.dtype)
        return (x if branch is None else r), (r * weight.to(x.dtype)).to(out_dtype)
    args = (*(_dense(t) for t in (x, branch, weight, post_weight, gate)), float(scale), float(eps), out_dtype)
    if _recorded(x, branch, weight, post_weight, gate):
        r, y = _ResidualNorm.apply(*args)
    else:
        r, y = _norm_forward(*args)
    return (x if branch is None else r), y
